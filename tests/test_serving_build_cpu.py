"""How the package is imported: host-only functions need no GPU."""
import subprocess
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]
PKG = ROOT / "wrinklefree-inference-engine_amd"


def test_ops_import_without_a_gpu_backend():
    """A torch without the GPU's private entries: the module imports, host-only functions run."""
    code = ("import torch, sys\n"
            "for n in ('_cuda_getCurrentRawStream', '_cuda_getDevice'):\n"
            "    if hasattr(torch._C, n): delattr(torch._C, n)\n"
            f"sys.path.insert(0, {str(PKG / 'python')!r})\n"
            "from wfamd import ops\n"
            "f, s = ops.rotary_frequencies(64, device='cpu')\n"
            "assert f.shape == (32,) and s == 1.0\n"
            "try: ops.token_logprobs(torch.zeros(4, 10))\n"
            "except ValueError as e: assert 'device tensors only' in str(e)\n"
            "else: raise AssertionError\n")
    subprocess.run([sys.executable, "-c", code], check=True, timeout=300)
