"""How the library is built and the package imported: objects follow the flags, study builds take the
product's, and host-only functions need no GPU."""
import os
import re
import subprocess
import sys
from pathlib import Path

import pytest

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


def make_rules(*args):
    """make's data base for the package: target -> prerequisites."""
    out = subprocess.run(["make", "-C", str(PKG), "-pn", *args], capture_output=True, text=True, timeout=60).stdout
    return {m[1]: m[2].split() for m in re.finditer(r"^([^\s#:=%]+):(?!=)[ ]*(.*)$", out, re.M)}


def test_objects_follow_the_flags():
    """The Makefile holds the flags: every object, the study objects too, is older than it after a change there."""
    rules = make_rules("all", "stamps")
    for f in (PKG / "csrc").glob("*.hip"):
        for at in ("build", "build/stamps"):
            assert "Makefile" in rules[f"{at}/{f.stem}.o"] and f"csrc/{f.name}" in rules[f"{at}/{f.stem}.o"]
        assert f"build/{f.stem}.o" in rules["lib/libwfbitnet.so"]


def test_build_compiles_whatever_is_there(monkeypatch):
    import __graft_entry__ as entry
    calls = []
    monkeypatch.setattr(entry.subprocess, "run", lambda cmd, **kw: calls.append(cmd))
    try:
        entry.build()
    except (ImportError, OSError):  # nothing built yet: the library cannot load
        pass
    assert any(cmd[0] == "make" and str(PKG) in cmd and "-B" in cmd for cmd in calls)


@pytest.mark.parametrize("script,args", [("build_variant.sh", ["name", "-DWF_X=1", "-DWF_Y"]), ("build_var.sh", ["name", "-DWF_X=1 -DWF_Y"]),
                                         ("build_rev.sh", ["HEAD", "name"])])
def test_study_builds_take_the_products_flags(script, args):
    """Every source with the Makefile's flags (packed fp32 instructions off among them) into a library of its own."""
    if script == "build_rev.sh" and not (ROOT / ".git").exists():
        pytest.skip("needs the history")
    out = subprocess.run(["bash", str(ROOT / "tools" / script), *args], env={**os.environ, "MAKEFLAGS": "n"}, capture_output=True, text=True,
                         timeout=60, check=True).stdout  # n: what would be run
    compiled = [line.split() for line in out.splitlines() if " -c " in line]
    assert {Path(next(a for a in c if a.endswith(".hip"))).name for c in compiled} == {f.name for f in (PKG / "csrc").glob("*.hip")}
    flags = re.search(r"^HIPFLAGS \?= (.*)$", (PKG / "Makefile").read_text(), re.M)[1].replace("$(ARCH)", "gfx950").split()
    assert "-packed-fp32-ops" in flags
    for c in compiled:
        assert all(f in c for f in flags) and "build/" in c[c.index("-o") + 1] and not c[c.index("-o") + 1].startswith("build/wf_")
        assert script == "build_rev.sh" or ("-DWF_X=1" in c and "-DWF_Y" in c)
    links = [line.split() for line in out.splitlines() if " -shared " in line]
    assert len(links) == 1 and links[0][links[0].index("-o") + 1] == "lib/libwfbitnet_name.so"
