"""The serving operators' integration recipe, run as it is printed, and the decoder's own calls after it."""
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from wfamd import _lib
    assert _lib.kernel_available(), "gfx950 kernels must load (no fallback)"
    torch.cuda.set_device(0)


@pytest.mark.parametrize("new", [[1] * 16, [1 + 7 * b for b in range(16)]])
def test_recipe_keeps_the_decoders_pages(new):
    """Planned pages stay a sequence's when the decoder reserves more for it, and go back to the pool when it is released."""
    from sgl_kernel.kvcache import KVCacheManager
    from wfamd.model import BitNetConfig, BitNetDecoder, from_kv_tiles, synthetic_weights
    text = (ROOT / "INTEGRATION.md").read_text()
    recipe = text.split("## Serving operators around the decode path")[1].split("```python")[1].split("```")[0]
    hq, hkv, layer, batch = 4, 2, 1, 16
    cfg = BitNetConfig(hidden=512, layers=2, n_heads=hq, n_kv_heads=hkv, head_dim=128, inter=768, vocab=1024, max_seq=256)
    dec = BitNetDecoder(cfg, synthetic_weights(cfg), batch=batch, num_pages=96, page_seed=3)
    mgr = KVCacheManager.from_decoder(dec)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    n = sum(new)
    blocks = [-(-m // 32) for m in new]
    qkv = torch.randn(n, hq + 2 * hkv, 128, generator=torch.Generator("cuda").manual_seed(1), device="cuda").bfloat16()
    names = dict(dec=dec, kv_manager=mgr, layer=layer, hq=hq, hkv=hkv, n=n, num_tokens=n, qkv=qkv, v=qkv[:, hq + hkv:].reshape(n, -1).contiguous(),
                 cached_lens=i32([0] * batch), new_lens=i32(new), seq_lens=i32(new), prefix_rows=i32([-1] * batch), prefix_lens=i32([0] * batch),
                 num_pages=sum(blocks) + 3, blocks_held=blocks, torch=torch)
    if "num_pages" not in recipe:
        names["free_pages"] = mgr.allocate_pages(sum(blocks) + 3).cuda()
    exec(recipe, names)
    table, k, v = names.get("table", dec.page_table).clone(), names["k"], names["v"]
    assert int(names["plan"].counts[3]) == 0 and names["o"].shape == (batch, hq, 128)
    dec.reserve(3, 200)
    dec.reserve_batch([32 * x + 1 for x in blocks])
    at = 0
    for b, m in enumerate(new):
        assert torch.equal(dec.page_table[b, :blocks[b]], table[b, :blocks[b]])
        assert len(dec.seq_pages[b]) == (7 if b == 3 else blocks[b] + 1)
        ids = dec.page_table[b, :blocks[b]].long()
        kl, vl = from_kv_tiles(*(c[layer][ids].transpose(0, 1).reshape(hkv, blocks[b] * 32, 128) for c in (dec.k_cache, dec.v_cache)))
        assert torch.equal(kl[:, :m].transpose(0, 1).reshape(m, -1), k[at:at + m].reshape(m, -1))
        assert torch.equal(vl[:, :m].transpose(0, 1).reshape(m, -1), v[at:at + m])
        at += m
    held = torch.cat([torch.as_tensor(p) for p in dec.seq_pages])
    assert held.unique().numel() == held.numel()
    for b in range(batch):
        dec.release(b)
    assert sorted(dec.pool._free) == list(range(96))  # every page once
