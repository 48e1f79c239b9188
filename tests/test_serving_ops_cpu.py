"""Serving operators, host side: the C entry points' refusals (no kernel is launched: every call here returns before
one), the Python wrappers' refusals, and rotary_frequencies against its formulas."""
import ctypes as C
import math

import pytest
import torch

BUF = (C.c_uint8 * 4096)()
P = (C.addressof(BUF) + 255) // 256 * 256  # a host address: never read, every call below is refused


def refused(name, args, text):
    from wfamd import _lib
    lib = _lib.load()
    assert getattr(lib, name)(*args) == _lib.WF_EINVAL
    assert text in lib.wf_last_error().decode(), lib.wf_last_error()


def test_page_plan_refusals():
    good = dict(c=P, n=P, B=4, free=P, F=8, table=P, ts=16, cols=16, page=32, T=8, pages=P, slots=P, rows=P, pos=P, cu=P, counts=P,
                ws=None, st=None)

    def call(text, **kw):
        refused("wf_kv_page_plan", list({**good, **kw}.values()), text)
    call("negative", B=-1)
    call("negative", F=-1)
    call("negative", T=-1)
    call("page_size", page=0)
    call("page_size", page=65537)
    call("stride", ts=15)
    call("2^31", ts=1 << 30, cols=1 << 27)
    call("null cu_tokens", cu=None)
    call("null cu_tokens", counts=None)
    call("null lengths", n=None)
    call("null lengths", table=None)
    call("free list", free=None)
    call("token arrays", slots=None)
    call("too many tokens", T=0x7fffffff)
    call("workspace", B=100000)


def test_rotary_refusals():
    good = dict(q=P, qst=512, qsh=128, hq=4, k=P, kst=128, ksh=128, hk=1, dt=1, pos=P, p64=0, f=P, T=2, D=128, r=128, inter=0, s=1.0,
                qo=P, qost=512, qosh=128, ko=P, kost=128, kosh=128, st=None)

    def call(text, **kw):
        refused("wf_rotary_embed", list({**good, **kw}.values()), text)
    call("dtype", dt=3)
    call("negative", T=-1)
    call("negative", hq=-1)
    call("head_dim", D=0)
    call("head_dim", D=513, r=64)
    for r in (0, 7, 130, -2):
        call("rotary_dim", r=r)
    call("null", q=None)
    call("null", ko=None)
    call("null", f=None)
    call("null", pos=None)
    from wfamd import _lib
    lib = _lib.load()
    assert lib.wf_rotary_embed(*{**good, "T": 0}.values()) == _lib.WF_OK  # nothing to do, nothing launched
    assert lib.wf_rotary_embed(*{**good, "hq": 0, "hk": 0}.values()) == _lib.WF_OK


def test_token_logprobs_refusals():
    good = dict(x=P, dt=1, ld=100, R=2, V=100, tok=P, t64=0, k=5, lp=P, rank=P, ent=P, ids=P, top=P, ws=P, st=None)

    def call(text, **kw):
        refused("wf_token_logprobs", list({**good, **kw}.values()), text)
    call("dtype", dt=4)
    call("shape", V=0)
    call("shape", R=-1)
    call("shape", V=(1 << 30) + 1)
    call("top_k", k=65)
    call("top_k", k=-1)
    call("top_k", V=4, ld=4)
    call("stride", ld=99)
    call("null logits", x=None)
    call("null logits", ws=None)
    call("not 16-byte", ws=P + 8)
    call("logprobs / ranks", rank=None)
    call("top_ids", ids=None)
    from wfamd import _lib
    lib = _lib.load()
    assert lib.wf_token_logprobs(*{**good, "R": 0}.values()) == _lib.WF_OK
    assert lib.wf_token_logprobs_ws_bytes(0, 100, 5) == 0 and lib.wf_token_logprobs_ws_bytes(3, 100, 5) >= 3 * (16 + 40)


def test_python_wrappers_refuse_host_tensors():
    from wfamd import ops
    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(ValueError, match="device tensors only"):
        ops.kv_page_plan(i, i, i, torch.zeros(4, 4, dtype=torch.int32), 4)
    q = torch.zeros(4, 2, 64)
    with pytest.raises(ValueError, match="device tensors only"):
        ops.rotary_embed(q, None, i, torch.zeros(32, dtype=torch.float64))
    with pytest.raises(ValueError, match="device tensors only"):
        ops.token_logprobs(torch.zeros(4, 10))


def test_no_overlap():
    from wfamd.ops import _no_overlap
    assert _no_overlap(torch.zeros(4, 3, 8)) and _no_overlap(torch.zeros(4, 6, 8)[:, 1:3]) and _no_overlap(torch.zeros(3, 4, 8).transpose(0, 1))
    assert not _no_overlap(torch.zeros(1, 3, 8).expand(4, 3, 8)) and not _no_overlap(torch.zeros(100).as_strided((3, 2, 8), (4, 8, 1)))
    assert _no_overlap(torch.zeros(1, 1, 8).expand(1, 1, 8))


@pytest.mark.parametrize("r", [2, 4, 64, 80, 128])
def test_rotary_frequencies(r):
    from wfamd.ops import rotary_frequencies
    f, s = rotary_frequencies(r, 500000.0, device="cpu")
    assert f.dtype == torch.float64 and s == 1.0
    for j in range(r // 2):
        assert f[j].item() == pytest.approx(500000.0 ** (-2 * j / r), rel=1e-14)
    lin, s = rotary_frequencies(r, 500000.0, scaling="linear", factor=8.0, device="cpu")
    assert torch.equal(lin, f / 8) and s == 1.0
    ntk, s = rotary_frequencies(r, 500000.0, scaling="ntk", factor=8.0, device="cpu")
    assert ntk[0] == 1.0 and s == 1.0
    if r > 2:
        assert ntk[-1].item() == pytest.approx(f[-1].item() / 8, rel=1e-12)  # the lowest frequency: as 'linear'
    yarn, s = rotary_frequencies(r, 500000.0, scaling="yarn", factor=8.0, original_max_position=4096, device="cpu")
    assert s == pytest.approx(0.1 * math.log(8) + 1)
    turns = f * 4096 / (2 * math.pi)
    assert ((yarn <= f * (1 + 1e-15)) & (yarn >= f / 8 * (1 - 1e-15))).all()
    if r >= 64:
        # a pair and more away from the ramp's rounded ends
        assert torch.equal(yarn[:-1][turns[1:] > 32], f[:-1][turns[1:] > 32])
        assert torch.allclose(yarn[1:][turns[:-1] < 1], f[1:][turns[:-1] < 1] / 8, rtol=1e-14, atol=0)


def test_rotary_frequencies_refusals():
    from wfamd.ops import rotary_frequencies
    for a, kw in (((7,), {}), ((0,), {}), ((64, 1.0), {}), ((64,), {"factor": 0.5, "scaling": "linear"}), ((64,), {"scaling": "x"}),
                  ((64,), {"scaling": "yarn", "factor": 2.0}),
                  ((64,), {"scaling": "yarn", "factor": 2.0, "original_max_position": 64, "beta_fast": 1.0, "beta_slow": 1.0}),
                  ((64,), {"scaling": "yarn", "factor": 2.0, "original_max_position": 64, "beta_slow": 0.0})):
        with pytest.raises(ValueError):
            rotary_frequencies(*a, device="cpu", **kw)


def test_shared_prefix_attention_refusals():
    good = dict(q=P, dt=1, qsb=512, qsh=128, k=P, v=P, kvq=0, pgs=4096, hs=4096, pages=4, pt=P, pts=8, cols=8, lens=P, rows=P, plens=P,
                ks=1.0, vs=1.0, sm=0.1, B=2, hq=4, hkv=1, D=128, out=P, osb=512, osh=128, lse=None, ws=P, st=None)

    def call(text, **kw):
        refused("wf_shared_prefix_attention", list({**good, **kw}.values()), text)
    call("dtype", dt=3)
    call("kv_quant", kvq=3)
    call("head_dim 128", D=64)
    call("bad heads", hq=5, hkv=2)
    call("bad heads", hkv=0)
    call("bad heads", B=-1)
    call("too many", B=65536)
    call("too many", B=60000, hq=64)
    call("bad pool or table", pages=0)
    call("bad pool or table", cols=0)
    call("bad pool or table", pts=7)
    call("bad pool or table", cols=1 << 27, pts=1 << 27)
    call("strides", pgs=4100)
    call("strides", hs=-4096)
    call("strides", kvq=1, hs=4104)
    for kw in ({"sm": 0.0}, {"ks": 0.0}, {"sm": float("inf")}, {"ks": float("nan")}):
        call("finite, not 0", **kw)
    for p in ("q", "k", "v", "pt", "lens", "rows", "plens", "out", "ws"):
        call("null pointer", **{p: None})
    call("aligned", k=P + 8)
    call("aligned", ws=P + 4)
    from wfamd import _lib
    lib = _lib.load()
    assert lib.wf_shared_prefix_attention(*{**good, "B": 0}.values()) == _lib.WF_OK
    assert lib.wf_shared_prefix_attention_ws_bytes(1, 0, 4, 1, 8) == 0 and lib.wf_shared_prefix_attention_ws_bytes(1, 2, 4, 3, 8) == 0
    assert lib.wf_shared_prefix_attention_ws_bytes(1, 2, 4, 1, 8) >= 2 * 4 * 2 * 520


def test_launch_sizes_refused():
    """A grid's threads are counted in 32 bits: sizes past that are refused before the launch."""
    plan = [P, P, 4, P, 8, P, 16, 16, 32, 8, P, P, P, P, P, P, P, None]
    for at, v in ((2, (1 << 24) + 1), (2, 0x7fffffff), (9, 0x7ffff800)):
        refused("wf_kv_page_plan", plan[:at] + [v] + plan[at + 1:], "too many")
    rope = [P, 512, 128, 4, P, 128, 128, 1, 1, P, 0, P, 2, 128, 128, 0, 1.0, P, 512, 128, P, 128, 128, None]
    for at, v in ((12, 1 << 24), (12, 0x7fffffff), (3, 65536), (7, 0x7fffffff)):
        refused("wf_rotary_embed", rope[:at] + [v] + rope[at + 1:], "too many")
    refused("wf_token_logprobs", [P, 1, 100, 1 << 26, 100, P, 0, 5, P, P, P, P, P, P, None], "too many rows")
    pre = dict(q=P, dt=1, qsb=512, qsh=128, k=P, v=P, kvq=0, pgs=4096, hs=4096, pages=4, pt=P, pts=8, cols=8, lens=P, rows=P, plens=P,
               ks=1.0, vs=1.0, sm=0.1, B=2, hq=4, hkv=1, D=128, out=P, osb=512, osh=128, lse=None, ws=P, st=None)
    for kw in ({"B": 65535, "hq": 65535, "hkv": 65535}, {"B": 65535, "hq": 512, "hkv": 512}, {"B": 65535, "hq": 2048, "hkv": 128}):
        refused("wf_shared_prefix_attention", list({**pre, **kw}.values()), "too many")


def _places(t):
    return set((t.data_ptr() + t.element_size() * (t.stride(0) * i + t.stride(1) * h + d)) for i in range(t.shape[0]) for h in range(t.shape[1])
               for d in range(t.shape[2]))


def test_apart():
    """_apart never calls overlapping tensors apart, and knows the arrangements that q and k come in."""
    from wfamd.ops import _apart
    x = torch.zeros(4096, dtype=torch.bfloat16)
    D = 4
    row = x[:5 * 32].view(5, 8, D)           # heads of one row: q, k, v slices
    groups = x[:5 * 48].view(5, 3, 4, D)     # kv groups of (q, q, k, v)
    three = x[:5 * 24].view(5, 6, D)         # q and k heads in turn
    yes = [(row[:, :4], row[:, 4:6]), (row[:, 4:6], row[:, :4]), (three[:, 0::2], three[:, 1::2]), (row[:1, :3], row[:1, 3:]),
           (groups[:, :, 0], groups[:, :, 2]), (x[:160].view(5, 8, D), x[160:240].view(5, 4, D)), (row[:2], row[2:4]),
           (row[:1, :, :2].as_strided((1, 4, D), (0, 8, 1)), row[:1].as_strided((1, 4, D), (0, 8, 1), D))]
    no = [(row, row), (row[:, :4], row[:, 3:6]), (row[:, :4], row[:, :2]), (row[:2], row[1:3]), (three[:, 0::2], three[:, 2::2]),
          (row[:, :4], x[130:130 + 5 * 32].view(5, 8, D)[:, :4]), (groups[:, :, 0], groups[:, :, 0])]
    for a, b in yes:
        assert not _places(a) & _places(b)
        assert _apart(a, b) and _apart(b, a), (a.stride(), b.stride())
    for a, b in no:
        assert _places(a) & _places(b)
        assert not _apart(a, b) and not _apart(b, a), (a.stride(), b.stride())
    g = torch.Generator().manual_seed(0)
    for _ in range(4000):  # any two views: a 'yes' is one
        def view():
            h, t = torch.randint(1, 4, (2,), generator=g).tolist()
            sh = D + int(torch.randint(0, 10, (1,), generator=g))
            st = (h - 1) * sh + D + int(torch.randint(0, 40, (1,), generator=g)) if torch.rand((), generator=g) < .5 else sh * (h + 2)
            return x.as_strided((t, h, D), (st, sh, 1), int(torch.randint(0, 120, (1,), generator=g)))
        a, b = view(), view()
        if torch.rand((), generator=g) < .5:
            b = x.as_strided(b.shape, a.stride(), b.storage_offset())
        from wfamd.ops import _no_overlap
        if _no_overlap(a) and _no_overlap(b) and _apart(a, b):
            assert not _places(a) & _places(b), (a.shape, a.stride(), a.storage_offset(), b.shape, b.stride(), b.storage_offset())
