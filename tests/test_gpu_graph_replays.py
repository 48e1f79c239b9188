"""Ops that clear a word or tickets before they reduce, captured into a graph: every replay gives the eager result, with the program's own
work between the replays."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from wfamd import _lib
    assert _lib.kernel_available(), "gfx950 kernels must load (no fallback)"
    torch.cuda.set_device(0)


def replayed(call, change, times=5):
    call()  # whatever the first call loads
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = call()
    for i in range(times):
        change(i)
        g.replay()
        torch.cuda.synchronize()
        held = [t.clone() for t in got]
        torch.randn(1 << 20, device="cuda").sum().item()
        assert all(torch.equal(a, b) for a, b in zip(held, call())), i


@pytest.mark.parametrize("n", [1, 1000, 300001])
def test_absmax_and_quantizer(n):
    from wfamd import _lib, ops
    x = torch.zeros(n, device="cuda")

    def absmax():
        out = torch.empty(1, device="cuda")
        _lib.call("wf_absmax", x.data_ptr(), _lib.WF_F32, n, out.data_ptr(), ops._stream())
        return out

    def change(i):  # a smaller maximum each time: one that was not cleared would stay
        x.normal_().clamp_(-3, 3).mul_(10.0 ** -i)
    replayed(lambda: [ops.kv_absmax(x), absmax()], change)
    change(7)
    assert ops.kv_absmax(x).item() == absmax().item() == x.abs().max().item()


@pytest.mark.parametrize("b,hq,hkv,s", [(1, 4, 1, 2000), (3, 8, 2, 700), (40, 4, 4, 130)])
def test_decode_attention(b, hq, hkv, s):
    from wfamd import ops
    d = 128
    q, k, v = torch.zeros(b, hq, d, device="cuda").bfloat16(), *(torch.zeros(b, hkv, s, d, device="cuda").bfloat16() for _ in range(2))
    lens = torch.full((b,), s, dtype=torch.int32, device="cuda")

    def change(i):
        for t in (q, k, v):
            t.normal_()
        lens.fill_(max(1, s - 97 * i))
    replayed(lambda: [ops.decode_attention(q, k, v, kv_strides=(hkv * s * d, s * d, d), B=b, Hq=hq, Hkv=hkv, D=d, S=s, seq_lens=lens)], change)
