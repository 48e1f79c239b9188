"""token_logprobs' alternatives where their selection can go wrong: zeros of both signs and +inf."""
import math

import pytest
import torch

from test_gpu_serving_ops import DT

pytestmark = pytest.mark.gpu
HELD = 4096  # logits of a chunk that stay in registers


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from wfamd import _lib
    assert _lib.kernel_available(), "gfx950 kernels must load (no fallback)"
    torch.cuda.set_device(0)


def chunk_of(rows, vocab):
    """Logits of a chunk, from the workspace that the library asks for: (16 + 8 k) bytes a chunk."""
    from wfamd import _lib
    splits, rest = divmod(_lib.load().wf_token_logprobs_ws_bytes(rows, vocab, 1), 24 * rows)
    assert rest == 0
    return -(-(-(-vocab // splits)) // 32) * 32


def check_order(x, tokens, k):
    """Ranks and alternatives alone: by value, -0 and +0 alike, equal ones by index."""
    from wfamd import ops
    p = ops.token_logprobs(x, torch.as_tensor(tokens, device="cuda"), top_k=k)
    order = torch.sort(x.float() + 0.0, dim=1, descending=True, stable=True).indices
    assert torch.equal(p.top_ids.long(), order[:, :k])
    assert p.ranks.tolist() == [int((order[r] == t).nonzero()) + 1 for r, t in enumerate(tokens)]
    return p


# one chunk in registers, several of them, a chunk that is read again
@pytest.mark.parametrize("vocab", [2048, 40011, 300001])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_zeros_of_both_signs_among_negatives(dtype, vocab):
    assert (chunk_of(4, vocab) > HELD) == (vocab == 300001)
    x = torch.full((4, vocab), -1.0, device="cuda")
    x[0, 3], x[0, 100], x[0, 300] = -0.0, 0.0, 0.0          # the first one negative
    x[1, 3], x[1, 100], x[1, 300] = 0.0, -0.0, 0.0
    x[2, 5:1900:24] = 0.0                                   # more than are asked for, in many lanes, every third -0
    x[2, 5:1900:72] = -0.0
    x[3, 7:2000:31] = -0.0                                  # all of them -0, and one +0 last
    x[3, 2001] = 0.0
    x = x.to(DT[dtype])
    for k in (1, 2, 3, 20, 33, 64):
        for tokens in ((3, 3, 5, 7), (100, 100, 29, 2001), (300, 300, 1877, 38)):
            check_order(x, tokens, k)
    for sign in (1.0, -1.0):  # the two zeros alone in their chunks
        y = torch.full((1, vocab), -3.0, device="cuda")
        y[0, 1111], y[0, vocab - 40] = -0.0 * sign, 0.0 * sign
        assert check_order(y.to(DT[dtype]), [1111], 2).top_ids.tolist() == [[1111, vocab - 40]]


@pytest.mark.parametrize("vocab", [2048, 40011, 300001])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_several_infinities(dtype, vocab):
    assert (chunk_of(6, vocab) > HELD) == (vocab == 300001)
    g = torch.Generator("cuda").manual_seed(vocab)
    x = torch.randn(6, vocab, generator=g, device="cuda").to(DT[dtype])
    inf, high = math.inf, torch.finfo(DT[dtype]).max
    x[0, 777] = inf                          # k = 1: the least that can be among them is +inf itself
    x[1, 9:1900:8] = inf                     # in every lane, more than there are places
    x[2, 11:2000:80] = inf                   # 25 of them
    x[3, 1500], x[3, 20], x[3, 1200] = inf, high, high
    x[4] = inf
    x[5, 64:96], x[5, 1000:1100] = inf, high  # few lanes; the type's highest value behind them
    for k in (1, 2, 3, 20, 33, 64):
        for tokens in ((777, 9, 11, 1500, 0, 64), (0, 17, 2, 20, vocab - 1, 1000), (778, 1897, 1931, 1200, 900, 1099)):
            p = check_order(x, tokens, k)
            assert p.logprobs.isnan().all() and p.entropy.isnan().all() and p.top_logprobs.isnan().all()
