"""token_logprobs' alternatives where their selection can go wrong: zeros of both signs, +inf, and chunks too long for registers."""
import math

import pytest
import torch

from test_gpu_serving_ops import DT, close, logprobs_ref

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


def check_long(x, tokens, k):
    """Against the definition in 64 bits, in units of u = 2^-24. A chunk of c logits: a lane adds n = c / 64 + 16 terms one after the
    other, whose exponent is a difference and a product (2 |y|, weighted by 2^y: under 2 (1 + 1.45 H)) and whose exp2 is good
    to 2; at each of its c / 1024 tiles its max may rise, which scales the sums by a power (its exponent's 2 |d| 2^d, under
    1.1; exp2's 2; the product: 5 together); lanes and chunks are joined in 12 sums and 5 more such factors; log2, the
    products and differences behind it 4 and 3 |log p|."""
    from wfamd import ops
    R, V = x.shape
    c = chunk_of(R, V)
    assert c > HELD, "this shape's chunks stay in registers"
    p = ops.token_logprobs(x, torch.as_tensor(tokens, device="cuda"), top_k=k)
    lp, rank, ent, ids, top = logprobs_ref(x, tokens, k)
    u = 2.0 ** -24
    base = c / 64 + 16 + 2 + 2 * (1 + 1.45 * ent.clamp(min=0)) + 5 * (c / 1024 + 1) + 12 + 10 + 4
    assert torch.equal(p.ranks.cpu().long(), rank)
    assert torch.equal(p.top_ids.cpu().long(), ids)
    close(p.logprobs, lp, u * (base + 3 * lp.abs().nan_to_num(posinf=0.0)))
    close(p.top_logprobs, top, u * (base[:, None] + 3 * top.abs().nan_to_num(posinf=0.0)))
    close(p.entropy, ent, u * (2 * base * (1 + ent) + 4))  # log z's error, and that of the mean of y, which carries its factors'
    q = ops.token_logprobs(x, None, top_k=k)
    assert q.logprobs is None and torch.equal(q.top_ids, p.top_ids) and torch.equal(q.entropy, p.entropy)
    z = ops.token_logprobs(x, torch.as_tensor(tokens, device="cuda"))
    assert torch.equal(z.ranks, p.ranks) and torch.equal(z.logprobs, p.logprobs)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,vocab,ks", [(3, 300001, (1, 5, 20, 33, 64)), (2, 524321, (20,)), (700, 40003, (5,))])
def test_long_chunks(rows, vocab, ks, dtype):
    g = torch.Generator("cuda").manual_seed(rows)
    x = torch.randn(rows, vocab, generator=g, device="cuda") * 3
    x[1::2] += 8.0 * (torch.arange(vocab, device="cuda") // 8 % 64 < 19)  # the greatest in a few lanes
    x = x.to(DT[dtype])
    tokens = torch.randint(0, vocab, (rows,), generator=g, device="cuda").tolist()
    for k in ks:
        check_long(x, tokens, k)


@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "two values", "masked", "few left", "none left", "lowest", "one group", "edges"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_long_chunks_of_awkward_rows(kind, dtype):
    g = torch.Generator("cuda").manual_seed(1)
    R, V = 3, 300001
    whole = torch.randn(R, V + 1, generator=g, device="cuda") * 2
    x = whole[:, 1:]  # rows that begin off any 16-byte line
    ramp = torch.arange(V, device="cuda") / 50000
    if kind == "equal":
        x.fill_(1.25)
    elif kind == "rising":
        x.copy_(ramp.expand(R, V))
    elif kind == "falling":
        x.copy_(ramp.flip(0).expand(R, V))
    elif kind == "two values":
        x.copy_((x > 3).float())
    elif kind == "masked":
        x[torch.rand(R, V, generator=g, device="cuda") < 0.999] = -math.inf
    elif kind in ("few left", "none left"):
        keep = x[:, 70777:70777 + (11 if kind == "few left" else 0)].clone()
        x.fill_(-math.inf)
        x[:, 70777:70777 + keep.shape[1]] = keep
    elif kind == "lowest":
        x[torch.rand(R, V, generator=g, device="cuda") < 0.9] = torch.finfo(DT[dtype]).min
        x[2] = torch.finfo(DT[dtype]).min
    elif kind == "one group":  # the greatest 40 next to each other
        x[:, 100003:100043] += 30.0
    else:  # the greatest where chunks begin and end
        c = chunk_of(R, V)
        for e in range(-4, 5):
            x[:, c + e::c] += 20.0
        x[:, :3] += 20.0
        x[:, -3:] += 20.0
    x = whole.to(DT[dtype])[:, 1:]
    for k in (1, 20, 64):
        check_long(x, [0, V - 1, 70780], k)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_long_chunks_among_nan_of_both_signs(dtype):
    from wfamd import ops
    g = torch.Generator("cuda").manual_seed(4)
    R, V, k = 3, 300001, 33
    assert chunk_of(R, V) > HELD
    x = torch.randn(R, V, generator=g, device="cuda").to(DT[dtype])
    bits = x.view(torch.int32 if dtype == "f32" else torch.int16)
    bad = torch.rand(R, V, generator=g, device="cuda") < 0.5
    bad[1] = True
    bad[1, [5, 4700, 123456, V - 1]] = False
    bad[2] = True
    neg = torch.rand(R, V, generator=g, device="cuda") < 0.5
    nan = torch.full((), math.nan, dtype=DT[dtype], device="cuda").view(bits.dtype)
    bits[bad] = nan & (2 ** (31 if dtype == "f32" else 15) - 1)
    bits[bad & neg] |= -2 ** (31 if dtype == "f32" else 15)
    assert (x.isnan() == bad).all()
    p = ops.token_logprobs(x, top_k=k)
    want = torch.sort(x.float().nan_to_num(-math.inf), dim=1, descending=True, stable=True).indices[:, :k]
    want[torch.arange(k, device="cuda") >= (~bad).sum(1, keepdim=True)] = -1
    assert torch.equal(p.top_ids.long(), want) and p.top_logprobs.isnan().all() and p.entropy.isnan().all()


@pytest.mark.parametrize("vocab", [1, 700, 40011, 300001])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_probabilities_stay_below_one(dtype, vocab):
    """One logit far above the others, at any level: its log probability is at most 0, the entropy at least 0."""
    from wfamd import ops
    g = torch.Generator("cuda").manual_seed(vocab)
    R = 5 if vocab > 100000 else 60
    for below in (math.inf, 40.0, 15.0):
        level = (torch.rand(R, 1, generator=g, device="cuda") * 200 - 100).to(DT[dtype])
        x = (level.float() - below).to(DT[dtype]).expand(R, vocab).clone()
        at = torch.randint(0, vocab, (R, 1), generator=g, device="cuda")
        x.scatter_(1, at, level)
        p = ops.token_logprobs(x, at[:, 0], top_k=1)
        assert (p.logprobs <= 0).all() and (p.top_logprobs <= 0).all() and (p.entropy >= 0).all()
        lp, rank, ent, ids, top = logprobs_ref(x, at[:, 0].tolist(), 1)
        # in units of 2^-24: a lane adds 1 and c / 64 + 16 terms (90 for the longest chunk here), 40 for exponents' errors, joins and
        # the logarithm as in check_long; 2^-16 of the small terms' sum, |log p|, for their own errors
        close(p.logprobs, lp, 2.0 ** -24 * (90 + 40 + 3 * lp.abs()) + 2.0 ** -16 * lp.abs())
        assert torch.equal(p.ranks.cpu().long(), rank)
