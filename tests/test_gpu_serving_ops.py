"""Serving operators on the GPU (page plans, rotary positions, token log probabilities) against plain implementations in
64 bits; whole numbers are equal, each tolerance is derived where it stands."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from wfamd import _lib
    assert _lib.kernel_available(), "gfx950 kernels must load (no fallback)"
    torch.cuda.set_device(0)


def i32(x):
    return torch.as_tensor(np.asarray(x), dtype=torch.int32).cuda()


# ------------------------------------------------------------------------------------------------
# page plans
# ------------------------------------------------------------------------------------------------
def plan_ref(cached, new, free, table, n, page):
    """Request after request, token after token."""
    table = table.copy()
    out = {k: np.full(n, -1, np.int64) for k in ("pages", "slots", "rows", "positions")}
    cu, at, asked, taken, refused = [0], 0, 0, 0, 0
    for b, (c, m) in enumerate(zip(cached, new)):
        c, m = max(int(c), 0), max(int(m), 0)
        have, total = -(-c // page), -(-(c + m) // page)
        ok = total <= table.shape[1]
        if ok:
            asked += total - have
            ok = total == have or asked <= len(free)
            if ok and total > have:
                table[b, have:total] = free[asked - (total - have):asked]
                taken = asked
        refused += not ok
        for i in range(m):
            if at < n:
                out["rows"][at], out["positions"][at] = b, c + i
                if ok:
                    out["pages"][at], out["slots"][at] = table[b, (c + i) // page], (c + i) % page
            at += 1
        cu.append(at)
    return out, table, cu, [at, asked, taken, refused]


def check_plan(cached, new, free, table, n, page, view=None):
    from wfamd import ops
    want, wtable, cu, counts = plan_ref(cached, new, free, table, n, page)
    t = i32(table) if view is None else view(table)
    p = ops.kv_page_plan(i32(cached), i32(new), i32(free), t, n, page_size=page)
    for k, w in want.items():
        assert np.array_equal(getattr(p, k).cpu().numpy(), w), k
    assert np.array_equal(t.cpu().numpy(), wtable)
    assert p.cu_tokens.tolist() == cu and p.counts.tolist() == counts


@pytest.mark.parametrize("batch,new,ctx,page", [(1, 1, 0, 32), (1, 1, 31, 32), (1, 1, 32, 32), (3, 7, 40, 1), (128, 1, 4095, 32),
                                                (63, 200, 500, 16), (64, 65, 300, 33), (1025, 9, 100, 32), (2048, 5, 70, 64),
                                                (2049, 5, 70, 64), (5000, 3, 40, 16)])
def test_page_plan(batch, new, ctx, page):
    rng = np.random.default_rng(batch * 31 + page)
    cached, fresh = rng.integers(0, ctx + 1, batch), rng.integers(0, new + 1, batch)  # sequences with no new token among them
    cols = -(-(ctx + new) // page)
    free = rng.permutation(batch * cols + 5)
    table = rng.integers(0, 10 ** 6, (batch, cols))
    n = int(fresh.sum())
    for tokens in {n, n + 11, n // 2}:  # exact, spare places, too few
        check_plan(cached, fresh, free, table, tokens, page)


def test_page_plan_refuses_what_does_not_fit():
    rng = np.random.default_rng(5)
    cached, new = rng.integers(0, 300, 40), rng.integers(1, 200, 40)
    new[7], new[20], cached[25], new[30] = 60000, 0, 5000, 2 ** 31 - 1  # too long for the row, nothing, already too long, far too long
    cached[30] = 2 ** 31 - 1
    table = rng.integers(0, 1000, (40, 16))
    n = int(new[:30].sum()) + 100
    for free in (0, 1, 37, 1000):  # the pool runs out on the way
        check_plan(cached[:30], new[:30], rng.permutation(free), table[:30], n - 100, 32)
    # sums past 31 bits are reported as 2^31 - 1, and nothing else suffers
    from wfamd import ops
    t = i32(table)
    p = ops.kv_page_plan(i32(cached), i32(new), i32(np.arange(1000)), t, n, page_size=32)
    want, wtable, cu, counts = plan_ref(cached[:30], new[:30], np.arange(1000), table[:30], n, 32)
    assert np.array_equal(t.cpu().numpy()[:30], wtable) and np.array_equal(t.cpu().numpy()[30], table[30])
    m = cu[30]
    for k, w in want.items():
        assert np.array_equal(getattr(p, k).cpu().numpy()[:m], w[:m])
    assert (p.rows[m:] == 30).all() and (p.pages[m:] == -1).all() and p.cu_tokens[31].item() == 2 ** 31 - 1


def test_page_plan_negative_lengths_empty_batch_strided_table():
    check_plan([-5, 10, -1], [3, -2, -7], [9, 8, 7], np.zeros((3, 4), np.int64), 5, 4)
    check_plan([], [], [1, 2], np.zeros((0, 4), np.int64), 3, 32)
    check_plan([], [], [], np.zeros((0, 4), np.int64), 0, 32)
    check_plan([5], [0], [], np.zeros((1, 0), np.int64), 0, 32)
    whole = torch.full((6, 20), -9, dtype=torch.int32, device="cuda")

    def view(t):
        v = whole[1:5, 3:11]
        v.copy_(torch.as_tensor(t, dtype=torch.int32))
        return v
    check_plan([40, 0, 3, 100], [100, 1, 40, 156], np.arange(100, 150), np.arange(32).reshape(4, 8), 297, 32, view)
    rest = whole.clone()
    rest[1:5, 3:11] = -9
    assert (rest == -9).all()  # nothing around the table


def test_page_plan_feeds_the_engine_pool_writer():
    """kv_page_plan's pages / slots are scatter_kv's: rows written by one are where the table says."""
    from sgl_kernel.kvcache import KVCacheManager
    from wfamd import ops
    from wfamd.model import BitNetConfig, BitNetDecoder, from_kv_tiles, synthetic_weights
    cfg = BitNetConfig(hidden=512, layers=2, n_heads=4, n_kv_heads=2, head_dim=128, inter=768, vocab=1024, max_seq=256)
    dec = BitNetDecoder(cfg, synthetic_weights(cfg), batch=16, num_pages=64)
    mgr = KVCacheManager.from_decoder(dec)
    new = [5, 0, 40, 64, 33] + [1] * 11
    n = sum(new)
    p = ops.kv_page_plan(i32([0] * 16), i32(new), mgr.allocate_pages(40).cuda(), dec.page_table, n)
    k = torch.randn(n, 2 * 128, device="cuda").bfloat16()
    v = torch.randn(n, 2 * 128, device="cuda").bfloat16()
    mgr.scatter_kv(k, v, p.pages, p.slots, 1)
    assert mgr.invalid_page_count() == 0
    at = 0
    for b, m in enumerate(new):
        nb = -(-m // 32)
        ids = dec.page_table[b, :nb].long()
        kt = dec.k_cache[1][ids].transpose(0, 1).reshape(2, nb * 32, 128)
        vt = dec.v_cache[1][ids].transpose(0, 1).reshape(2, nb * 32, 128)
        if m:
            kl, vl = from_kv_tiles(kt, vt)
            assert torch.equal(kl[:, :m].transpose(0, 1).reshape(m, 256), k[at:at + m])
            assert torch.equal(vl[:, :m].transpose(0, 1).reshape(m, 256), v[at:at + m])
        at += m


# ------------------------------------------------------------------------------------------------
# rotary positions
# ------------------------------------------------------------------------------------------------
def rotary_ref(x, pos, freqs, scale, interleaved):
    x, r = x.double().cpu(), 2 * freqs.shape[0]
    a = pos.double().cpu()[:, None] * freqs.cpu()
    c, s = (a.cos() * scale)[:, None], (a.sin() * scale)[:, None]
    i = torch.arange(0, r, 2) if interleaved else torch.arange(r // 2)
    j = i + 1 if interleaved else i + r // 2
    y = x.clone()
    y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., j] * c + x[..., i] * s
    size = torch.zeros_like(y)
    size[..., i] = size[..., j] = x[..., i].abs() + x[..., j].abs()
    return y, size


def check_rotary(got, x, pos, freqs, scale, interleaved):
    want, size = rotary_ref(x, pos, freqs, scale, interleaved)
    # one rounding to the type (half a step; 2^-25 for f16's subnormals), and in 32 bits: the half turn's 2^-25 times pi and
    # sincos' 2^-23 on cos and sin, 2^-24 each for the scale, a product and the sum: under 2^-21 of |x1| + |x2|
    # the angle itself has 64 bits: 2^-53 of it for this reference's product, and for each of the kernel's 1 / 2pi, its product
    # with the frequency and that with the position (at 10^12, 4e-4: 64 bits say no more there)
    angle = (pos.double().cpu().abs() * freqs.max().item())[:, None, None]
    tol = torch.finfo(x.dtype).eps / 2 * want.abs() + size * scale * (2.0 ** -21 + 4 * 2.0 ** -53 * angle) + (2.0 ** -25 if x.dtype == torch.float16 else 1e-38)
    assert got.dtype == x.dtype and got.shape == x.shape
    worst = ((got.double().cpu() - want).abs() / tol).max().item() if got.numel() else 0.0
    assert worst <= 1.0
    r = 2 * freqs.shape[0]
    assert torch.equal(got[..., r:], x[..., r:])


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,hq,hk,dim,rdim", [(1, 20, 5, 128, 128), (7, 1, 1, 64, 2), (130, 8, 2, 96, 64), (33, 3, 3, 80, 50),
                                                   (5, 2, 1, 33, 32), (2051, 4, 1, 128, 128), (2050, 2, 2, 72, 70), (9, 2, 1, 512, 512)])
def test_rotary(tokens, hq, hk, dim, rdim, interleaved, dtype):
    from wfamd import ops
    g = torch.Generator("cuda").manual_seed(tokens + rdim)
    qkv = (torch.randn(tokens, hq + 2 * hk, dim, generator=g, device="cuda") * 3).to(DT[dtype])
    q, k = qkv[:, :hq], qkv[:, hq:hq + hk]  # columns of one projection
    pos = torch.randint(0, 1 << 20, (tokens,), generator=g, device="cuda")
    freqs, scale = ops.rotary_frequencies(rdim, 500000.0, scaling="yarn", factor=4.0, original_max_position=8192)
    before = qkv.clone()
    yq, yk = ops.rotary_embed(q, k, pos, freqs, interleaved=interleaved, scale=scale)
    assert torch.equal(qkv, before)
    check_rotary(yq, q, pos, freqs, scale, interleaved)
    check_rotary(yk, k, pos, freqs, scale, interleaved)
    # int32 positions, q alone, in place: the same bits, the neighbours untouched
    assert torch.equal(ops.rotary_embed(q, None, pos.int(), freqs, interleaved=interleaved, scale=scale)[0], yq)
    zq, zk = ops.rotary_embed(q, k, pos, freqs, interleaved=interleaved, scale=scale, inplace=True)
    assert zq.data_ptr() == q.data_ptr() and torch.equal(q, yq) and torch.equal(k, yk) and torch.equal(qkv[:, hq + hk:], before[:, hq + hk:])


def test_rotary_far_positions_strides_and_emptiness():
    from wfamd import ops
    freqs, _ = ops.rotary_frequencies(64)
    x = torch.randn(6, 4, 64, device="cuda")
    far = torch.tensor([0, 1, -3, 2 ** 31 - 1, 2 ** 31 + 12345, 10 ** 12], device="cuda")
    check_rotary(ops.rotary_embed(x, None, far, freqs)[0], x, far, freqs, 1.0, False)
    pos = torch.arange(6, device="cuda")
    t = torch.randn(4, 6, 64, device="cuda").transpose(0, 1)  # heads outermost
    check_rotary(ops.rotary_embed(t, None, pos, freqs)[0], t, pos, freqs, 1.0, False)
    e = torch.randn(1, 4, 64, device="cuda").expand(6, 4, 64)  # one row for all positions
    check_rotary(ops.rotary_embed(e, None, pos, freqs)[0], e, pos, freqs, 1.0, False)
    odd = torch.randn(6 * 4 * 64 + 1, device="cuda")[1:].view(6, 4, 64)  # no 16-byte alignment
    check_rotary(ops.rotary_embed(odd, None, pos, freqs, interleaved=True)[0], odd, pos, freqs, 1.0, True)
    d = torch.randn(6, 64, 4, device="cuda").transpose(1, 2)  # dims apart: copied
    check_rotary(ops.rotary_embed(d, None, pos, freqs)[0], d, pos, freqs, 1.0, False)
    q, k = ops.rotary_embed(x[:0], x[:0, :1], pos[:0], freqs)
    assert q.shape == (0, 4, 64) and k.shape == (0, 1, 64)
    with pytest.raises(ValueError):
        ops.rotary_embed(e, None, pos, freqs, inplace=True)
    with pytest.raises(ValueError):
        ops.rotary_embed(d, None, pos, freqs, inplace=True)
    with pytest.raises(ValueError):
        ops.rotary_embed(x, x, pos, freqs, inplace=True)
    for bad in (dict(positions=pos[:5]), dict(positions=pos.float()), dict(freqs=freqs.float()), dict(freqs=torch.zeros(33, device="cuda").double()),
                dict(k=x[:5]), dict(k=x.half()), dict(k=x[..., :32]), dict(q=x[0]), dict(q=x.double()), dict(positions=pos.cpu())):
        kw = dict(q=x, k=None, positions=pos, freqs=freqs)
        kw.update(bad)
        with pytest.raises(ValueError):
            ops.rotary_embed(**kw)


def test_rotary_rotation_is_relative():
    """q . k after turning depends on the distance alone."""
    from wfamd import ops
    freqs, _ = ops.rotary_frequencies(128, 500000.0)
    q, k = torch.randn(1, 1, 128, device="cuda").expand(64, 1, 128), torch.randn(1, 1, 128, device="cuda").expand(64, 1, 128)
    at = torch.arange(64, device="cuda") * 16411
    a, b = ops.rotary_embed(q, None, at + 7, freqs)[0].double(), ops.rotary_embed(k, None, at, freqs)[0].double()
    dots = (a * b).sum(-1).flatten()
    # each turned element is off by under 2^-20 of its pair's size (check_rotary's bound with the rounding)
    tol = 4 * 2.0 ** -20 * (q[0].norm() * k[0].norm()).item()
    assert (dots - dots[0]).abs().max().item() <= tol


# ------------------------------------------------------------------------------------------------
# log probabilities
# ------------------------------------------------------------------------------------------------
def logprobs_ref(x, tokens, k):
    x = x.double().cpu()
    R, V = x.shape
    m = x.amax(1, True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    e = (x - m).exp()
    z = e.sum(1, True)
    ln = z.log()
    y = torch.where(z == 0, torch.full_like(x, -math.inf), x - m - ln)
    ent = -(torch.where(e == 0, torch.zeros_like(y), y) * e / torch.where(z == 0, torch.ones_like(z), z)).sum(1)
    xn = x.numpy()
    order = np.stack([np.lexsort((np.arange(V), -r)) for r in xn]) if V else None
    ids = torch.from_numpy(order[:, :k].astype(np.int64))
    lp, rank = torch.zeros(R, dtype=torch.float64), torch.zeros(R, dtype=torch.int64)
    for r, t in enumerate(tokens):
        if t >= V:
            lp[r] = math.nan
        elif t >= 0:
            lp[r] = y[r, t]
            rank[r] = int(np.nonzero(order[r] == t)[0][0]) + 1
    return lp, rank, ent, ids, y.gather(1, ids)


def close(got, want, tol):
    got = got.double().cpu()
    same = (got == want) | (got.isnan() & want.isnan())
    bad = int((~(same | ((got - want).abs() <= tol))).sum())
    assert bad == 0


def check_logprobs(x, tokens, k):
    """Tolerances in units of 2^-24: a lane adds n <= V / 64 + 16 terms one after the other (n), each exponent y comes of a
    difference and a product (2 |y|, weighted by 2^y: under 2 (1 + 1.45 H)) and an exp2 good to 2, the join adds 12 more
    sums and factors; log2, the products and differences behind it 4 and 3 |log p|. A chunk of a row is at most
    4096 logits long in these tests (rows <= 64, vocabulary <= 2^17 + 2^16), so n <= 80."""
    from wfamd import ops
    R, V = x.shape
    p = ops.token_logprobs(x, torch.as_tensor(tokens, device="cuda"), top_k=k)
    lp, rank, ent, ids, top = logprobs_ref(x, tokens, k)
    u, n = 2.0 ** -24, min(V / 64, 64) + 16
    base = n + 2 + 2 * (1 + 1.45 * ent.clamp(min=0)) + 12 + 4
    assert torch.equal(p.ranks.cpu().long(), rank)
    assert torch.equal(p.top_ids.cpu().long(), ids)
    close(p.logprobs, lp, u * (base + 3 * lp.abs().nan_to_num(posinf=0.0)))
    close(p.top_logprobs, top, u * (base[:, None] + 3 * top.abs().nan_to_num(posinf=0.0)))
    # entropy: log z's error, and that of the mean of y, each term of which carries its factor's
    close(p.entropy, ent, u * (2 * base * (1 + ent) + 4))
    q = ops.token_logprobs(x, None, top_k=k)
    assert q.logprobs is None and q.ranks is None and torch.equal(q.top_ids, p.top_ids) and torch.equal(q.entropy, p.entropy)
    z = ops.token_logprobs(x, torch.as_tensor(tokens, device="cuda"))
    assert z.top_ids.shape == (R, 0) and torch.equal(z.ranks, p.ranks) and torch.equal(z.logprobs.nan_to_num(7.0), p.logprobs.nan_to_num(7.0))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (3, 2, 2), (5, 7, 3), (4, 63, 20), (2, 64, 64), (3, 65, 64), (7, 1000, 20), (2, 2049, 5),
                                          (64, 8193, 33), (1, 128256, 20), (33, 128256, 1), (5, 32000, 64), (2, 196607, 20)])
def test_logprobs(rows, vocab, k, dtype):
    g = torch.Generator("cuda").manual_seed(vocab + rows)
    x = (torch.randn(rows, vocab, generator=g, device="cuda") * 3).to(DT[dtype])
    tokens = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    tokens[0] = x[0].argmax()
    if rows > 2:
        tokens[1], tokens[2] = -1, vocab + 3
    check_logprobs(x, tokens.tolist(), min(k, vocab))


@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "two values", "masked", "few left", "one left", "none left", "lowest", "highest",
                                  "far apart", "zeros of both signs"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_logprobs_awkward_rows(kind, dtype):
    g = torch.Generator("cuda").manual_seed(1)
    R, V = 6, 20011
    x = torch.randn(R, V, generator=g, device="cuda") * 2
    lo = torch.finfo(DT[dtype])
    ramp = torch.arange(V, device="cuda") / 4000
    if kind == "equal":
        x = torch.full_like(x, 1.25)
    elif kind == "rising":
        x = ramp.expand(R, V).clone()
    elif kind == "falling":
        x = ramp.flip(0).expand(R, V).clone()
    elif kind == "two values":
        x = (x > 3).float()
    elif kind == "masked":
        x[torch.rand(R, V, generator=g, device="cuda") < 0.99] = -math.inf
    elif kind in ("few left", "one left", "none left"):
        keep = x[:, 777:777 + {"few left": 11, "one left": 1, "none left": 0}[kind]].clone()
        x[:] = -math.inf
        x[:, 777:777 + keep.shape[1]] = keep
    elif kind == "lowest":  # a mask of the type's lowest value, one row of nothing else
        x[torch.rand(R, V, generator=g, device="cuda") < 0.9] = lo.min
        x[2] = lo.min
    elif kind == "highest":
        x[:, 5] = lo.max
        x[:, 11] = lo.max
        x[:, 12] = lo.min
    elif kind == "far apart":
        x = x * 1000
    else:
        x = torch.where(x > 0, 0.0, -0.0)
    x = x.to(DT[dtype])
    tokens = [0, V - 1, 777, 5, 12345, 20000]
    check_logprobs(x, tokens, 20)
    check_logprobs(x[:, 1:], [0, 776, V - 2, 4, 1, 2], 64)  # rows that begin off any 16-byte line


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,vocab,k", [(600, 32000, 20), (600, 32000, 33), (90, 20000, 32), (3, 20000, 32)])
def test_logprobs_long_and_short_chunks(rows, vocab, k, dtype):
    """Chunks that stay in registers and chunks that do not; the greatest logits spread out, and all in a few lanes."""
    g = torch.Generator("cuda").manual_seed(3)
    x = torch.randn(rows, vocab, generator=g, device="cuda")
    x[1::2] += 8.0 * (torch.arange(vocab, device="cuda") // 8 % 64 < 19)
    x[2::4] += 8.0 * (torch.arange(vocab, device="cuda") // 4 % 64 == 5)
    check_logprobs(x.to(DT[dtype]), torch.randint(0, vocab, (rows,), generator=g, device="cuda").tolist(), k)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_logprobs_alternatives_among_nan_of_both_signs(dtype):
    from wfamd import ops
    g = torch.Generator("cuda").manual_seed(4)
    for vocab in (50, 700, 20000):
        x = torch.randn(5, vocab, generator=g, device="cuda").to(DT[dtype])
        bits = x.view(torch.int32 if dtype == "f32" else torch.int16)
        bad = torch.rand(5, vocab, generator=g, device="cuda") < 0.5
        neg = torch.rand(5, vocab, generator=g, device="cuda") < 0.5
        nan = torch.full((), math.nan, dtype=DT[dtype], device="cuda").view(bits.dtype)
        bits[bad] = nan & (2 ** (31 if dtype == "f32" else 15) - 1)
        bits[bad & neg] |= -2 ** (31 if dtype == "f32" else 15)
        assert (x.isnan() == bad).all()
        p = ops.token_logprobs(x, top_k=20)
        want = torch.sort(x.float().nan_to_num(-math.inf), dim=1, descending=True, stable=True).indices[:, :20]
        want[torch.arange(20, device="cuda") >= (~bad).sum(1, keepdim=True)] = -1  # fewer than 20 numbers in the row
        assert torch.equal(p.top_ids.long(), want) and p.top_logprobs.isnan().all() and p.entropy.isnan().all()


def test_logprobs_nan_and_infinity():
    from wfamd import ops
    x = torch.randn(4, 5000, device="cuda")
    x[1, 4000] = math.nan
    x[2, 17] = math.inf
    x[3] = math.nan
    x[3, 100] = 2.0
    p = ops.token_logprobs(x, torch.tensor([3, 3, 17, 5], device="cuda"), top_k=8)
    assert torch.isfinite(p.logprobs[0]) and torch.isfinite(p.entropy[0])
    assert p.logprobs[1:].isnan().all() and p.entropy[1:].isnan().all() and p.top_logprobs[1:].isnan().all()
    assert 4000 not in p.top_ids[1].tolist() and p.top_ids[2, 0] == 17 and p.ranks[2] == 1
    assert p.top_ids[3].tolist() == [100] + [-1] * 7
    y = torch.full((2, 700), -math.inf, device="cuda")
    y[1, 3] = math.inf
    p = ops.token_logprobs(y, torch.tensor([699, 3], device="cuda"), top_k=3)
    assert p.logprobs[0] == -math.inf and p.entropy[0] == 0 and p.top_ids[0].tolist() == [0, 1, 2] and p.ranks[0] == 700
    assert (p.top_logprobs[0] == -math.inf).all() and p.top_ids[1].tolist() == [3, 0, 1] and p.logprobs[1].isnan()


def test_logprobs_strides_many_rows_and_refusals():
    from wfamd import ops
    g = torch.Generator("cuda").manual_seed(2)
    whole = torch.randn(300, 1111, generator=g, device="cuda").bfloat16()
    t = torch.randint(0, 900, (300,), generator=g, device="cuda", dtype=torch.int32)
    v = whole[:, 55:955]
    a, b = ops.token_logprobs(v, t, 7), ops.token_logprobs(v.contiguous(), t.long(), 7)
    # the same rows at other alignments: the same ranks and ids; sums in another order, within check_logprobs' units
    assert torch.equal(a.ranks, b.ranks) and torch.equal(a.top_ids, b.top_ids)
    assert (a.logprobs - b.logprobs).abs().max() <= 2 * 2.0 ** -24 * (60 + 3 * 30) and torch.allclose(a.entropy, b.entropy, rtol=2e-5, atol=0)
    lp, rank, ent, ids, top = logprobs_ref(v, t.tolist(), 7)
    assert torch.equal(a.ranks.cpu().long(), rank) and torch.equal(a.top_ids.cpu().long(), ids)
    c = ops.token_logprobs(v[:1].t().contiguous().t(), t[:1], 7)  # one row of any stride
    assert torch.equal(c.top_ids, a.top_ids[:1])
    d = ops.token_logprobs(v[:, :1].expand(300, 5), None, 5)  # logits of stride 0: copied
    assert d.top_ids.tolist() == [[0, 1, 2, 3, 4]] * 300
    e = ops.token_logprobs(v[:0], t[:0], 3)
    assert e.logprobs.shape == (0,) and e.top_ids.shape == (0, 3)
    for args in ((v[0], t[:1], 1), (v, t[:5], 1), (v, t.float(), 1), (v, t, 65), (v, t, -1), (v[:, :4], t, 5), (v.to(torch.float64), t, 1),
                 (v[:, :0], t, 0), (v, t.cpu(), 1), (v, t[:, None], 1)):
        with pytest.raises(ValueError):
            ops.token_logprobs(*args)


def test_serving_ops_in_a_graph_and_on_another_stream():
    """Captured once and replayed with other inputs, the eager call between the replays; two streams at once."""
    from wfamd import ops
    freqs, _ = ops.rotary_frequencies(128, 500000.0)
    x = torch.randn(16, 5000, device="cuda").bfloat16()
    t = torch.zeros(16, dtype=torch.int32, device="cuda")
    q, pos = torch.randn(16, 4, 128, device="cuda").bfloat16(), torch.zeros(16, dtype=torch.int32, device="cuda")
    cached, new = i32(np.zeros(16)), i32(np.ones(16))
    free, table = i32(np.arange(200)), i32(np.zeros((16, 8)))

    def all_three():
        p = ops.kv_page_plan(cached, new, free, table, 40)
        return [*ops.token_logprobs(x, t, 5), ops.rotary_embed(q, None, pos, freqs)[0], *p]
    all_three()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        all_three()
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = all_three()
    for i in range(4):
        x.normal_()
        q.normal_()
        t.fill_(100 * i)
        pos.fill_(1000 * i)
        cached.fill_(31 * i)
        new.fill_(2 - i % 2)
        table.fill_(5)
        g.replay()
        torch.cuda.synchronize()
        held, after = [y.clone() for y in got], table.clone()
        table.fill_(5)
        for a, b in zip(held, all_three()):
            assert torch.equal(a, b)
        assert torch.equal(table, after)
    a, b = torch.randn(40, 9000, device="cuda"), torch.randn(40, 9000, device="cuda")
    want = [ops.token_logprobs(y, None, 9) for y in (a, b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    both = []
    for _ in range(5):
        for st, y in zip(streams, (a, b)):
            with torch.cuda.stream(st):
                both.append(ops.token_logprobs(y, None, 9))
    torch.cuda.synchronize()
    for i, p in enumerate(both):
        assert torch.equal(p.top_ids, want[i % 2].top_ids) and torch.equal(p.top_logprobs, want[i % 2].top_logprobs)


def test_offsets_past_32_bits():
    """Rows 2^30 elements apart: the third begins at element 2^31."""
    from wfamd import ops
    base = torch.empty((1 << 31) + 4096, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator("cuda").manual_seed(6)
    x = base.as_strided((3, 1000), (1 << 30, 1))
    x.copy_(torch.randn(3, 1000, generator=g, device="cuda"))
    a, b = ops.token_logprobs(x, torch.tensor([3, 4, 5], device="cuda"), 20), ops.token_logprobs(x.contiguous(), torch.tensor([3, 4, 5], device="cuda"), 20)
    assert all(torch.equal(u, v) for u, v in zip(a, b))
    q = base.as_strided((3, 4, 64), (1 << 30, 128, 1))
    k = base.as_strided((3, 4, 64), (1 << 30, 128, 1), 64)
    q.copy_(torch.randn(3, 4, 64, generator=g, device="cuda"))
    k.copy_(torch.randn(3, 4, 64, generator=g, device="cuda"))
    pos = torch.tensor([5, 0, 70000], device="cuda")
    freqs, _ = ops.rotary_frequencies(64)
    want = ops.rotary_embed(q.contiguous(), k.contiguous(), pos, freqs)
    got = ops.rotary_embed(q, k, pos, freqs)
    assert all(torch.equal(u, v) for u, v in zip(got, want))
    got = ops.rotary_embed(q, k, pos, freqs, inplace=True)  # heads of q and k in turn
    assert got[0] is q and got[1] is k and torch.equal(q, want[0]) and torch.equal(k, want[1])


def test_rotary_in_place_on_slices_of_one_projection():
    from wfamd import ops
    g = torch.Generator("cuda").manual_seed(7)
    qkv = torch.randn(9, 12, 64, generator=g, device="cuda")
    pos = torch.arange(9, device="cuda", dtype=torch.int32) * 100
    freqs, _ = ops.rotary_frequencies(64)
    before = qkv.clone()
    q, k = ops.rotary_embed(before[:, :8], before[:, 8:10], pos, freqs)
    ops.rotary_embed(qkv[:, :8], qkv[:, 8:10], pos, freqs, inplace=True)
    assert torch.equal(qkv[:, :8], q) and torch.equal(qkv[:, 8:10], k) and torch.equal(qkv[:, 10:], before[:, 10:])
    for bad in (qkv[:, 7:9], qkv[:, :2], qkv[:, 4:8]):
        with pytest.raises(ValueError, match="share memory"):
            ops.rotary_embed(qkv[:, :8], bad, pos, freqs, inplace=True)


def test_two_graphs_of_each_operator_replayed_in_turn():
    """Workspaces and results of two captured calls of one operator stay their own."""
    from wfamd import ops
    g = torch.Generator("cuda").manual_seed(8)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    x = [torch.randn(130, 9000, generator=g, device="cuda").bfloat16() for _ in range(2)]
    lens = [torch.randint(0, 40, (3000,), generator=g, device="cuda", dtype=torch.int32) for _ in range(2)]
    free, tables = torch.arange(9000, device="cuda", dtype=torch.int32), [torch.zeros(3000, 8, dtype=torch.int32, device="cuda") for _ in range(2)]
    q, pos = [torch.randn(50, 4, 64, generator=g, device="cuda") for _ in range(2)], i32(list(range(50)))
    freqs, _ = ops.rotary_frequencies(64)
    calls = [lambda i: ops.token_logprobs(x[i], None, 20), lambda i: ops.kv_page_plan(lens[i], lens[1 - i], free, tables[i], 60000),
             lambda i: (ops.rotary_embed(q[i], None, pos, freqs)[0],)]
    for call in calls:
        want = [[t.clone() for t in call(i) if t is not None] for i in range(2)]
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            call(0)
        s.synchronize()
        graphs = []
        for i in range(2):
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr):
                out = call(i)
            graphs.append((gr, [t for t in out if t is not None]))
        for _ in range(3):
            for gr, _out in graphs:
                gr.replay()
            torch.cuda.synchronize()
            for (_gr, out), w in zip(graphs, want):
                assert all(torch.equal(a.nan_to_num(), b.nan_to_num()) for a, b in zip(out, w))
            call(0)  # the program's own work in between
            torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim,rdim", [(80, 80), (96, 58), (128, 40), (67, 66), (24, 22)])
def test_rotary_off_any_alignment(dim, rdim, dtype):
    """Heads that begin at any element, odd strides: the same bits as from contiguous rows, in place too."""
    from wfamd import ops
    g = torch.Generator("cuda").manual_seed(dim)
    base = torch.randn(40 * (5 * dim + 9) + 8, generator=g, device="cuda").to(DT[dtype])
    pos = torch.randint(0, 5000, (40,), generator=g, device="cuda")
    freqs, _ = ops.rotary_frequencies(rdim)
    for first, th, hh in ((1, 5 * dim + 9, dim + 1), (3, 5 * dim + 1, dim), (0, 5 * dim + 8, dim + 2)):
        for inter in (False, True):
            x = base.clone()
            q, k = x.as_strided((40, 3, dim), (th, hh, 1), first), x.as_strided((40, 1, dim), (th, hh, 1), first + 3 * hh)
            before = x.clone()
            want = ops.rotary_embed(q.contiguous(), k.contiguous(), pos, freqs, interleaved=inter)
            got = ops.rotary_embed(q, k, pos, freqs, interleaved=inter)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(x, before)
            ops.rotary_embed(q, k, pos, freqs, interleaved=inter, inplace=True)
            assert torch.equal(q, want[0]) and torch.equal(k, want[1])
            q.copy_(before.as_strided(q.shape, q.stride(), first))
            k.copy_(before.as_strided(k.shape, k.stride(), first + 3 * hh))
            assert torch.equal(x, before)  # nothing beside the heads was written
