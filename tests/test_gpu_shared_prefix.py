"""shared_prefix_attention on the GPU against the definition in 64 bits, and the serving operators in a row."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
D = 128
O, E = torch.arange(32)[:, None], torch.arange(D)[None]
K_AT = ((((O >> 2) & 1) * 16 + (E >> 3)) * 16 + 4 * (O >> 3) + (O & 3)) * 8 + (E & 7)  # key o, dim e in a K page (wf_bitnet.h)
V_AT = (((E >> 4) * 4 + (O >> 3)) * 16 + (E & 15)) * 8 + (O & 7)


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    from wfamd import _lib
    assert _lib.kernel_available(), "gfx950 kernels must load (no fallback)"
    torch.cuda.set_device(0)


def i32(x):
    return torch.as_tensor(x, dtype=torch.int32, device="cuda")


def widen(x, kv):
    if kv == "int8":
        return x.view(torch.int8).double()
    return x.view(torch.float8_e4m3fn).float().double() if kv == "fp8" else x.double()


def random_pool(pages, hkv, kv, g):
    x = torch.randn(pages, hkv, 32 * D, generator=g, device="cuda")
    if kv == "bf16":
        return x.bfloat16()
    if kv == "int8":
        return (x * 40).round().clamp(-127, 127).to(torch.int8).view(torch.uint8)
    return (x * 2).to(torch.float8_e4m3fn).view(torch.uint8)


def case(b, hkv, gq, lens, rows, plens, kv="bf16", dtype="bf16", seed=0, cols=None, size=1.0):
    """Every table row has pages of its own (a sequence's keys below its prefix stand on the owner's)."""
    g = torch.Generator("cuda").manual_seed(seed)
    cols = cols or -(-max(max(lens), max(plens), 1) // 32)
    n = b * cols + 3
    table = torch.randperm(n, generator=g, device="cuda")[: b * cols].reshape(b, cols).to(torch.int32)
    k, v = random_pool(n, hkv, kv, g), random_pool(n, hkv, kv, g)
    q = (torch.randn(b, hkv * gq, D, generator=g, device="cuda") * size).to(DT[dtype])
    return dict(q=q, k_pool=k, v_pool=v, page_table=table, seq_lens=i32(lens), prefix_rows=i32(rows), prefix_lens=i32(plens), kv_dtype=kv,
                k_scale=0.02 if kv == "int8" else 0.5 if kv == "fp8" else 1.0, v_scale=0.03 if kv == "int8" else 1.0)


def reference(q, k_pool, v_pool, page_table, seq_lens, prefix_rows, prefix_lens, kv_dtype="bf16", k_scale=1.0, v_scale=1.0, sm_scale=None):
    """out, lse, and of each row: sum p |v| / l, the largest |score|, the largest sum of |q k| scale, the keys."""
    b, hq, _ = q.shape
    pages, hkv = k_pool.shape[:2]
    table, cols = page_table.cpu().long(), page_table.shape[1]
    sm = D ** -0.5 if sm_scale is None else sm_scale
    out, mean = torch.zeros(b, hq, D, dtype=torch.float64), torch.zeros(b, hq, D, dtype=torch.float64)
    lse = torch.full((b, hq), -math.inf, dtype=torch.float64)
    top, size, keys = (torch.zeros(b, hq, dtype=torch.float64) for _ in range(3))
    for i in range(b):
        n = min(max(int(seq_lens[i]), 0), 32 * cols)
        r = int(prefix_rows[i])
        p = min(max(int(prefix_lens[i]), 0), n) if 0 <= r < b else 0
        r = r if p else i
        j = torch.arange(n)
        page = torch.cat([table[r][j[:p] // 32], table[i][j[p:] // 32]])
        live = (page >= 0) & (page < pages)
        j, page = j[live], page[live]
        if len(j) == 0:
            continue
        pg, h = page.cuda()[:, None, None], torch.arange(hkv, device="cuda")[None, :, None]
        k, v = (widen(x[pg, h, at[j % 32].cuda()[:, None]], kv_dtype) * s for x, at, s in ((k_pool, K_AT, k_scale), (v_pool, V_AT, v_scale)))
        qq, kk, vv = q[i].double().reshape(hkv, hq // hkv, D), k.permute(1, 2, 0).contiguous(), v.permute(1, 0, 2).contiguous()
        s = torch.matmul(qq, kk) * sm
        m = s.amax(-1, True)
        e = (s - m).exp()
        l = e.sum(-1, True)
        out[i] = (torch.matmul(e, vv) / l).reshape(hq, D).cpu()
        mean[i] = (torch.matmul(e, vv.abs()) / l).reshape(hq, D).cpu()
        lse[i] = (m + l.log()).reshape(hq).cpu()
        top[i] = s.abs().amax(-1).reshape(hq).cpu()
        size[i] = (torch.matmul(qq.abs(), kk.abs()).amax(-1) * abs(sm)).reshape(hq).cpu()
        keys[i] = len(j)
    return out, lse, mean, top, size, keys


def check(c, sm_scale=None):
    from wfamd import ops
    out, lse = ops.shared_prefix_attention(**c, sm_scale=sm_scale, return_lse=True)
    want, wlse, mean, top, size, keys = reference(**c, sm_scale=sm_scale)
    t = c["q"].dtype
    half = t == torch.float16 and c["kv_dtype"] != "bf16"  # f16 products: q as it is, p rounded once to f16
    terms = {torch.bfloat16: 1, torch.float16: 2 - half, torch.float32: 3}[t]
    u = 2.0 ** -24
    # a score: 128 products and sums for each term of q, the scale's 3 roundings, the exponent's and exp2's (64 + 4)
    ds = u * ((128 * terms + 8) * size + 3 * top + 68)
    # p: 2^-8 for each of its bf16 terms, 2^-11 for one of f16 (and 2^-32 of the row's largest where it is below 2^-21 of
    # it, less than its share of the sum's u); twice the score's error; l and o: a sum over the keys, 24 more of the joins
    rel = (2.0 ** -11 if half else 2.0 ** -(8 * terms)) + 2 * ds + u * (keys + 24)
    tol = mean * rel[..., None] + torch.finfo(t).eps / 2 * want.abs() + (2.0 ** -25 if t == torch.float16 else 1e-37)
    assert out.dtype == t and torch.isfinite(out).all()
    assert ((out.double().cpu() - want).abs() / tol).max().item() <= 1.0
    got = lse.double().cpu()
    none = wlse == -math.inf
    assert torch.equal(got == -math.inf, none) and (out.cpu()[none] == 0).all()
    dl = (got - wlse).abs()[~none]
    ltol = (ds + u * (keys + 24 + 4 * wlse.abs()))[~none]
    assert dl.numel() == 0 or (dl / ltol).max().item() <= 1.0
    assert torch.equal(ops.shared_prefix_attention(**c, sm_scale=sm_scale), out)  # the same bits again
    return out, lse


SHAPES = [  # batch, kv heads, query heads a kv head, prefix
    (1, 1, 1, 40), (2, 5, 4, 31), (2, 1, 1, 32), (4, 5, 4, 500), (3, 2, 7, 33), (16, 1, 4, 100), (17, 2, 3, 1000), (5, 1, 20, 64),
    (3, 2, 64, 70), (65, 1, 1, 96), (130, 1, 1, 200), (70, 2, 8, 45), (128, 5, 4, 257), (2, 1, 33, 1)]


@pytest.mark.parametrize("b,hkv,gq,prefix", SHAPES)
@pytest.mark.parametrize("dtype,kv", [("bf16", "bf16"), ("f16", "int8"), ("f32", "fp8")])
def test_one_prefix(b, hkv, gq, prefix, dtype, kv):
    lens = [prefix + 1 + (i * 37) % 150 for i in range(b)]
    check(case(b, hkv, gq, lens, [0] * b, [prefix] * b, kv, dtype, seed=b + prefix))


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("kv", ["bf16", "fp8", "int8"])
def test_types(dtype, kv):
    check(case(9, 2, 4, [300 + 11 * i for i in range(9)], [2] * 9, [290] * 9, kv, dtype, seed=3, size=3.0))


def test_long_prefix_and_suffix_many_ranges():
    check(case(3, 1, 2, [9000, 8003, 20000], [1, 1, 1], [8000] * 3, seed=4))
    check(case(2, 2, 4, [12345, 33], [0, 1], [0, 0], "int8", "f32", seed=5))  # no prefix at all


def test_groups_of_every_kind():
    """Uneven groups, groups of one, owners far off, out of range or absent, neighbours that differ in one of the two."""
    b = 40
    rows = [0] * 7 + [7] + [8] * 17 + [39] * 2 + [-1] * 3 + [40] * 2 + [5, 6, 5, 6] + [35] * 4
    plens = [100] * 7 + [50] + [333] * 17 + [64] * 2 + [10] * 3 + [10] * 2 + [70] * 4 + [32, 32, 96, 96]
    lens = [plens[i] + (i * 29) % 90 for i in range(b)]  # the first of them ends with the prefix
    for gq, dtype in ((4, "bf16"), (1, "f32"), (6, "f16")):
        check(case(b, 2, gq, lens, rows, plens, dtype=dtype, seed=6))


def test_short_empty_and_padded_sequences():
    """Lengths of 0 and 1, shorter than the prefix, longer than the table, negative; rows of nothing behind the last."""
    lens = [0, 1, 31, 32, 33, 64, 100, 100, 200, 200, -7, 10 ** 9, 0, 0, 0]
    c = case(15, 2, 4, [max(x, 0) for x in lens[:10]] + [200] * 5, [3] * 15, [100] * 15, seed=7, cols=7)
    c["seq_lens"] = i32(lens)
    out, lse = check(c)
    assert (out[[0, 10, 12, 13, 14]] == 0).all() and (lse[[0, 10, 12]] == -math.inf).all()
    c["prefix_lens"] = i32([10 ** 9, -5] + [224] * 13)
    check(c)


def test_pages_outside_the_pool_count_as_absent():
    c = case(8, 1, 4, [200] * 8, [0] * 8, [130] * 8, seed=8)
    t = c["page_table"]
    t[0, 2], t[3, 5], t[4, 6], t[5, 4:] = -1, 10 ** 9, c["k_pool"].shape[0], -2 ** 31
    check(c)
    t[0, :] = -1
    t[5, :] = -1
    out, lse = check(c)
    assert (out[0] == 0).all() and (out[5] == 0).all() and (lse[5] == -math.inf).all()


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
def test_what_is_masked_may_hold_anything(kv):
    """NaN behind a sequence's end and on pages' unused places; infinity in keys that only others have."""
    from wfamd import ops
    lens, p = [70, 83, 83, 40, 90], 69
    c = case(5, 2, 3, lens, [1] * 5, [p] * 5, kv, seed=9)
    nan = math.nan if kv == "bf16" else 0x7f
    want = check(c)[0]
    for i, n in enumerate(lens):
        for j in range(32 * c["page_table"].shape[1]):
            if not (p <= j < n or (i == 1 and j < p)):
                page = int(c["page_table"][i, j // 32])
                c["k_pool"][page][:, K_AT[j % 32].cuda()] = nan
                c["v_pool"][page][:, V_AT[j % 32].cuda()] = nan
    assert torch.equal(ops.shared_prefix_attention(**c), want)
    # the shared keys from 40 on: sequence 3 has 40 keys and must not see them
    for j in range(40, 64):
        c["v_pool"][int(c["page_table"][1, 1])][:, V_AT[j % 32].cuda()] = math.inf if kv == "bf16" else 0x7f
    got = ops.shared_prefix_attention(**c)
    assert torch.equal(got[3], want[3]) and not torch.isfinite(got[[0, 1, 2, 4]]).any()


def test_extreme_scores():
    from wfamd import ops
    for size in (0.0, 60.0, 2000.0):
        check(case(6, 1, 4, [150] * 6, [0] * 6, [100] * 6, seed=10, size=size))
        check(case(6, 1, 4, [150] * 6, [0] * 6, [100] * 6, "int8", "f32", seed=10, size=size))
    check(case(6, 1, 4, [150] * 6, [0] * 6, [100] * 6, seed=11), sm_scale=-0.3)
    c = case(6, 1, 4, [150] * 6, [0] * 6, [100] * 6, seed=12)
    c["k_pool"].fill_(-math.inf)
    c["q"].abs_().add_(0.1)
    out, lse = ops.shared_prefix_attention(**c, return_lse=True)  # every score -inf
    assert (out == 0).all() and (lse == -math.inf).all()
    c["q"].fill_(math.nan)
    out, lse = ops.shared_prefix_attention(**c, return_lse=True)
    assert out.isnan().all() and lse.isnan().all()


@pytest.mark.parametrize("kv", ["fp8", "int8"])
def test_f16_over_one_byte_pools(kv):
    """f16 products: flat and steep rows, a rising score, every code, what is masked."""
    from wfamd import ops
    shape = (6, 1, 4, [150, 150, 97, 150, 0, 101], [0] * 6, [100] * 6, kv, "f16")
    for size in (0.0, 1.0, 30.0, 300.0):
        check(case(*shape, seed=20, size=size))
    check(case(*shape, seed=21), sm_scale=-0.3)
    # scores that rise by a little with every tile: the frame is raised time and again, or (0.02) not at all
    for step in (0.02, 1.5):
        c = case(40, 1, 2, [640] * 40, [0] * 40, [600] * 40, kv, "f16", seed=22)
        c["q"].zero_()
        c["q"][..., 0] = step / c["k_scale"] * D ** 0.5
        for j in range(20):
            level = torch.tensor([float(j)], device="cuda")
            code = level.to(torch.float8_e4m3fn).view(torch.uint8).item() if kv == "fp8" else j
            for b in (range(40) if j > 17 else (0,)):
                c["k_pool"][int(c["page_table"][b, j])] = code
        check(c)
    # a sequence of one key gives its values: all codes that are numbers
    codes = torch.arange(256, device="cuda").to(torch.uint8)
    if kv == "fp8":
        codes = torch.where(codes & 0x7f == 0x7f, 0, codes).to(torch.uint8)
    c = case(2, 1, 1, [1, 1], [-1, -1], [0, 0], kv, "f16", seed=23)
    for i in range(2):
        c["v_pool"][int(c["page_table"][i, 0])][0, V_AT[0].cuda()] = codes[128 * i:128 * i + 128]
    c["v_scale"] = 1.0
    assert torch.equal(ops.shared_prefix_attention(**c).reshape(-1), widen(codes, kv).half())


def test_strides_layers_and_offsets_past_32_bits():
    from wfamd import ops
    c = case(12, 2, 4, [100 + i for i in range(12)], [0] * 12, [90] * 12, seed=13)
    want, cols, n = check(c)[0], c["page_table"].shape[1], c["k_pool"].shape[0]
    qkv = torch.randn(12, 16, D, device="cuda").bfloat16()
    qkv[:, 3:11] = c["q"]
    layers = [torch.randn(3, n, 5, 32 * D, device="cuda").bfloat16() for _ in range(2)]
    for x, y in zip(layers, ("k_pool", "v_pool")):
        x[1, :, 2:4] = c[y]
    wide = torch.full((20, cols + 5), -1, dtype=torch.int32, device="cuda")
    wide[4:16, 2:2 + cols] = c["page_table"]
    d = dict(c, q=qkv[:, 3:11], k_pool=layers[0][1][:, 2:4], v_pool=layers[1][1][:, 2:4], page_table=wide[4:16, 2:2 + cols])
    assert torch.equal(ops.shared_prefix_attention(**d), want)
    for dims in ((0, 1), (1, 2)):  # heads outermost; dims apart (copied)
        assert torch.equal(ops.shared_prefix_attention(**dict(c, q=c["q"].transpose(*dims).contiguous().transpose(*dims))), want)
    # more than 2^31 elements in front of the pages
    shift = (1 << 31) // (2 * 32 * D) + 5
    far = [torch.empty(shift + n, 2, 32 * D, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    for x, y in zip(far, ("k_pool", "v_pool")):
        x[shift:] = c[y]
    d = dict(c, k_pool=far[0], v_pool=far[1], page_table=c["page_table"] + shift)
    assert torch.equal(ops.shared_prefix_attention(**d), want)


def test_refusals():
    from wfamd import ops
    c = case(4, 2, 2, [40] * 4, [0] * 4, [33] * 4, seed=14)
    k, v, t, q = c["k_pool"], c["v_pool"], c["page_table"], c["q"]
    bad = [dict(q=q[0]), dict(q=q[:, :3]), dict(q=q[..., :64]), dict(q=q.double()), dict(q=q.cpu()), dict(k_pool=k.half()), dict(k_pool=k[:-1]),
           dict(k_pool=k[..., :-8], v_pool=v[..., :-8]), dict(kv_dtype="int8"), dict(kv_dtype="x"), dict(page_table=t.long()),
           dict(page_table=t[:3]), dict(page_table=t[:, :0]), dict(page_table=t.t().contiguous().t()), dict(seq_lens=c["seq_lens"].long()),
           dict(prefix_rows=c["prefix_rows"][:3]), dict(prefix_lens=c["prefix_lens"][:, None]), dict(k_scale=0.0),
           dict(sm_scale=math.inf), dict(k_pool=k.transpose(0, 1).contiguous().transpose(0, 1))]
    for kw in bad:
        with pytest.raises(ValueError):
            ops.shared_prefix_attention(**{**c, **kw})
    e = ops.shared_prefix_attention(**{**c, **{n: c[n][:0] for n in ("q", "page_table", "seq_lens", "prefix_rows", "prefix_lens")}}, return_lse=True)
    assert e[0].shape == (0, 4, D) and e[1].shape == (0, 4)


def test_graph_replays_and_two_streams():
    from wfamd import ops
    c = case(20, 2, 4, [300] * 20, [0] * 20, [200] * 20, seed=15)
    d = case(20, 2, 4, [900 - i for i in range(20)], [3] * 20, [500] * 20, seed=16)
    want = [ops.shared_prefix_attention(**x) for x in (c, d)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for _ in range(5):
        for st, x in zip(streams, (c, d)):
            with torch.cuda.stream(st):
                got.append(ops.shared_prefix_attention(**x))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i % 2]) for i, y in enumerate(got))
    graphs = []
    for x in (c, d):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            ops.shared_prefix_attention(**x)
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = ops.shared_prefix_attention(**x, return_lse=True)
        graphs.append((g, out, x))
    for i in range(4):
        for g, out, x in graphs:
            x["q"].normal_()
            x["seq_lens"].fill_(50 + 75 * i)
            x["prefix_lens"].fill_(200 - 60 * i)
            x["prefix_rows"].fill_(i)
            g.replay()
            torch.cuda.synchronize()
            a, b = ops.shared_prefix_attention(**x, return_lse=True)
            assert torch.equal(out[0], a) and torch.equal(out[1], b)


def test_a_decode_step_from_lengths_to_log_probabilities():
    """Plan the slots, rotate, write the pages, attend over the shared prompt, score: against the same in 64 bits."""
    from sgl_kernel.kvcache import KVCacheManager
    from wfamd import ops
    from wfamd.model import BitNetConfig, BitNetDecoder, synthetic_weights
    b, hq, hkv, prompt = 16, 4, 2, 77
    cfg = BitNetConfig(hidden=512, layers=2, n_heads=hq, n_kv_heads=hkv, head_dim=D, inter=768, vocab=1024, max_seq=256)
    dec = BitNetDecoder(cfg, synthetic_weights(cfg), batch=b, num_pages=128)
    mgr = KVCacheManager.from_decoder(dec)
    freqs, scale = ops.rotary_frequencies(D, 500000.0)
    free = mgr.allocate_pages(100).cuda()
    used = 0
    kept = [[[] for _ in range(b)] for _ in range(2)]  # the k and v rows written so far, by sequence
    whole = prompt // 32 * 32
    cached = [0] * b

    def append(new):
        nonlocal used, cached
        n = sum(new)
        p = ops.kv_page_plan(i32(cached), i32(new), free[used:], dec.page_table, n)
        used += int(p.counts[2])
        qkv = torch.randn(n, hq + 2 * hkv, D, device="cuda").bfloat16()
        q, k = ops.rotary_embed(qkv[:, :hq], qkv[:, hq:hq + hkv], p.positions, freqs, scale=scale)
        v = qkv[:, hq + hkv:]
        mgr.scatter_kv(k.reshape(n, -1), v.reshape(n, -1).contiguous(), p.pages, p.slots, 1)
        for t, r in enumerate(p.rows.tolist()):
            kept[0][r].append(k[t])
            kept[1][r].append(v[t])
        cached = [c + m for c, m in zip(cached, new)]
        return q, p
    append([prompt] + [0] * (b - 1))  # the system prompt, in sequence 0
    dec.page_table[1:, :whole // 32] = dec.page_table[0, :whole // 32]  # the others begin with its whole pages
    for r in range(1, b):
        cached[r] = whole
        for x in kept:
            x[r] = x[0][:whole]
    append([0] + [1 + 5 * i for i in range(b - 1)])
    q, p = append([1] * b)
    out = ops.shared_prefix_attention(q, dec.k_cache[1], dec.v_cache[1], dec.page_table, i32(cached), i32([0] * b), i32([whole] * b))
    assert mgr.invalid_page_count() == 0 and p.positions.tolist() == [c - 1 for c in cached]
    for r in range(b):
        k, v = (torch.stack(x[r]).double() for x in kept)
        assert len(k) == cached[r]
        s = (q[r].double().reshape(hkv, -1, 1, D) * k.permute(1, 0, 2)[:, None]).sum(-1) / math.sqrt(D)
        w = s.softmax(-1)
        y = (w[..., None] * v.permute(1, 0, 2)[:, None]).sum(2).reshape(hq, D)
        mean = (w[..., None] * v.abs().permute(1, 0, 2)[:, None]).sum(2).reshape(hq, D)
        # P's rounding, the output's, and 2^-12 for the rest (scores of a few units in 32 bits)
        assert ((out[r].double() - y).abs() <= mean * (2.0 ** -8 + 2.0 ** -12) + y.abs() * 2.0 ** -8).all()
    logits = out.reshape(b, -1) @ dec.embed[:, :512].t().contiguous()
    lp = ops.token_logprobs(logits, logits.argmax(1), top_k=3)
    ref = logits.double().log_softmax(1)
    assert (lp.top_logprobs[:, 0].double() - ref.amax(1)).abs().max().item() <= 2.0 ** -24 * 300  # 300 roundings: 16 terms a lane, |log p| < 20
    best = lp.ranks == 1
    assert best.any() and torch.equal(lp.logprobs[best], lp.top_logprobs[:, 0][best])


@pytest.mark.parametrize("kv", ["bf16", "int8", "fp8"])
def test_decoder_reserves_a_batch_and_attends_over_its_pool(kv):
    """BitNetDecoder.reserve_batch gives the pages that reserve gives one sequence after the other; its
    shared_prefix_attention reads what a step's cache holds; token_logprobs is over the step's logits."""
    from wfamd import ops
    from wfamd.model import BitNetConfig, BitNetDecoder, synthetic_weights
    cfg = BitNetConfig(hidden=512, layers=2, n_heads=4, n_kv_heads=2, head_dim=D, inter=768, vocab=1024, max_seq=256)
    w = synthetic_weights(cfg)
    a, b = (BitNetDecoder(cfg, w, batch=16, num_pages=96, page_seed=5, kv_dtype=kv, kv_scale=(0.05, 0.03) if kv != "bf16" else None)
            for _ in range(2))
    rng = torch.Generator().manual_seed(1)
    for counts in (torch.randint(0, 70, (16,), generator=rng).tolist(), [0] * 16, torch.randint(40, 160, (16,), generator=rng).tolist()):
        a.reserve_batch(counts)
        for i, n in enumerate(counts):
            b.reserve(i, n)
        assert torch.equal(a.page_table, b.page_table) and all((x == y).all() for x, y in zip(a.seq_pages, b.seq_pages))
    free = a.pool.num_free_pages()
    with pytest.raises(RuntimeError):
        a.reserve_batch([256] * 16)
    assert a.pool.num_free_pages() == free
    for bad in ([1] * 15, [257] + [1] * 15, [-1] + [1] * 15):
        with pytest.raises(ValueError):
            a.reserve_batch(bad)
    pos = [len(p) * 32 - 1 for p in a.seq_pages]
    k = torch.randn(16, 2, 160, D, generator=torch.Generator("cuda").manual_seed(2), device="cuda").bfloat16()
    for layer in range(2):
        a.load_kv(layer, k, -k, lengths=pos)
    a.set_state(list(range(16)), [p - 1 for p in pos])
    a.step(graph=False)
    a.check()
    p = a.token_logprobs(a.tokens, top_k=2)
    assert (p.ranks == 1).all() and torch.equal(p.top_ids[:, 0], a.tokens)
    ref = a.logits.double().log_softmax(1)
    assert (p.logprobs.double() - ref.gather(1, a.tokens.long()[:, None])[:, 0]).abs().max().item() <= 2.0 ** -24 * 300
    # the last layer's attention of the step, from the pool by this operator: within the two kernels' roundings of P and of the output
    q = a.attention_records()[0]
    got, want = a.shared_prefix_attention(1, q, i32(pos), i32([-1] * 16), i32([0] * 16)), a.attention_row()
    assert (got.double() - want.double()).abs().max().item() <= 6 * 2.0 ** -8 * want.double().abs().max().item()
    c = dict(q=q, k_pool=a.k_cache[1], v_pool=a.v_cache[1], page_table=a.page_table, seq_lens=i32(pos), prefix_rows=i32([0] * 16),
             prefix_lens=i32([60] * 16), kv_dtype=kv, k_scale=0.05 if kv != "bf16" else 1.0, v_scale=0.03 if kv != "bf16" else 1.0)
    assert torch.equal(a.shared_prefix_attention(1, q, c["seq_lens"], c["prefix_rows"], c["prefix_lens"]), check(c)[0])


@pytest.mark.parametrize("dtype,kv", [("bf16", "bf16"), ("f16", "bf16"), ("f16", "fp8"), ("f32", "int8")])
@pytest.mark.parametrize("hkv,gq,sizes", [(1, 1, [7, 1, 9, 8, 5]), (4, 4, [3, 2, 2, 1, 2, 4, 2, 3]), (1, 3, [2] * 20), (5, 4, [40, 17, 100]), (2, 1, [33] * 6)])
def test_runs_of_every_size(hkv, gq, sizes, dtype, kv):
    """Groups of all sizes next to each other, more of them than a row tile's workgroups, prefixes of several ranges."""
    b = sum(sizes)
    rows, plens, lens = [], [], []
    for i, n in enumerate(sizes):
        first = len(rows)
        p = 40 + 67 * (i % 5) + 300 * (i % 2)
        rows += [first] * n
        plens += [p] * n
        lens += [p + (11 * j + 5 * i) % 70 for j in range(n)]
    check(case(b, hkv, gq, lens, rows, plens, kv, dtype, seed=30 + b))
