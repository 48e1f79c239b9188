"""The serving operators around the paged decode path, as cases that can be timed and checked: page plans,
rotary positions, attention over a shared prefix, token log probabilities.

`run` computes a case in its plain form (elementary torch operations in 32 bits, 64 for angles), or, where `own`
is true, through this repository's operators; `exact` computes it in 64 bits from the definition."""
import functools
import math
import os
import sys

import torch

own = False

DEV = "cuda"
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
PAGE, DIM = 32, 128  # the paged pool's tokens per page and head size


@functools.lru_cache(maxsize=None)
def _ops():
    """This repository's operators, from its package folder as the benchmark finds it."""
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "wrinklefree-inference-engine_amd", "python")
    if at not in sys.path:
        sys.path.insert(0, at)
    from wfamd import ops
    return ops


def listed():
    return [
        # one decode step of a full batch: every request gets one token, few need a page
        {"name": "plan decode b128", "op": "plan", "batch": 128, "new": 1, "ctx": 4095, "page": 32, "spare": 0, "tight": False},
        # many ragged prompts admitted at once, among requests that go on
        {"name": "plan prompts b1024", "op": "plan", "batch": 1024, "new": 1500, "ctx": 2000, "page": 32, "spare": 0, "tight": False},
        # q and k of one decode step
        {"name": "rotary decode b128", "op": "rotary", "tokens": 128, "hq": 20, "hk": 5, "dim": 128, "rdim": 128, "dtype": "bf16",
         "interleaved": False, "scaling": "none", "maxpos": 4096},
        # prompts of 8 x 2048 tokens at far positions of a context that was extended
        {"name": "rotary prompts extended", "op": "rotary", "tokens": 16384, "hq": 20, "hk": 5, "dim": 128, "rdim": 128, "dtype": "bf16",
         "interleaved": False, "scaling": "yarn", "maxpos": 131072},
        # part of the head, neighbouring pairs, an odd number of rows, 32 bits
        {"name": "rotary partial interleaved", "op": "rotary", "tokens": 4097, "hq": 8, "hk": 2, "dim": 96, "rdim": 64, "dtype": "f32",
         "interleaved": True, "scaling": "linear", "maxpos": 32768},
        # a few requests behind one short system prompt: latency
        {"name": "attend b4 prefix 500", "op": "attend", "batch": 4, "groups": 1, "hq": 20, "hkv": 5, "prefix": 500, "suffix": 64,
         "dtype": "bf16", "kv": "bf16", "pad": 0},
        # the batch of the decode benchmark behind one system prompt
        {"name": "attend b128 prefix 1024", "op": "attend", "batch": 128, "groups": 1, "hq": 20, "hkv": 5, "prefix": 1024, "suffix": 512,
         "dtype": "bf16", "kv": "bf16", "pad": 0},
        # several tenants, each with a prompt of its own; int8 pages, a padded batch
        {"name": "attend b96 groups int8", "op": "attend", "batch": 96, "groups": 6, "hq": 32, "hkv": 4, "prefix": 2011, "suffix": 700,
         "dtype": "f16", "kv": "int8", "pad": 3},
        # many questions about one long document
        {"name": "attend b128 prefix 32768", "op": "attend", "batch": 128, "groups": 1, "hq": 20, "hkv": 5, "prefix": 32768, "suffix": 1024,
         "dtype": "bf16", "kv": "bf16", "pad": 0},
        # the logits of one request
        {"name": "logprobs b1", "op": "logprobs", "rows": 1, "vocab": 128256, "dtype": "bf16", "top": 20, "masked": 0.0},
        # the logits of a decode step, part of the vocabulary barred by a grammar
        {"name": "logprobs b128 masked", "op": "logprobs", "rows": 128, "vocab": 128256, "dtype": "bf16", "top": 20, "masked": 0.5},
        # scoring a prompt: every position's token
        {"name": "logprobs prompt 2048", "op": "logprobs", "rows": 2048, "vocab": 128256, "dtype": "bf16", "top": 5, "masked": 0.0},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "rotary", "attend", "logprobs"])
    if op == "plan":
        return {"op": op, "batch": _log(rng, 1, 1024), "new": _log(rng, 1, 1500), "ctx": _log(rng, 1, 8000),
                "page": rng.choice([16, 32, 64]), "spare": rng.choice([0, 0, 9]), "tight": rng.random() < 0.3}
    if op == "rotary":
        dim = rng.choice([64, 80, 96, 128])
        rdim = rng.choice([dim, dim // 2, 2 * rng.randint(1, dim // 2)])
        hk = _log(rng, 1, 8)
        return {"op": op, "tokens": _log(rng, 1, 16384), "hq": hk * rng.randint(1, 3), "hk": hk, "dim": dim, "rdim": rdim,
                "dtype": rng.choice(["bf16", "f16", "f32"]), "interleaved": rng.random() < 0.5,
                "scaling": rng.choice(["none", "linear", "ntk", "yarn"]), "maxpos": _log(rng, 16, 1 << 20)}
    if op == "attend":
        hkv = _log(rng, 1, 8)
        batch = _log(rng, 1, 128)
        return {"op": op, "batch": batch, "groups": min(batch, _log(rng, 1, 16)), "hq": hkv * rng.choice([1, 2, 3, 4, 7, 8]), "hkv": hkv,
                "prefix": _log(rng, 1, 4096), "suffix": _log(rng, 1, 1024), "dtype": rng.choice(["bf16", "bf16", "f16", "f32"]),
                "kv": rng.choice(["bf16", "bf16", "int8", "fp8"]), "pad": rng.choice([0, 0, 1, 5])}
    return {"op": op, "rows": _log(rng, 1, 1024), "vocab": _log(rng, 100, 160000), "dtype": rng.choice(["bf16", "f16", "f32"]),
            "top": rng.choice([0, 1, 5, 20, 64]), "masked": rng.choice([0.0, 0.0, 0.9])}


def _gen(seed, salt):
    return torch.Generator(device=DEV).manual_seed(seed * 16 + salt)


def _ints(lo, hi, n, g):
    return torch.randint(lo, hi + 1, (n,), generator=g, device=DEV, dtype=torch.int32)


# ---- block tables and slot maps ---------------------------------------------------------------
def _prepare_plan(c, seed):
    g = _gen(seed, 0)
    b, page = c["batch"], c["page"]
    # lengths from 1 to `new` with one sum, whatever the seed: the token arrays are sized by the host
    new = (1 + torch.arange(b, device=DEV) * (c["new"] - 1) // max(b - 1, 1)).to(torch.int32)[torch.randperm(b, generator=g, device=DEV)]
    cached = _ints(0, c["ctx"], b, g)
    cached[torch.rand(b, generator=g, device=DEV) < (0.5 if c["new"] > 1 else 0.02)] = 0  # newly admitted requests
    cols = -(-(c["ctx"] + c["new"]) // page)
    have = (cached + page - 1) // page
    need = (cached + new + page - 1) // page - have
    tokens, pages, held = int(new.sum()), int(need.sum()), int(have.sum())
    ids = torch.randperm(held + pages + 64, generator=g, device=DEV).to(torch.int32)
    table = torch.zeros(b, cols, dtype=torch.int32, device=DEV)
    at = torch.arange(cols, device=DEV)[None] < have[:, None]
    table[at] = ids[:held]
    free = ids[held:]
    if c["tight"]:  # the pool runs out on the way
        free = free[: max(1, (2 * pages) // 3)].contiguous()
    return {"cached": cached, "new": new, "free": free, "table": table, "tokens": tokens + c["spare"], "page": page}


def _run_plan(s):
    if own:
        ops = _ops()
        p = ops.kv_page_plan(s["cached"], s["new"], s["free"], s["table"], s["tokens"], page_size=s["page"])
        return {"pages": p.pages, "slots": p.slots, "rows": p.rows, "positions": p.positions, "cu_tokens": p.cu_tokens,
                "counts": p.counts, "table": s["table"]}
    page, table, free = s["page"], s["table"], s["free"]
    cols = table.shape[1]
    cached, new = s["cached"].long(), s["new"].long()
    have = (cached + page - 1) // page
    blocks = (cached + new + page - 1) // page
    long = blocks > cols
    need = torch.where(long, torch.zeros_like(have), blocks - have)
    ends = need.cumsum(0)
    off = ends - need
    fit = ~long & ((need == 0) | (ends <= free.numel()))
    at = torch.arange(cols, device=DEV)[None]
    fresh = (at >= have[:, None]) & (at < blocks[:, None]) & fit[:, None]
    src = (off[:, None] + at - have[:, None]).clamp(0, free.numel() - 1)
    table.copy_(torch.where(fresh, free[src], table))
    cu = torch.cat([new.new_zeros(1), new.cumsum(0)])
    t = torch.arange(s["tokens"], device=DEV)
    live = t < cu[-1]
    rows = torch.searchsorted(cu, t, right=True).clamp(max=new.numel()) - 1
    pos = cached[rows] + t - cu[rows]
    ok = fit[rows] & live
    pages = torch.where(ok, table[rows, (pos // page).clamp(max=cols - 1)], -1)
    slots = torch.where(ok, pos % page, -1)
    rows, pos = torch.where(live, rows, -1), torch.where(live, pos, -1)
    taken = torch.where(fit & (need > 0), ends, torch.zeros_like(ends)).max()
    counts = torch.stack([cu[-1], ends[-1], taken, (~fit).sum()])
    i32 = lambda x: x.to(torch.int32)  # noqa: E731
    return {"pages": i32(pages), "slots": i32(slots), "rows": i32(rows), "positions": i32(pos), "cu_tokens": i32(cu),
            "counts": i32(counts), "table": table}


def _work_plan(c):
    tokens = sum(1 + i * (c["new"] - 1) // max(c["batch"] - 1, 1) for i in range(c["batch"]))
    pages = tokens // c["page"]
    return {"bytes": 12 * c["batch"] + 16 * tokens + 8 * pages + 4 * c["batch"], "flops": 4 * tokens}


# ---- rotary positions --------------------------------------------------------------------------
def _frequencies(c):
    """Radians a position of each pair, in 64 bits, and the factor on the rotated values."""
    r, base, factor, orig = c["rdim"], 500000.0, 8.0, 16384
    if c["scaling"] == "ntk" and r > 2:
        base *= factor ** (r / (r - 2))
    f = base ** (-torch.arange(0, r, 2, dtype=torch.float64) / r)
    scale = 1.0
    if c["scaling"] == "linear":
        f = f / factor
    if c["scaling"] == "yarn":
        dim_at = lambda turns: r * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        lo, hi = max(math.floor(dim_at(32.0)), 0), min(math.ceil(dim_at(1.0)), r - 1)
        ramp = ((torch.arange(r // 2, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        f = f / factor * ramp + f * (1 - ramp)
        scale = 0.1 * math.log(factor) + 1.0
    return f, scale


def _prepare_rotary(c, seed):
    g = _gen(seed, 1)
    n, dt = c["tokens"], DT[c["dtype"]]
    f, scale = _frequencies(c)
    # q and k as the projections leave them: column ranges of one row of q|k|v
    qkv = torch.randn(n, c["hq"] + 2 * c["hk"], c["dim"], generator=g, device=DEV).to(dt)
    pos = torch.randint(0, c["maxpos"], (n,), generator=g, device=DEV)
    return {"q": qkv[:, : c["hq"]], "k": qkv[:, c["hq"]: c["hq"] + c["hk"]], "pos": pos, "freqs": f.to(DEV), "scale": scale,
            "interleaved": c["interleaved"]}


def _turn(x, cos, sin, interleaved):
    r = 2 * cos.shape[1]
    y = x.float()
    a, b = (y[..., 0:r:2], y[..., 1:r:2]) if interleaved else (y[..., : r // 2], y[..., r // 2: r])
    cos, sin = cos[:, None], sin[:, None]
    u, v = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([u, v], -1).flatten(-2) if interleaved else torch.cat([u, v], -1)
    return torch.cat([turned, y[..., r:]], -1).to(x.dtype)


def _run_rotary(s):
    if own:
        ops = _ops()
        q, k = ops.rotary_embed(s["q"], s["k"], s["pos"], s["freqs"], interleaved=s["interleaved"], scale=s["scale"])
        return {"q": q, "k": k}
    a = s["pos"].double()[:, None] * s["freqs"]
    cos, sin = (a.cos() * s["scale"]).float(), (a.sin() * s["scale"]).float()
    return {"q": _turn(s["q"], cos, sin, s["interleaved"]), "k": _turn(s["k"], cos, sin, s["interleaved"])}


def _exact_rotary(c, seed):
    s = _prepare_rotary(c, seed)
    f, scale = _frequencies(c)
    r = c["rdim"]
    z = torch.polar(torch.full((1, 1), scale, dtype=torch.float64, device=DEV).expand(c["tokens"], r // 2).contiguous(),
                    torch.outer(s["pos"].double(), f.to(DEV)))[:, None]
    out = {}
    for name in ("q", "k"):
        x = s[name].double()
        i = torch.arange(0, r, 2, device=DEV) if c["interleaved"] else torch.arange(r // 2, device=DEV)
        j = i + 1 if c["interleaved"] else i + r // 2
        w = torch.complex(x[..., i], x[..., j]) * z
        x[..., i], x[..., j] = w.real, w.imag
        out[name] = x
    return out


def _work_rotary(c):
    n = c["tokens"] * (c["hq"] + c["hk"]) * c["dim"]
    return {"bytes": 2 * n * (4 if c["dtype"] == "f32" else 2) + 8 * c["tokens"] + 4 * c["rdim"],
            "flops": 3 * c["tokens"] * (c["hq"] + c["hk"]) * c["rdim"]}


# ---- attention of one token a sequence over pages whose first part a group shares --------------
def _prepare_attend(c, seed):
    g = _gen(seed, 2)
    b, ng, prefix = c["batch"], c["groups"], c["prefix"]
    # groups of uneven size, next to each other in the batch; prefixes of uneven length
    cut = (torch.arange(1, ng) * b // ng + torch.randint(-(b // ng) // 3, b // ng // 3 + 1, (ng - 1,), generator=torch.Generator().manual_seed(seed))).clamp(1, b - 1)
    starts = [0] + sorted(set(cut.tolist())) + [b]
    ng = len(starts) - 1
    group = torch.repeat_interleave(torch.arange(ng), torch.tensor([y - x for x, y in zip(starts, starts[1:])])).to(DEV)
    first = torch.tensor(starts[:-1], device=DEV)
    plen = torch.full((ng,), prefix, dtype=torch.int32, device=DEV)
    if ng > 1:
        plen = _ints(max(1, prefix // 2), prefix, ng, g)
    lens = plen[group] + _ints(1, c["suffix"], b, g)
    pad = min(c["pad"], b - 1)
    if pad:  # rows of the batch that hold no request
        lens[b - pad:] = 0
    cols = -(-(prefix + c["suffix"]) // PAGE)
    blocks = -(-lens.long() // PAGE)
    shared = (plen // PAGE).long()[group]  # whole pages of the prefix
    at = torch.arange(cols, device=DEV)[None]
    leads = torch.arange(b, device=DEV) == first[group]
    mine = (at < blocks[:, None]) & ((at >= shared[:, None]) | leads[:, None])
    n = int(mine.sum()) + 8
    table = torch.zeros(b, cols, dtype=torch.int32, device=DEV)
    table[mine] = torch.randperm(n, generator=g, device=DEV)[: n - 8].to(torch.int32)
    table = torch.where((at < shared[:, None]) & (at < blocks[:, None]), table[first[group]], table)
    shape = (n, c["hkv"], PAGE * DIM)
    scales = (1.0, 1.0)
    if c["kv"] == "bf16":
        k, v = (torch.empty(shape, dtype=torch.bfloat16, device=DEV).normal_(generator=g) for _ in range(2))
    elif c["kv"] == "int8":
        scales = (0.023, 0.019)
        k, v = (torch.empty(shape, device=DEV).normal_(generator=g).mul_(40).round_().clamp_(-127, 127).to(torch.int8).view(torch.uint8)
                for _ in range(2))
    else:
        scales = (0.5, 0.25)
        k, v = (torch.empty(shape, device=DEV).normal_(generator=g).mul_(2).to(torch.float8_e4m3fn).view(torch.uint8) for _ in range(2))
    q = (torch.randn(b, c["hq"], DIM, generator=g, device=DEV) * 1.5).to(DT[c["dtype"]])
    rank = torch.arange(b, device=DEV) - first[group]
    most = max(y - x for x, y in zip(starts, starts[1:]))
    return {"q": q, "k": k, "v": v, "table": table, "lens": lens, "kv": c["kv"], "scales": scales,
            "rows": first[group].to(torch.int32), "plens": plen[group], "group": group, "rank": rank, "first": first, "gplen": plen.long(),
            "most": most, "hkv": c["hkv"], "prefix": prefix, "suffix": c["suffix"]}


def _values(x, kv, scale):
    if kv == "int8":
        return x.view(torch.int8).float() * scale
    return x.view(torch.float8_e4m3fn).float() * scale if kv == "fp8" else x.float()


def _keys(pool, ids, kv, scale):
    """Pages [n, blocks] of a K pool -> [n, heads, keys, 128]: a page is [2 t][16 d][4 a][4 r][8 e], key 8a + 4t + r, dim 8d + e."""
    n, blocks = ids.shape
    x = _values(pool[ids.reshape(-1).long()], kv, scale).reshape(n, blocks, -1, 2, 16, 4, 4, 8)
    return x.permute(0, 2, 1, 5, 3, 6, 4, 7).reshape(n, -1, blocks * PAGE, DIM)


def _vals(pool, ids, kv, scale):
    """The same of a V pool: a page is [8 n][4 q][16 l][8 e], key 8q + e, dim 16n + l."""
    n, blocks = ids.shape
    x = _values(pool[ids.reshape(-1).long()], kv, scale).reshape(n, blocks, -1, 8, 4, 16, 8)
    return x.permute(0, 2, 1, 4, 6, 3, 5).reshape(n, -1, blocks * PAGE, DIM)


def _run_attend(s):
    if own:
        ops = _ops()
        out, lse = ops.shared_prefix_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], s["rows"], s["plens"], kv_dtype=s["kv"],
                                               k_scale=s["scales"][0], v_scale=s["scales"][1], return_lse=True)
        return {"out": out, "lse": lse}
    b, hq, d = s["q"].shape
    hkv, (ks, vs), cols = s["hkv"], s["scales"], s["table"].shape[1]
    gq, ng = hq // hkv, s["first"].numel()
    lens, plens = s["lens"].long(), s["plens"].long()
    q = s["q"].float().reshape(b, hkv, gq, d) / math.sqrt(d)
    low = float("-inf")
    # the prefix once a group: its queries side by side
    np_ = -(-s["prefix"] // PAGE)
    ids = s["table"][s["first"], :np_]
    kp, vp = _keys(s["k"], ids, s["kv"], ks), _vals(s["v"], ids, s["kv"], vs)
    qg = q.new_zeros(ng, s["most"], hkv, gq, d)
    qg[s["group"], s["rank"]] = q
    qg = qg.transpose(1, 2).reshape(ng, hkv, s["most"] * gq, d)
    sp = (qg @ kp.transpose(-1, -2).contiguous()).reshape(ng, hkv, s["most"], gq, -1).transpose(1, 2)[s["group"], s["rank"]]
    at = torch.arange(np_ * PAGE, device=DEV)[None]
    sp = sp.masked_fill((at >= torch.minimum(plens, lens)[:, None])[:, None, None], low)
    # the rest a sequence
    ns = (s["suffix"] + PAGE - 1) // PAGE + 1
    blk = (plens // PAGE)[:, None] + torch.arange(ns, device=DEV)
    ids = s["table"].gather(1, blk.clamp(max=cols - 1))
    at = (blk[..., None] * PAGE + torch.arange(PAGE, device=DEV)).reshape(b, -1)
    dead = (at < plens[:, None]) | (at >= lens[:, None])
    vz = _vals(s["v"], ids, s["kv"], vs).masked_fill(dead[:, None, :, None], 0.0)
    ss = (q @ _keys(s["k"], ids, s["kv"], ks).transpose(-1, -2).contiguous()).masked_fill(dead[:, None, None], low)
    m = torch.maximum(sp.amax(-1, True), ss.amax(-1, True))
    z = m.masked_fill(m == low, 0.0)
    ep, es = (sp - z).exp(), (ss - z).exp()
    l = ep.sum(-1, True) + es.sum(-1, True)
    eg = ep.new_zeros(ng, s["most"], hkv, gq, ep.shape[-1])
    eg[s["group"], s["rank"]] = ep
    op = (eg.transpose(1, 2).reshape(ng, hkv, s["most"] * gq, -1) @ vp).reshape(ng, hkv, s["most"], gq, d).transpose(1, 2)[s["group"], s["rank"]]
    o = (op + es @ vz) / l.masked_fill(l == 0, 1.0)
    return {"out": o.reshape(b, hq, d).to(s["q"].dtype), "lse": (m + l.log()).reshape(b, hq)}


def _exact_attend(c, seed):
    s = _prepare_attend(c, seed)
    b, hq, d = s["q"].shape
    hkv = c["hkv"]
    out = torch.zeros(b, hq, d, dtype=torch.float64, device=DEV)
    lse = torch.full((b, hq), float("-inf"), dtype=torch.float64, device=DEV)
    o, e = torch.arange(PAGE, device=DEV)[:, None], torch.arange(DIM, device=DEV)[None]
    kat = ((((o >> 2) & 1) * 16 + (e >> 3)) * 16 + 4 * (o >> 3) + (o & 3)) * 8 + (e & 7)  # where key o, dim e stands in a page
    vat = (((e >> 4) * 4 + (o >> 3)) * 16 + (e & 15)) * 8 + (o & 7)
    wide = {"bf16": lambda x: x.double(), "int8": lambda x: x.view(torch.int8).double(), "fp8": lambda x: x.view(torch.float8_e4m3fn).float().double()}[c["kv"]]
    lens, rows, plens = s["lens"].tolist(), s["rows"].tolist(), s["plens"].tolist()
    for i in range(b):
        n = lens[i]
        if n == 0:
            continue
        j = torch.arange(n, device=DEV)
        page = torch.where(j < plens[i], s["table"][rows[i]][j // PAGE], s["table"][i][j // PAGE]).long()
        k = wide(s["k"][page[:, None, None], torch.arange(hkv, device=DEV)[None, :, None], kat[j % PAGE][:, None]]) * s["scales"][0]
        v = wide(s["v"][page[:, None, None], torch.arange(hkv, device=DEV)[None, :, None], vat[j % PAGE][:, None]]) * s["scales"][1]
        q = s["q"][i].double().reshape(hkv, -1, d)
        w = torch.bmm(q, k.permute(1, 2, 0).contiguous()) * d ** -0.5
        lse[i] = w.logsumexp(-1).reshape(-1)
        out[i] = torch.bmm(w.softmax(-1), v.permute(1, 0, 2).contiguous()).reshape(hq, d)
    return {"out": out, "lse": lse}


def _work_attend(c):
    size = 2 if c["kv"] == "bf16" else 1
    mean = (1.0 if c["groups"] == 1 else 0.75) * c["prefix"]
    rows = c["batch"] - min(c["pad"], c["batch"] - 1)
    keys = c["groups"] * mean + rows * (c["suffix"] + 1) / 2
    io = 2 * c["batch"] * c["hq"] * DIM * (4 if c["dtype"] == "f32" else 2) + 4 * c["batch"] * c["hq"]
    return {"bytes": keys * 2 * c["hkv"] * DIM * size + io, "flops": rows * (mean + (c["suffix"] + 1) / 2) * 4 * c["hq"] * DIM}


# ---- log probabilities -------------------------------------------------------------------------
def _prepare_logprobs(c, seed):
    g = _gen(seed, 3)
    r, v = c["rows"], c["vocab"]
    x = torch.empty(r, v, dtype=DT[c["dtype"]], device=DEV).normal_(0.0, 2.5, generator=g)
    hot = torch.randint(0, v, (r, min(4, v)), generator=g, device=DEV)  # a few likely tokens a row
    x.scatter_add_(1, hot, torch.rand(hot.shape, generator=g, device=DEV).mul_(12.0).to(x.dtype))
    tokens = torch.randint(0, v, (r,), generator=g, device=DEV, dtype=torch.int32)
    tokens = torch.where(torch.rand(r, generator=g, device=DEV) < 0.7, hot[:, 0].to(torch.int32), tokens)
    if c["masked"]:
        keep = torch.rand(r, v, generator=g, device=DEV) >= c["masked"]
        keep.scatter_(1, hot, True)
        x.masked_fill_(~keep, float("-inf"))
    return {"x": x, "tokens": tokens, "top": c["top"]}


def _run_logprobs(s):
    if own:
        ops = _ops()
        p = ops.token_logprobs(s["x"], s["tokens"], top_k=s["top"])
        return {"logprobs": p.logprobs, "ranks": p.ranks, "entropy": p.entropy, "top_ids": p.top_ids, "top_logprobs": p.top_logprobs}
    x, k = s["x"].float() + 0.0, s["top"]
    t = s["tokens"].long()[:, None]
    m = x.amax(1, True)
    d = x - m
    e = d.exp()
    z = e.sum(1, True)
    log_z = z.log()
    entropy = log_z - torch.where(e > 0, d * e, 0.0).sum(1, True) / z
    xt = x.gather(1, t)
    at = torch.arange(x.shape[1], device=DEV)
    ranks = 1 + ((x > xt) | ((x == xt) & (at < t))).sum(1)
    # distinct whole keys: the value's order above, the lower index first below
    bits = x.view(torch.int32)
    key = (torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() << 32) + (0x7FFFFFFF - at)
    ids = 0x7FFFFFFF - (key.topk(k, 1).values & 0x7FFFFFFF)
    return {"logprobs": (xt - m - log_z)[:, 0], "ranks": ranks.to(torch.int32), "entropy": entropy[:, 0], "top_ids": ids.to(torch.int32),
            "top_logprobs": x.gather(1, ids) - m - log_z}


def _exact_logprobs(c, seed):
    s = _prepare_logprobs(c, seed)
    lp, ent, top = [], [], []
    for x, t in zip(s["x"].split(64), s["tokens"].split(64)):
        y = x.double()
        y = y - y.logsumexp(1, True)
        lp.append(y.gather(1, t.long()[:, None])[:, 0])
        ent.append(torch.special.entr(y.exp()).sum(1))
        top.append(y.topk(c["top"], 1).values)
    return {"logprobs": torch.cat(lp), "ranks": None, "entropy": torch.cat(ent), "top_ids": None, "top_logprobs": torch.cat(top)}


def _work_logprobs(c):
    n = c["rows"] * c["vocab"]
    return {"bytes": n * (4 if c["dtype"] == "f32" else 2) + c["rows"] * (16 + 8 * c["top"]), "flops": 5 * n}


# ---- the cases' functions ----------------------------------------------------------------------
def prepare(case, seed):
    fn = {"plan": _prepare_plan, "rotary": _prepare_rotary, "attend": _prepare_attend, "logprobs": _prepare_logprobs}[case["op"]]
    return {"op": case["op"], **fn(case, seed)}


def run(state):
    return {"plan": _run_plan, "rotary": _run_rotary, "attend": _run_attend, "logprobs": _run_logprobs}[state["op"]](state)


def work(case):
    return {"plan": _work_plan, "rotary": _work_rotary, "attend": _work_attend, "logprobs": _work_logprobs}[case["op"]](case)


def exact(case, seed):
    if case["op"] == "plan":  # whole numbers alone
        return None
    return {"rotary": _exact_rotary, "attend": _exact_attend, "logprobs": _exact_logprobs}[case["op"]](case, seed)
