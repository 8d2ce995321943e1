"""Operators around the paged shared-KV cache: their cases, plain forms and exact values.

Two operators.  ``append`` writes new K = V rows into a paged cache, rotating the positional tail of
each row (and, where given, of the query heads) on the way; the cache holds 16-bit rows, or 8-bit
(e4m3) rows with one power-of-two scale per block of tokens and head.  ``attend`` is the sparse
shared-KV attention (sliding window, first tokens, compressed rows, sink) over such an 8-bit cache.
"""

import math

import numpy as np
import torch

own = False

DEV = "cuda"
E4M3_MAX = 448.0
EXP_MIN, EXP_MAX = -60, 60  # range of the scales' exponents
ROPE = 64
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp8": torch.float8_e4m3fn}


def listed():
    a = dict(op="append", dim=576, block=128, pool="fp8", src="bf16", heads=0, interleaved=True, step=1, new_lo=1, new_hi=1)
    t = dict(op="attend", dim=576, block=128, heads=128, src="bf16", topk=2048, ratio=4, scenario=3, win_left=127, first=0, new=1)
    return [
        # one request generates one token: the latency of a call
        dict(a, name="append one token, 8 bits", requests=1, ctx_lo=300, ctx_hi=300),
        # a decode step of 64 requests with 128 query heads, 16-bit cache: rows and queries in one call
        dict(a, name="append 64 tokens and q, 16 bits", requests=64, pool="bf16", heads=128, ctx_lo=64, ctx_hi=512),
        # a decode step of a large batch, blocks partly filled
        dict(a, name="append 512 tokens, 8 bits", requests=512, ctx_lo=1, ctx_hi=256),
        # chunked prefill: 4 requests of 8192 new tokens, odd positions where the chunk begins
        dict(a, name="append 4 x 8192 rows, 8 bits", requests=4, new_lo=8192, new_hi=8192, ctx_lo=0, ctx_hi=1000),
        # compressed rows (one for 4 tokens) of ragged chunks, 16-bit cache of 48-row blocks, halves rotated
        dict(a, name="append ragged rows, 16 bits", requests=29, dim=512, block=48, pool="fp16", src="fp16", interleaved=False,
             step=4, new_lo=0, new_hi=700, ctx_lo=0, ctx_hi=300),
        # one request decodes one token of a long context: the latency of a call
        dict(t, name="attend decode 1", requests=1, ctx_lo=32000, ctx_hi=32000),
        # a decode step of 64 requests
        dict(t, name="attend decode 64", requests=64, ctx_lo=8192, ctx_hi=32768),
        # drafted tokens verified: 32 requests of 2 tokens, 64 heads
        dict(t, name="attend 32 x 2, 64 heads", requests=32, new=2, heads=64, ctx_lo=4096, ctx_hi=65536),
        # a decode step of many requests of very different lengths
        dict(t, name="attend decode 256 mixed", requests=256, ctx_lo=1000, ctx_hi=60000, dim=512, topk=1000),
        # a prefill chunk on earlier context
        dict(t, name="attend prefill 2 x 1024", requests=2, new=1024, ctx_lo=1024, ctx_hi=16384),
        # streaming decode: a long window, the first 4 tokens stay visible, no compressed rows
        dict(t, name="attend window and first tokens", requests=48, heads=16, dim=512, topk=0, scenario=1, win_left=1023, first=4,
             ctx_lo=1, ctx_hi=9000),
        # every compressed row is visible (no index), few requests
        dict(t, name="attend all compressed rows", requests=9, topk=0, scenario=2, ctx_lo=3, ctx_hi=14000),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.4:
        pool = rng.choice(["fp8", "fp8", "bf16", "fp16"])
        src = pool if pool != "fp8" else rng.choice(["bf16", "fp16"])
        requests = _log(rng, 1, 512)
        hi = max(1, min(8192, 30000 // requests))
        new_hi = _log(rng, 1, hi)
        return dict(op="append", dim=rng.choice([512, 576]), block=rng.choice([16, 48, 64, 128, 128]), pool=pool, src=src,
                    heads=rng.choice([0, 0, rng.randint(1, 128)]) if new_hi * requests <= 2048 else 0,
                    interleaved=rng.random() < 0.5, step=rng.choice([1, 1, 4]), requests=requests,
                    new_lo=rng.randint(0, new_hi), new_hi=new_hi, ctx_lo=rng.randint(0, 5), ctx_hi=rng.randint(5, 400))
    scenario = rng.choice([1, 2, 3, 3, 3])
    requests = _log(rng, 1, 256)
    new = rng.choice([1, 1, 2, 3, _log(rng, 1, max(2, 1500 // requests))])
    ctx_hi = _log(rng, 200, 60000 if scenario != 2 else 8000)
    if requests * new > 400:
        requests = max(1, 400 // new) if scenario == 2 else requests
    requests = max(1, min(requests, 1500 // new))
    if scenario == 2:
        requests = max(1, min(requests, 400 // new))
    return dict(op="attend", dim=rng.choice([512, 576]), block=rng.choice([16, 64, 128, 128]), heads=rng.randint(1, 128), src="bf16",
                topk=rng.randint(1, 2048) if scenario == 3 else 0, ratio=rng.choice([4, 4, 8, 128]), scenario=scenario,
                win_left=rng.choice([127, 127, rng.randint(0, 1023)]), first=rng.choice([0, 0, 4, rng.randint(1, 70)]), new=new,
                requests=requests, ctx_lo=rng.randint(1, 200), ctx_hi=ctx_hi)


# ---- inputs ---------------------------------------------------------------------------------------

def _lengths(case, seed):
    """Contexts before the call and new tokens, per request: the same lengths for every seed, in an order of its own."""
    rng = np.random.default_rng(1)
    n = case["requests"]
    lo, hi = case["ctx_lo"], case["ctx_hi"]
    ctx = np.floor(np.exp(rng.uniform(np.log(lo + 1), np.log(hi + 1.999), size=n))).astype(np.int64) - 1
    ctx = np.clip(ctx, lo, hi)
    if case["op"] == "append":
        new = rng.integers(case["new_lo"], case["new_hi"] + 1, size=n)
    else:
        new = np.full(n, case["new"], dtype=np.int64)
    rng = np.random.default_rng(seed)
    order = rng.permutation(n)
    return rng, ctx[order].tolist(), new[order].tolist()


def _table(rng, lens, block):
    """A block table over a pool of exactly the blocks that ``lens`` need, in a random order."""
    per = [(n + block - 1) // block for n in lens]
    total, width = max(sum(per), 1), max(max(per), 1)
    phys = rng.permutation(total).astype(np.int32)
    table = np.full((len(lens), width), -1, dtype=np.int32)
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = phys[at:at + n]
        at += n
    return torch.from_numpy(table).to(DEV), total


def _scale_exp(amax):
    """Exponent k of the smallest power of two with amax <= 448 * 2^k, within the scales' range."""
    m, e = torch.frexp(amax)  # amax = m * 2^e, m in [0.5, 1)
    k = torch.where(m <= 0.875, e - 9, e - 8)
    return torch.where(amax > 0, k, torch.full_like(k, EXP_MIN)).clamp(EXP_MIN, EXP_MAX)


def _pool8(gen, blocks, block, dim):
    """A filled 8-bit pool and its scales [blocks, 1]."""
    pool = torch.empty((blocks, block, 1, dim), dtype=torch.float8_e4m3fn, device=DEV)
    scale = torch.empty((blocks, 1), dtype=torch.float32, device=DEV)
    step = max(1, (1 << 28) // (block * dim))
    for s in range(0, blocks, step):
        e = min(blocks, s + step)
        x = torch.randn((e - s, block, 1, dim), generator=gen, device=DEV)
        x *= 0.5 * torch.exp2(torch.rand((e - s, 1, 1, 1), generator=gen, device=DEV) * 2 - 1)  # blocks differ in size
        sc = torch.exp2(_scale_exp(x.abs().amax(dim=(1, 2, 3))).float())
        pool[s:e] = (x / sc[:, None, None, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
        scale[s:e, 0] = sc
    return pool, scale


def _rope_table(positions):
    inv = 10000.0 ** (-torch.arange(0, ROPE, 2, dtype=torch.float64, device=DEV) / ROPE)
    ang = torch.arange(positions, dtype=torch.float64, device=DEV)[:, None] * inv[None, :]
    return torch.cat([ang.cos(), ang.sin()], dim=1).to(torch.float32)


def prepare(case, seed):
    rng, ctx, new = _lengths(case, seed)
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    lens = [c + n for c, n in zip(ctx, new)]
    T, dim, block = sum(new), case["dim"], case["block"]
    src = TYPES[case["src"]]
    cu = torch.tensor(np.concatenate([[0], np.cumsum(new)]).astype(np.int32), device=DEV)
    seq = torch.tensor(lens, dtype=torch.int32, device=DEV)
    st = dict(case=case, cu=cu, seq=seq, max_new=max(new))
    if case["op"] == "append":
        table, blocks = _table(rng, lens, block)
        st.update(table=table, rope=_rope_table(case["step"] * max(lens) + 1))
        if case["pool"] == "fp8":
            st["pool"], st["scale"] = _pool8(gen, blocks, block, dim)
        else:
            st["pool"] = (torch.randn((blocks, block, 1, dim), generator=gen, device=DEV) * 0.5).to(TYPES[case["pool"]])
            st["scale"] = None
        st["kv"] = (torch.randn((T, dim), generator=gen, device=DEV) * 0.5).to(src)
        st["q"] = (torch.randn((T, case["heads"], dim), generator=gen, device=DEV) * 0.5).to(src) if case["heads"] else None
        return st
    N1 = case["heads"]
    st["table"], blocks = _table(rng, lens, block)
    st["pool"], st["scale"] = _pool8(gen, blocks, block, dim)
    st["q"] = (torch.randn((T, N1, dim), generator=gen, device=DEV) * torch.exp2(torch.rand((T, N1, 1), generator=gen, device=DEV) * 3 - 1)).to(src)
    st["sinks"] = torch.rand((N1,), generator=gen, device=DEV) * 2 - 1
    st["softmax_scale"] = dim ** -0.5
    st["cmp_table"] = st["cmp_pool"] = st["cmp_scale"] = st["idx"] = None
    if case["scenario"] >= 2:
        st["cmp_table"], blocks = _table(rng, [n // case["ratio"] for n in lens], block)
        st["cmp_pool"], st["cmp_scale"] = _pool8(gen, blocks, block, dim)
    if case["scenario"] == 3:
        limit = (torch.repeat_interleave(torch.tensor([c + 1 for c in ctx], device=DEV), torch.tensor(new, device=DEV))
                 + torch.cat([torch.arange(n, device=DEV) for n in new])) // case["ratio"]
        K, most = case["topk"], max(1, max(lens) // case["ratio"])
        idx = torch.full((T, K), -1, dtype=torch.int32, device=DEV)
        step = max(1, (1 << 26) // most)
        for s in range(0, T, step):
            keys = torch.rand((min(T, s + step) - s, most), generator=gen, device=DEV)
            keys = keys.masked_fill(torch.arange(most, device=DEV)[None, :] >= limit[s:s + step, None], -1.0)
            v, at = torch.topk(keys, min(K, most), dim=1)
            idx[s:s + step, :at.shape[1]] = torch.where(v >= 0, at, -1).to(torch.int32)
        st["idx"] = idx[:, None, :]
    return st


# ---- the operators ----------------------------------------------------------------------------------

def run(st):
    case = st["case"]
    if case["op"] == "append":
        if own:
            from dsv4_planb_b200.cache import sharedkv_cache_append

            q = sharedkv_cache_append(st["kv"], cache=st["pool"], cache_scale=st["scale"], block_table=st["table"], cu_seqlens_q=st["cu"],
                                      seqused_kv=st["seq"], rope_table=st["rope"], rope_interleaved=case["interleaved"],
                                      rope_step=case["step"], q=st["q"])
        else:
            q = _append_plain(st)
        return dict(pool=st["pool"], scale=st["scale"], q=q)
    if own:
        from dsv4_planb_b200.attn_fp8 import sparse_attn_sharedkv_fp8

        out, lse = sparse_attn_sharedkv_fp8(st["q"], ori_kv=st["pool"], ori_kv_scale=st["scale"], cmp_kv=st["cmp_pool"],
                                            cmp_kv_scale=st["cmp_scale"], cmp_sparse_indices=st["idx"], ori_block_table=st["table"],
                                            cmp_block_table=st["cmp_table"], cu_seqlens_q=st["cu"], seqused_kv=st["seq"], sinks=st["sinks"],
                                            softmax_scale=st["softmax_scale"], cmp_ratio=case["ratio"], ori_win_left=case["win_left"],
                                            ori_first=case["first"], v_head_dim=512, return_softmax_lse=True)
    else:
        out, lse = _attend_plain(st)
    return dict(out=out, lse=lse)


def _tokens(st, T):
    """Request and position of every new token."""
    t = torch.arange(T, device=DEV)
    b = torch.searchsorted(st["cu"][1:].contiguous(), t.to(torch.int32), right=True)
    cu = st["cu"].long()
    pos = st["seq"].long()[b] - (cu[b + 1] - cu[b]) + (t - cu[b])
    return b, pos


def _rotate(x, cs, interleaved):
    """The last ROPE dims of ``x`` (32 bits) turned by the angles of ``cs`` = (cos | sin)."""
    c, s = cs[..., :ROPE // 2], cs[..., ROPE // 2:]
    head, tail = x[..., :-ROPE], x[..., -ROPE:]
    if interleaved:
        a, b = tail[..., 0::2], tail[..., 1::2]
        tail = torch.stack([a * c - b * s, a * s + b * c], dim=-1).flatten(-2)
    else:
        a, b = tail[..., :ROPE // 2], tail[..., ROPE // 2:]
        tail = torch.cat([a * c - b * s, a * s + b * c], dim=-1)
    return torch.cat([head, tail], dim=-1)


def _append_plain(st):
    case, pool, bs = st["case"], st["pool"], st["case"]["block"]
    T, dim = st["kv"].shape
    if T == 0:
        return None if st["q"] is None else st["q"].clone()
    b, pos = _tokens(st, T)
    phys, off = st["table"].long()[b, pos // bs], pos % bs
    cs = st["rope"][pos * case["step"]]
    x = _rotate(st["kv"].float(), cs, case["interleaved"])
    q = None
    if st["q"] is not None:
        q = _rotate(st["q"].float(), cs[:, None, :], case["interleaved"]).to(st["q"].dtype)
    if st["scale"] is None:
        pool[phys, off, 0] = x.to(pool.dtype)
        return q
    n = pool.shape[0]
    amax = torch.zeros(n, device=DEV).scatter_reduce_(0, phys, x.abs().amax(dim=1), "amax")
    start = torch.full((n,), bs, device=DEV, dtype=torch.long).scatter_reduce_(0, phys, off, "amin")
    need = torch.exp2(_scale_exp(amax).float())
    old = st["scale"][:, 0]
    scale = torch.where(start == bs, old, torch.where(start == 0, need, torch.maximum(old, need)))
    grown = torch.nonzero((start > 0) & (start < bs) & (scale > old)).flatten()  # rows already there are rounded again
    rows = (pool[grown].float() * (old[grown] / scale[grown])[:, None, None, None]).to(pool.dtype)
    keep = torch.arange(bs, device=DEV)[None, :] < start[grown, None]
    pool.view(torch.uint8)[grown] = torch.where(keep[:, :, None, None], rows.view(torch.uint8), pool.view(torch.uint8)[grown])
    codes = (x / scale[phys, None]).clamp(-E4M3_MAX, E4M3_MAX).to(pool.dtype)
    pool.view(torch.uint8)[phys, off, 0] = codes.view(torch.uint8)
    st["scale"][:, 0] = scale
    return q


def _rows(pool, scale, table, b, pos, ok):
    """Rows at positions ``pos`` [T, n] of requests ``b`` in 32 bits; what is not ``ok`` reads as zeros."""
    bs, dim = pool.shape[1], pool.shape[3]
    pos = pos.masked_fill(~ok, 0)
    phys = table.long()[b[:, None], pos // bs]
    flat = (phys.clamp(min=0) * bs + pos % bs).masked_fill(~ok, 0)
    x = pool.view(torch.uint8).reshape(-1, dim)[flat].view(torch.float8_e4m3fn).float()
    return x.mul_((scale[:, 0][phys.clamp(min=0)] * ok)[:, :, None])


def _attend_plain(st):
    case, q = st["case"], st["q"]
    T, N1, dim = q.shape
    b, pos = _tokens(st, T)
    left = (pos - case["win_left"]).clamp(min=0)
    w = torch.arange(min(case["win_left"] + 1, int(st["table"].shape[1]) * case["block"]), device=DEV)[None, :]
    at = left[:, None] + w
    ok = at <= pos[:, None]
    if case["first"]:
        f = torch.arange(case["first"], device=DEV)[None, :].expand(T, -1)
        at, ok = torch.cat([f, at], 1), torch.cat([f < left[:, None], ok], 1)
    kv = _rows(st["pool"], st["scale"], st["table"], b, at, ok)
    if case["scenario"] >= 2:
        limit = (pos + 1) // case["ratio"]
        if case["scenario"] == 3:
            at = st["idx"][:, 0].long()
        else:
            at = torch.arange(st["cmp_table"].shape[1] * case["block"], device=DEV)[None, :].expand(T, -1)
        ok2 = (at >= 0) & (at < limit[:, None])
        kv = torch.cat([kv, _rows(st["cmp_pool"], st["cmp_scale"], st["cmp_table"], b, at, ok2)], 1)
        ok = torch.cat([ok, ok2], 1)
    s = torch.matmul(q.float(), kv.transpose(1, 2)).mul_(st["softmax_scale"]).masked_fill_(~ok[:, None, :], -math.inf)
    sink = st["sinks"][None, :]
    top = torch.maximum(s.amax(dim=2), sink)
    p = s.sub_(top[:, :, None]).exp_()
    total = p.sum(dim=2) + (sink - top).exp()
    out = torch.matmul(p, kv[:, :, :512]).div_(total[:, :, None])
    return out.to(q.dtype), top + total.log()


# ---- what a pass cannot do without --------------------------------------------------------------------

def work(case):
    _, ctx, new = _lengths(case, 1)
    T, dim, block = sum(new), case["dim"], case["block"]
    if case["op"] == "append":
        size = 1 if case["pool"] == "fp8" else 2
        spans = sum((c + n + block - 1) // block - c // block for c, n in zip(ctx, new) if n)
        data = T * (dim * 2 + dim * size + ROPE * 4 + case["heads"] * dim * 2 * 2) + spans * (4 + (8 if size == 1 else 0))
        return {"bytes": data + 8 * len(new), "flops": 3 * ROPE * T * (1 + case["heads"]) + (2 * T * dim if size == 1 else 0)}
    keys = rows = 0
    for c, n in zip(ctx, new):
        L = c + n
        spread = set()
        for s in range(n):
            p = c + s
            w = min(p, case["win_left"]) + 1 + min(case["first"], max(0, p - case["win_left"]))
            thr = (p + 1) // case["ratio"] if case["scenario"] >= 2 else 0
            keys += w + (min(thr, case["topk"]) if case["scenario"] == 3 else thr)
        rows += min(L, case["win_left"] + n) + min(case["first"], max(0, L - case["win_left"]))
        # distinct compressed rows: all that are below the limit, or as many as the indices can name
        top = L // case["ratio"] if case["scenario"] >= 2 else 0
        rows += min(top, n * case["topk"]) if case["scenario"] == 3 else top
    H = case["heads"]
    data = rows * (dim + 4.0 / block) + T * H * (dim * 2 + 512 * 2 + 4) + (T * case["topk"] * 4 if case["scenario"] == 3 else 0)
    return {"bytes": data, "flops": 2 * H * keys * (dim + 512)}


# ---- exact values -------------------------------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    cu, lens = st["cu"].tolist(), st["seq"].tolist()
    if case["op"] == "append":
        return _append_exact(st, cu, lens)
    N1 = case["heads"]
    out = torch.zeros((cu[-1], N1, 512), dtype=torch.float64, device=DEV)
    lse = torch.zeros((cu[-1], N1), dtype=torch.float64, device=DEV)
    table = st["table"].cpu().numpy().astype(np.int64)
    cmp_table = st["cmp_table"].cpu().numpy().astype(np.int64) if st["cmp_table"] is not None else None
    idx = st["idx"].cpu().numpy() if st["idx"] is not None else None
    bs = case["block"]

    def fetch(pool, scale, tab, at):
        blk = torch.from_numpy(tab[at // bs]).to(DEV)
        codes = pool.view(torch.uint8)[blk, torch.from_numpy(at % bs).to(DEV), 0].view(torch.float8_e4m3fn)
        return codes.double() * scale.double()[blk]

    sink = st["sinks"].double()
    for r, n in enumerate(lens):
        for t in range(cu[r], cu[r + 1]):
            p = n - (cu[r + 1] - t)
            lo = max(0, p - case["win_left"])
            seen = np.concatenate([np.arange(min(case["first"], lo)), np.arange(lo, p + 1)])
            k = fetch(st["pool"], st["scale"], table[r], seen)
            if case["scenario"] >= 2:
                limit = (p + 1) // case["ratio"]
                c = np.arange(limit) if idx is None else idx[t, 0][(idx[t, 0] >= 0) & (idx[t, 0] < limit)].astype(np.int64)
                if len(c):
                    k = torch.cat([k, fetch(st["cmp_pool"], st["cmp_scale"], cmp_table[r], c)])
            s = torch.cat([st["q"][t].double() @ k.T * st["softmax_scale"], sink[:, None]], dim=1)
            lse[t] = torch.logsumexp(s, dim=1)
            out[t] = torch.softmax(s, dim=1)[:, :-1] @ k[:, :512]
    return dict(out=out, lse=lse)


def _append_exact(st, cu, lens):
    case, bs = st["case"], st["case"]["block"]
    half = ROPE // 2
    pool, table = st["pool"].double(), st["table"].cpu().numpy()
    scale = None if st["scale"] is None else st["scale"].double()
    q = None if st["q"] is None else st["q"].double()
    for r, n in enumerate(lens):
        a, e = cu[r], cu[r + 1]
        if a == e:
            continue
        p0 = n - (e - a)
        where = np.arange(p0, n)
        cs = st["rope"].double()[torch.from_numpy(where * case["step"]).to(DEV)]
        z = torch.complex(cs[:, :half], cs[:, half:])

        def turn(x, z):
            y = x.clone()
            tail = x[..., -ROPE:]
            if case["interleaved"]:
                w = torch.complex(tail[..., 0::2], tail[..., 1::2]) * z
                y[..., -ROPE::2], y[..., -ROPE + 1::2] = w.real, w.imag
            else:
                w = torch.complex(tail[..., :half], tail[..., half:]) * z
                y[..., -ROPE:-half], y[..., -half:] = w.real, w.imag
            return y

        x = turn(st["kv"][a:e].double(), z)
        if q is not None:
            q[a:e] = turn(q[a:e], z[:, None, :])
        for blk in range(p0 // bs, (n - 1) // bs + 1):
            lo, hi = max(p0, blk * bs), min(n, (blk + 1) * bs)
            ph = int(table[r, blk])
            part = x[lo - p0:hi - p0]
            if scale is not None:
                amax = float(part.abs().max())
                k = EXP_MIN if amax == 0 else min(max(math.ceil(math.log2(amax / E4M3_MAX)), EXP_MIN), EXP_MAX)
                s = 2.0 ** k if lo == blk * bs else max(2.0 ** k, float(scale[ph, 0]))
                pool[ph, :lo - blk * bs] *= float(scale[ph, 0]) / s
                scale[ph, 0] = s
                part = part / s
            pool[ph, lo - blk * bs:hi - blk * bs, 0] = part
    return dict(pool=pool, scale=scale, q=q)
