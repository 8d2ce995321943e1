"""Plain 64-bit implementations of the cache append and of the attention over an 8-bit cache, token by
token, for the tests."""

import math

import numpy as np
import torch

E4M3_MAX = 448.0


def rotate(x, cs, interleaved):
    """Rows ``x`` [..., D] (float64) with the last R dims turned by ``cs`` [R] (cos then sin)."""
    R = cs.numel()
    y = x.clone()
    c, s = cs[: R // 2], cs[R // 2:]
    tail = x[..., x.shape[-1] - R:]
    if interleaved:
        a, b = tail[..., 0::2], tail[..., 1::2]
        new = torch.stack([a * c - b * s, a * s + b * c], dim=-1).flatten(-2)
    else:
        a, b = tail[..., : R // 2], tail[..., R // 2:]
        new = torch.cat([a * c - b * s, a * s + b * c], dim=-1)
    y[..., x.shape[-1] - R:] = new
    return y


def smallest_scale(amax):
    """Smallest power of two s with amax <= 448 s, in [2^-60, 2^60]."""
    k = -60
    while k < 60 and amax > E4M3_MAX * 2.0 ** k:
        k += 1
    return 2.0 ** k


def positions(q_lens, kv_lens):
    """(request, position) of every flat TND row."""
    return [(b, kv_lens[b] - n + s) for b, n in enumerate(q_lens) for s in range(n)]


def append(kv, cache, scale, table, where, rope, interleaved=True, step=1):
    """Expected cache after an append, in place of copies.

    ``kv`` float64 [T, D] on the CPU; ``cache`` float64 values [blocks, bs, D] (16 bits) or codes' values (8
    bits, with ``scale`` float64 [blocks]); ``where[t]`` = (request, position) or None.  Returns (cache,
    scale, written): new rows unrounded (8 bits: divided by the scale), rows rounded again as
    code * old / new, and a mask: 0 untouched, 1 written by this call, 2 rounded again."""
    cache = cache.clone()
    scale = None if scale is None else scale.clone()
    bs = cache.shape[1]
    written = torch.zeros(cache.shape[:2], dtype=torch.int32)
    touched = {}
    for t, w in enumerate(where):
        if w is None or w[1] < 0 or w[1] // bs >= table.shape[1]:
            continue
        b, p = w
        phys = int(table[b, p // bs])
        if not 0 <= phys < cache.shape[0]:
            continue
        x = kv[t]
        if rope is not None:
            if p * step >= rope.shape[0]:
                continue
            x = rotate(x, rope[p * step], interleaved)
        touched.setdefault(phys, []).append((p % bs, x))
    for phys, rows in touched.items():
        s = 1.0
        if scale is not None:
            finite = [float(x[torch.isfinite(x)].abs().max()) if torch.isfinite(x).any() else 0.0 for _, x in rows]
            need, o0, old = smallest_scale(max(finite)), min(o for o, _ in rows), float(scale[phys])
            ok = 2.0 ** -60 <= old <= 2.0 ** 60
            s = need if o0 == 0 or not ok else max(old, need)
            if o0 > 0 and ok and s > old:
                cache[phys, :o0] *= old / s
                written[phys, :o0] = 2
            scale[phys] = s
        for o, x in rows:
            cache[phys, o] = x / s
            written[phys, o] = 1
    return cache, scale, written


def visible(case, t_req, pos, idx_row):
    """Positions of the window's keys and of the compressed keys of a token."""
    left = max(pos - case["win_left"], 0)
    ori = list(range(min(case["first"], left))) + list(range(left, pos + 1)) if pos >= 0 else []
    cmp_ = []
    if case["scenario"] >= 2 and pos >= 0:
        limit = (pos + 1) // case["ratio"]
        if case["scenario"] == 2:
            cmp_ = list(range(limit))
        else:
            for i, v in enumerate(idx_row[: max(limit, 0)]):
                if v == -1:
                    break
                if 0 <= v < limit:
                    cmp_.append(int(v))
    return ori, cmp_


def gather(codes, scale, table_row, at):
    """Rows [n, D] in float64: code * scale; unmapped blocks and blocks without a scale read as zeros."""
    bs, D = codes.shape[1], codes.shape[2]
    if not at:
        return torch.zeros((0, D), dtype=torch.float64, device=codes.device)
    at = np.asarray(at)
    blk = at // bs
    phys = np.where(blk < len(table_row), np.asarray(table_row)[np.minimum(blk, len(table_row) - 1)], -1)
    ok = (phys >= 0) & (phys < codes.shape[0])
    ph = torch.from_numpy(np.where(ok, phys, 0)).to(codes.device)
    x = codes.view(torch.uint8)[ph, torch.from_numpy(at % bs).to(codes.device)].view(torch.float8_e4m3fn).double()
    s = scale.double().reshape(-1)[ph]
    good = torch.from_numpy(ok).to(codes.device) & (s >= 2.0 ** -60) & (s <= 2.0 ** 60)
    return torch.where(good[:, None], x * torch.where(good, s, torch.ones_like(s))[:, None], torch.zeros_like(x))


def attend(case, q, pos, req, ori, cmp_, idx_row, sinks, scale, Dv):
    """One token: (out, lse, spread, top, reach) in float64.  ``spread`` = sum_j w_j |v_j|, ``top`` =
    max_j w_j sum_j |v_j| (both [N1, Dv]) and ``reach`` = max_j scale sum_d |q_d k_jd| ([N1]) are what the
    kernels' rounding errors scale with."""
    o_at, c_at = visible(case, req, pos, idx_row)
    k = gather(*ori, o_at)
    if c_at:
        k = torch.cat([k, gather(*cmp_, c_at)])
    N1 = q.shape[0]
    sink = torch.full((N1,), -math.inf, dtype=torch.float64, device=q.device) if sinks is None else sinks.double()
    if k.shape[0] == 0:
        z = torch.zeros((N1, Dv), dtype=torch.float64, device=q.device)
        return z, sink, z, z, torch.zeros_like(sink)
    s = q.double() @ k.T * scale
    lse = torch.logsumexp(torch.cat([s, sink[:, None]], dim=1), dim=1)
    w = torch.exp(s - lse[:, None])
    v = k[:, :Dv]
    reach = (q.double().abs() @ k.abs().T * scale).amax(dim=1)
    return w @ v, lse, w @ v.abs(), w.amax(dim=1)[:, None] * v.abs().sum(dim=0)[None, :], reach
