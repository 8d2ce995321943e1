"""sparse_attn_sharedkv_fp8 on the GPU against the plain 64-bit implementation."""

import math

import numpy as np
import pytest
import torch

from dsv4_planb_b200.attn_fp8 import sparse_attn_sharedkv_fp8
from dsv4_planb_b200.cache import rope_table, sharedkv_cache_append
from tests import _cache_ref as ref

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
HALF_STEP = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11}


def pool(g, rng, lens, bs, D, size=0.5):
    per = [math.ceil(n / bs) if n > 0 else 0 for n in lens]
    blocks = sum(per) + 1
    phys = rng.permutation(blocks).astype(np.int32)
    table = np.full((len(lens), max(max(per), 1)), -1, np.int32)
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = phys[at:at + n]
        at += n
    scale = torch.exp2(torch.randint(-9, -5, (blocks, 1), generator=g).float())
    x = torch.randn((blocks, bs, 1, D), generator=g) * size
    codes = (x / scale[:, :, None, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    return codes.cuda(), scale.cuda(), table


def make(q_lens, kv_lens, *, N1=128, D=576, Dv=512, K=256, ratio=4, scenario=3, win_left=127, first=0, bs=128, src="bf16", seed=0,
         q_size=1.0, skips=False):
    g = torch.Generator().manual_seed(seed)
    rng = np.random.default_rng(seed)
    T = sum(q_lens)
    m = dict(case=dict(win_left=win_left, first=first, ratio=ratio, scenario=scenario), q_lens=q_lens, kv_lens=kv_lens, Dv=Dv, src=src)
    m["where"] = ref.positions(q_lens, kv_lens)
    m["q"] = (torch.randn((T, N1, D), generator=g) * q_size).to(TYPES[src]).cuda()
    m["ori"] = pool(g, rng, kv_lens, bs, D)
    m["cmp"] = pool(g, rng, [n // ratio for n in kv_lens], bs, D) if scenario >= 2 else None
    m["sinks"] = (torch.rand(N1, generator=g) * 2 - 1).cuda()
    m["idx"] = None
    if scenario == 3:
        idx = np.full((T, 1, K), -1, np.int32)
        for t, (b, p) in enumerate(m["where"]):
            limit = max((p + 1) // ratio, 0)
            take = rng.permutation(limit)[:K]
            idx[t, 0, :len(take)] = take
            if skips and len(take) > 3:
                idx[t, 0, 1] = limit + 5       # past the limit: skipped
                idx[t, 0, 2] = idx[t, 0, 0]    # twice the same row
                if t % 2:
                    idx[t, 0, len(take) // 2] = -1  # the scan stops here
        m["idx"] = torch.from_numpy(idx)
    m["scale"] = D ** -0.5
    return m


def kwargs(m):
    cu = torch.tensor(np.concatenate([[0], np.cumsum(m["q_lens"])]).astype(np.int32)).cuda()
    c = m["case"]
    a = dict(ori_kv=m["ori"][0], ori_kv_scale=m["ori"][1], ori_block_table=torch.from_numpy(m["ori"][2]).cuda(), cu_seqlens_q=cu,
             seqused_kv=torch.tensor(m["kv_lens"], dtype=torch.int32).cuda(), sinks=m["sinks"], softmax_scale=m["scale"],
             cmp_ratio=c["ratio"], ori_win_left=c["win_left"], ori_first=c["first"], v_head_dim=m["Dv"], return_softmax_lse=True)
    if m["cmp"] is not None:
        a.update(cmp_kv=m["cmp"][0], cmp_kv_scale=m["cmp"][1], cmp_block_table=torch.from_numpy(m["cmp"][2]).cuda())
    if m["idx"] is not None:
        a["cmp_sparse_indices"] = m["idx"].cuda()
    return a


def run(m, **kw):
    q = kw.pop("q", m["q"])
    return sparse_attn_sharedkv_fp8(q, **{**kwargs(m), **kw})


def check(m, out, lse, tokens=None, where=None):
    """Bars from the kernels' roundings.  Scores: sums of D products in 32 bits or on the tensor cores,
    whose 36 partial sums lose at most 2^-22 of the sum of magnitudes each: a score is off by
    d = 36 * 2^-22 * reach, with the softmax's exp (2^-21) and the log2-domain products of scores up to
    reach (3 * 2^-24 * reach).  Weights: off by a factor e^(2 d + 2^-20), rounded on the tensor cores to
    two e4m3 terms: relative 2^-9, after a rounding to fp16, 2^-12; and half of e4m3's smallest step,
    2^-10, where the second term is subnormal.  The weights' frame leaves the largest weight of a row at
    2^5.75 or more (the running maximum lags by less than 2^3 of 2^8.75), so 2^-10 is 2^-15.75 of it.
    The sums of out lose 2^-22 per step of the running magnitude.  One rounding at the end."""
    where = m["where"] if where is None else where
    cmp_ = m["cmp"]
    for t in (range(len(where)) if tokens is None else tokens):
        if where[t] is None:
            assert not out[t].any() and not lse[t].any()
            continue
        b, p = where[t]
        o, l, spread, top, reach = ref.attend(
            m["case"], m["q"][t], p, b, (m["ori"][0][:, :, 0], m["ori"][1], m["ori"][2][b]),
            None if cmp_ is None else (cmp_[0][:, :, 0], cmp_[1], cmp_[2][b]),
            None if m["idx"] is None else m["idx"][t, 0].numpy(), m["sinks"], m["scale"], m["Dv"])
        d = (36 * 2.0 ** -22 + 3 * 2.0 ** -24) * reach
        finite = torch.isfinite(l)
        assert torch.equal(l[~finite].float(), lse[t][~finite]), (t, lse[t])
        err = (lse[t].double() - l).abs()[finite]
        tol = (d + 2.0 ** -20 + 2.0 ** -22 * l.abs())[finite]
        assert (err <= tol).all(), (t, float((err - tol).max()), float(err.max()))
        tol = HALF_STEP[m["src"]] * o.abs() + 2.0 ** -24 + spread * (2 * d + 2.0 ** -20 + 2.0 ** -9 + 2.0 ** -12 + 70 * 2.0 ** -22)[:, None] + 2.0 ** -15.75 * top
        err = (out[t].double() - o).abs()
        assert (err <= tol).all(), (t, float((err - tol).max()), float(err.max()))


KERNELS = ["simt", "tc"]
SHAPES = [
    dict(q_lens=[1], kv_lens=[1]),
    dict(q_lens=[1], kv_lens=[3]),
    dict(q_lens=[1, 1, 1], kv_lens=[64, 65, 129], N1=1, K=7),
    dict(q_lens=[1] * 5, kv_lens=[128, 700, 1500, 9000, 4], N1=16),
    dict(q_lens=[3, 0, 40, 1], kv_lens=[900, 5, 40, 130], N1=64, D=512, skips=True),
    dict(q_lens=[2, 1], kv_lens=[3000, 20000], N1=128, K=2048, skips=True),
    dict(q_lens=[4, 1], kv_lens=[300, 77], N1=33, ratio=128, bs=16),
    dict(q_lens=[90], kv_lens=[400], N1=20, K=65, bs=48),
    dict(q_lens=[1] * 80, kv_lens=[10 + 61 * i for i in range(80)], N1=8, K=640),
    dict(q_lens=[3, 1], kv_lens=[700, 12], scenario=1, N1=128),
    dict(q_lens=[5, 1, 1], kv_lens=[5, 70, 1], scenario=1, N1=7, D=512, win_left=0),
    dict(q_lens=[2, 1, 9], kv_lens=[5000, 66, 9], scenario=1, N1=48, win_left=1023, first=4),
    dict(q_lens=[2, 1, 3], kv_lens=[500, 66, 9], scenario=1, N1=12, win_left=5, first=70),
    dict(q_lens=[1, 6], kv_lens=[2300, 700], scenario=2, N1=128, first=3),
    dict(q_lens=[1, 2, 2], kv_lens=[5, 900, 2], scenario=2, N1=11, ratio=8, win_left=60),
]


def ident(s):
    return "-".join(f"{k}{v}".replace(" ", "") if not isinstance(v, list) else f"{len(v)}x" for k, v in s.items())[:60]


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("shape", SHAPES, ids=ident)
def test_against_64_bits(cuda_device, shape, kernel):
    m = make(**shape, seed=len(shape["q_lens"]))
    out, lse = run(m, kernel=kernel, check_status=True)
    check(m, out, lse)


@pytest.mark.parametrize("shape", [dict(D=64, Dv=32), dict(D=1024, Dv=512, N1=3),
                                   dict(D=576, Dv=512, src="fp16", N1=130), dict(D=512, Dv=512, src="fp16", N1=64)], ids=ident)
def test_other_shapes(cuda_device, shape):
    """What the tensor-core kernel does not take runs on the CUDA cores under "auto"."""
    m = make([2, 1, 5], [400, 33, 900], K=100, **shape)
    out, lse = run(m, check_status=True)
    check(m, out, lse)


@pytest.mark.parametrize("kernel", KERNELS)
def test_sharp_and_flat_scores(cuda_device, kernel):
    """Scores of a few hundred (one key takes all) and of nearly zero; queries of very different sizes."""
    m = make([1] * 6, [3000] * 6, N1=128, seed=3)
    size = torch.exp2(torch.arange(128, device="cuda").float() / 4 - 20)  # 2^-20 .. 2^11.75
    m["q"] = (m["q"].float() * size[None, :, None]).to(torch.bfloat16)
    m["q"][2, 5] = 0
    m["q"][3, :, 100:] = 0
    check(m, *run(m, kernel=kernel, check_status=True))


@pytest.mark.parametrize("kernel", KERNELS)
def test_wide_elements_in_one_query(cuda_device, kernel):
    """Elements of one head between 2^-30 and 1: the small ones fall below e4m3's range beside the large."""
    m = make([1] * 4, [700] * 4, N1=64, seed=4)
    m["q"] = (m["q"].float() * torch.exp2(-torch.rand(m["q"].shape, device="cuda") * 30)).to(torch.bfloat16)
    check(m, *run(m, kernel=kernel, check_status=True))


@pytest.mark.parametrize("kernel", KERNELS)
def test_scales_far_apart(cuda_device, kernel):
    """Blocks whose scales differ by 2^40, the smallest and the largest scale among them."""
    m = make([1] * 4, [900] * 4, N1=32, seed=5)
    for p in (m["ori"], m["cmp"]):
        n = p[1].numel()
        p[1].copy_(torch.exp2(-torch.arange(n, device="cuda").float() * 40 / max(n - 1, 1) - 8).reshape(p[1].shape))
    check(m, *run(m, kernel=kernel, check_status=True))
    m["ori"][1][0], m["ori"][1][1] = 2.0 ** -60, 2.0 ** -59
    check(m, *run(m, kernel=kernel, check_status=True))


@pytest.mark.parametrize("kernel", KERNELS)
def test_any_scale_value(cuda_device, kernel):
    """Scales need not be powers of two."""
    m = make([1, 2], [900, 400], N1=32, seed=6)
    m["ori"][1].mul_(1.37)
    m["cmp"][1].mul_(0.71)
    check(m, *run(m, kernel=kernel, check_status=True))


@pytest.mark.parametrize("kernel", KERNELS)
def test_sinks(cuda_device, kernel):
    m = make([1, 1], [500, 3], N1=16, seed=7)
    m["sinks"] = torch.tensor([-math.inf, math.inf, 1e4, -1e4, 88.0, -88.0] + [0.5] * 10).cuda()
    check(m, *run(m, kernel=kernel))
    m["sinks"] = None
    check(m, *run(m, kernel=kernel))


@pytest.mark.parametrize("kernel", KERNELS)
def test_rows_that_see_nothing(cuda_device, kernel):
    """Rows before the sequence's start see no key: out 0, lse the sink.  Rows of no request: zeros."""
    m = make([4, 1], [4, 300], N1=16, seed=8)
    m["kv_lens"] = [2, 300]
    m["where"] = ref.positions(m["q_lens"], m["kv_lens"])
    assert m["where"][0][1] < 0
    out, lse = run(m, kernel=kernel, check_status=True)
    check(m, out, lse)
    assert not out[:2].any() and torch.equal(lse[0], m["sinks"])
    out, lse = run(m, kernel=kernel, sinks=None)
    assert torch.equal(lse[:2], torch.full_like(lse[:2], -math.inf)) and not out[:2].any()
    extra = torch.cat([m["q"], m["q"][:3]])  # three rows behind the last sequence
    idx = torch.cat([m["idx"], m["idx"][:3]]).cuda()
    out, lse = run(m, kernel=kernel, q=extra, cmp_sparse_indices=idx, check_status=True)
    assert not out[5:].any() and not lse[5:].any()
    check(m, out[:5], lse[:5])


@pytest.mark.parametrize("kernel", KERNELS)
def test_unmapped_blocks_and_bad_entries(cuda_device, kernel):
    m = make([1, 1, 1], [900, 900, 500], N1=24, seed=9)
    m["ori"][2][0, 6] = -1   # in the window: zero rows, no report
    m["cmp"][2][1, 0] = -1
    check(m, *run(m, kernel=kernel, check_status=True))
    m["ori"][2][2, 3] = 10 ** 6
    m["cmp"][2][0, 1] = -7
    out, lse = run(m, kernel=kernel)
    m["ori"][2][2, 3] = m["cmp"][2][0, 1] = -1
    check(m, out, lse)
    m["ori"][2][2, 3] = 10 ** 6
    with pytest.raises(RuntimeError, match="bad_block"):
        run(m, kernel=kernel, check_status=True)


@pytest.mark.parametrize("kernel", KERNELS)
def test_bad_scales_and_indices(cuda_device, kernel):
    m = make([1, 1], [900, 500], N1=24, seed=10)
    for i, s in enumerate([0.0, -1.0, math.nan, math.inf, 2.0 ** -61]):
        m["ori"][1][i + 4] = s
    m["cmp"][1][0] = math.nan
    out, lse = run(m, kernel=kernel)
    check(m, out, lse)
    with pytest.raises(RuntimeError, match="bad_scale"):
        run(m, kernel=kernel, check_status=True)
    m = make([1, 1], [900, 500], N1=24, seed=10)
    m["idx"][0, 0, 3] = -5
    check(m, *run(m, kernel=kernel))
    with pytest.raises(RuntimeError, match="bad_index"):
        run(m, kernel=kernel, check_status=True)


@pytest.mark.parametrize("kernel", KERNELS)
def test_nan_outside_what_is_visible(cuda_device, kernel):
    """NaN codes in rows that a token does not see (behind its position, before its window) do not reach it."""
    m = make([2, 1], [130, 300], N1=16, seed=11, K=8)
    codes = m["ori"][0].view(torch.uint8)
    for b, row in ((0, 0), (1, 299 - 128), (1, 0)):
        t = m["ori"][2][b]
        codes[int(t[row // 128]), row % 128] = 0x7F if row else 0xFF
    t = m["ori"][2][1]
    codes[int(t[2]), 300 % 128:] = 0x7F
    out, lse = run(m, kernel=kernel, check_status=True)  # token 0 of request 0: window [1, 128]
    assert torch.isfinite(out.float()).all() and torch.isfinite(lse).all()
    check(m, out, lse)


@pytest.mark.parametrize("kernel", KERNELS)
def test_nan_and_infinite_queries_stay_in_their_row(cuda_device, kernel):
    m = make([1, 1], [500, 600], N1=16, seed=12)
    good = run(m, kernel=kernel)
    m["q"][0, 3, 100], m["q"][1, 4, 7] = math.nan, math.inf
    out, lse = run(m, kernel=kernel, check_status=True)
    assert torch.isnan(out[0, 3].float()).all() and torch.isnan(lse[0, 3])
    assert torch.isnan(out[1, 4].float()).all()
    keep = torch.ones((2, 16), dtype=torch.bool, device="cuda")
    keep[0, 3] = keep[1, 4] = False
    assert torch.equal(out[keep], good[0][keep]) and torch.equal(lse[keep], good[1][keep])


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("scenario", [1, 2, 3])
def test_bsnd(cuda_device, scenario, kernel):
    S, act, seq = 3, [3, 1, 0, 2], [400, 5, 77, 1000]
    m = make([S] * 4, [max(s, S) for s in seq], N1=16, scenario=scenario, seed=13, K=128)
    where = [(b, seq[b] - act[b] + s) if s < act[b] else None for b in range(4) for s in range(S)]
    if scenario == 3:
        for t, w in enumerate(where):  # indices within the token's own limit
            if w is not None:
                lim = (w[1] + 1) // 4
                row = m["idx"][t, 0].numpy()
                m["idx"][t, 0] = torch.from_numpy(np.where(row >= lim, lim + 1, row))
    cu = torch.tensor([0] + list(np.cumsum(act)), dtype=torch.int32).cuda()
    kw = dict(cu_seqlens_q=cu, seqused_kv=torch.tensor(seq, dtype=torch.int32).cuda(), layout_q="BSND", kernel=kernel, check_status=True)
    if scenario == 3:
        kw["cmp_sparse_indices"] = m["idx"].cuda().reshape(4, S, 1, -1)
    out, lse = run(m, q=m["q"].reshape(4, S, 16, 576), **kw)
    assert out.shape == (4, S, 16, 512) and lse.shape == (4, S, 16)
    check(m, out.reshape(12, 16, 512), lse.reshape(12, 16), where=where)


def test_outputs_views_and_orders(cuda_device):
    """Caller-owned outputs (also inside a vector), a permuted q, int64 indices and tables, no lse."""
    m = make([1, 2], [700, 900], N1=32, seed=14)
    want, want_lse = run(m)
    check(m, want, want_lse)
    buf = torch.empty(3 * 32 * 512 + 3, dtype=torch.bfloat16, device="cuda")
    out, lse_out = buf[3:].view(3, 32, 512), torch.empty((3, 32), device="cuda")
    got, lse = run(m, out=out, lse_out=lse_out, q=m["q"].transpose(0, 1).contiguous().transpose(0, 1),
                   cmp_sparse_indices=m["idx"].cuda().long(), ori_block_table=torch.from_numpy(m["ori"][2]).cuda().long())
    assert got.data_ptr() == out.data_ptr() and lse.data_ptr() == lse_out.data_ptr()
    assert torch.equal(got, want) and torch.equal(lse, want_lse)
    assert torch.equal(run(m, return_softmax_lse=False), want)


def test_no_tokens(cuda_device):
    m = make([1], [700], N1=32, seed=14)
    out, lse = run(m, q=m["q"][:0], cu_seqlens_q=torch.zeros(2, dtype=torch.int32).cuda(), cmp_sparse_indices=m["idx"].cuda()[:0],
                   check_status=True)
    assert out.shape == (0, 32, 512) and lse.shape == (0, 32)


@pytest.mark.parametrize("kernel", KERNELS)
def test_same_bits_again(cuda_device, kernel):
    for lens in ([1] * 3, [1] * 90):
        m = make(lens, [4000 + 9 * i for i in range(len(lens))], N1=128, K=1500, seed=15)
        a, b = run(m, kernel=kernel), run(m, kernel=kernel)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_two_calls_at_once(cuda_device):
    """Calls on two streams have workspaces of their own."""
    ms = [make([1] * 20, [2000 + 7 * i for i in range(20)], N1=64, K=700, seed=s) for s in (16, 17)]
    want = [run(m) for m in ms]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ms]
    got = [[], []]
    for _ in range(5):
        for i, m in enumerate(ms):
            with torch.cuda.stream(streams[i]):
                got[i].append(run(m))
    torch.cuda.synchronize()
    for i in range(2):
        for o, l in got[i]:
            assert torch.equal(o, want[i][0]) and torch.equal(l, want[i][1])


def test_two_graphs_at_once(cuda_device):
    """Captured calls on two streams, replayed together: a split plan and one of whole tokens."""
    ms = [make([1] * n, [1900 + 7 * i for i in range(n)], N1=64, K=500, seed=s) for n, s in ((5, 22), (80, 23))]
    held = [kwargs(m) for m in ms]
    want = [run(m) for m in ms]
    torch.cuda.synchronize()
    graphs, got, streams = [], [], [torch.cuda.Stream() for _ in ms]
    for m, kw in zip(ms, held):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            got.append(sparse_attn_sharedkv_fp8(m["q"], **kw))
    for _ in range(6):
        for s, gr in zip(streams, graphs):
            with torch.cuda.stream(s):
                gr.replay()
    torch.cuda.synchronize()
    for (o, l), (wo, wl) in zip(got, want):
        assert torch.equal(o, wo) and torch.equal(l, wl)


@pytest.mark.parametrize("kernel", KERNELS)
def test_widest_arguments(cuda_device, kernel):
    """A window, first positions or a ratio past every position say "all" or "none", however large."""
    m = make([2, 1], [300, 900], N1=20, K=60, first=3, seed=24)
    for small, wide in ((dict(ori_win_left=5000), dict(ori_win_left=2**40)), (dict(ori_first=5000), dict(ori_first=2**35)),
                        (dict(cmp_ratio=5000), dict(cmp_ratio=2**33 + 4))):
        a, b = run(m, kernel=kernel, **small), run(m, kernel=kernel, **wide)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def draw(seed):
    rng = np.random.default_rng(seed)
    B = int(2 ** rng.uniform(0, 4))
    new = [int(rng.integers(0, 4)) for _ in range(B - 1)] + [1]
    kv = [max(int(2 ** rng.uniform(0, 12)), n) for n in new]
    scenario = int(rng.integers(1, 4))
    return make(new, kv, N1=int(rng.integers(1, 129)), D=int(rng.choice([512, 576])), K=int(rng.integers(1, 900)), scenario=scenario,
                ratio=int(rng.choice([2, 4, 7, 128])), win_left=int(rng.integers(0, 700)), first=int(rng.integers(0, 6)),
                bs=int(rng.choice([1, 16, 48, 64, 128])), skips=scenario == 3 and seed % 2 == 0, seed=seed)


@pytest.mark.parametrize("seed", range(100, 112))
def test_drawn(cuda_device, seed):
    m = draw(seed)
    check(m, *run(m, check_status=True), tokens=range(min(len(m["where"]), 10)))


@pytest.mark.parametrize("N1", [1, 31, 33, 64, 65, 96, 97])
def test_short_units_of_few_heads(cuda_device, N1):
    """Many tokens of one or two tiles each: warps without heads must keep the others' pace."""
    m = make([1] * 400, [1 + 7 * (i % 23) for i in range(400)], N1=N1, scenario=1, win_left=150, seed=N1)
    out, lse = run(m, kernel="tc", check_status=True)
    check(m, out, lse, tokens=list(range(0, 400, 37)))
    # every row against the other kernel: values below 4 are rounded twice (2^-6 each), and the weights differ
    # by 2^-8 at most; a score of magnitudes up to 100 is off by 36 * 2^-22 of them on either side
    simt = run(m, kernel="simt")
    assert torch.isfinite(out).all() and (out.float() - simt[0].float()).abs().max() < 0.05
    assert (lse - simt[1]).abs().max() < 1e-3


@pytest.mark.parametrize("kernel", KERNELS)
def test_rows_past_32_bits(cuda_device, kernel):
    """Blocks whose rows lie more than 2^32 bytes into the pool, written and read."""
    D, bs, blocks = 576, 128, 2 ** 32 // (576 * 128) + 40
    cache = torch.zeros((blocks, bs, 1, D), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    scale = torch.ones((blocks, 1), device="cuda")
    m = make([300], [300], N1=24, scenario=1, seed=25)
    kv = torch.randn((300, D), generator=torch.Generator().manual_seed(25)).to(torch.bfloat16).cuda()
    table = np.array([[blocks - 1, blocks - 7, blocks - 2]], np.int32)
    call = dict(cu_seqlens_q=torch.tensor([0, 300], dtype=torch.int32).cuda(), seqused_kv=torch.tensor([300], dtype=torch.int32).cuda())
    sharedkv_cache_append(kv, cache=cache, cache_scale=scale, block_table=torch.from_numpy(table).cuda(), check_status=True, **call)
    got = ref.gather(cache[:, :, 0], scale, table[0], list(range(300))).cpu()
    step = scale[:, 0].double().cpu()[torch.from_numpy(table[0]).long()[torch.arange(300) // bs]]
    x = kv.double().cpu()
    assert ((got - x).abs() <= 2.0 ** -4 * x.abs() + 2.0 ** -10 * step[:, None]).all()
    m["ori"] = (cache, scale, table)
    check(m, *run(m, kernel=kernel, check_status=True), tokens=[0, 1, 127, 128, 299])


@pytest.mark.parametrize("tokens", [2, 90])
def test_graph(cuda_device, tokens):
    """A captured call replayed on new queries, indices, lengths and tables."""
    ms = [make([1] * tokens, [1500 + 3 * i for i in range(tokens)], N1=32, K=300, seed=s) for s in (18, 19)]
    ms[1]["kv_lens"] = [1500 + 3 * i - 40 for i in range(tokens)]
    ms[1]["where"] = ref.positions(ms[1]["q_lens"], ms[1]["kv_lens"])
    run(ms[0])
    torch.cuda.synchronize()
    names = ("ori_kv", "ori_kv_scale", "ori_block_table", "cmp_kv", "cmp_kv_scale", "cmp_block_table", "cmp_sparse_indices", "seqused_kv", "sinks")
    q, held = ms[0]["q"].clone(), kwargs(ms[0])
    held.update({n: held[n].clone() for n in names})
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = sparse_attn_sharedkv_fp8(q, **held)
    for m in ms + ms[:1]:
        q.copy_(m["q"])
        for n in names:
            d, s = held[n], kwargs(m)[n]
            if n in ("ori_kv", "cmp_kv"):
                d, s = d.view(torch.uint8), s.view(torch.uint8)
            d.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        check(m, out, lse, tokens=range(min(tokens, 12)))


def test_compiled(cuda_device):
    m = make([1, 2], [700, 900], N1=32, seed=20)
    want = run(m)
    f = torch.compile(lambda q: sparse_attn_sharedkv_fp8(q, **kw), fullgraph=True, backend="aot_eager")
    kw = kwargs(m)
    out, lse = f(m["q"])
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])


def test_refusals(cuda_device):
    m = make([1, 2], [700, 900], N1=32, seed=21)
    bad = [
        (dict(ori_kv=m["ori"][0].to(torch.bfloat16)), "float8_e4m3fn"),
        (dict(ori_kv_scale=m["ori"][1][:-1]), "one entry per block"),
        (dict(ori_kv_scale=m["ori"][1].double()), "float32"),
        (dict(ori_kv_scale=m["ori"][1].cpu()), "must be on"),
        (dict(ori_kv=m["ori"][0].cpu()), "must be on"),
        (dict(ori_kv=m["ori"][0][:, ::2]), "contiguous"),
        (dict(cmp_kv=m["cmp"][0].view(torch.uint8)), "float8_e4m3fn"),
        (dict(cmp_block_table=None), "cmp_block_table"),
        (dict(cmp_sparse_indices=m["idx"].cuda()[:2]), "per token"),
        (dict(ori_block_table=torch.zeros((1, 3), dtype=torch.int32, device="cuda")), "ori_block_table"),
        (dict(seqused_kv=torch.zeros(1, dtype=torch.int32, device="cuda")), "seqused_kv"),
        (dict(sinks=m["sinks"][:5]), "sinks"),
        (dict(ori_first=-1), ">= 0"),
        (dict(out=torch.empty((3, 32, 512), device="cuda")), "out must be"),
        (dict(lse_out=torch.empty((3, 31), device="cuda")), "lse_out must be"),
        (dict(q=m["q"].float()), "unsupported torch dtype"),
        (dict(q=m["q"].clone().requires_grad_()), "no backward"),
        (dict(cmp_kv=None, cmp_kv_scale=None), "goes with cmp_kv"),
    ]
    for kw, text in bad:
        with pytest.raises(ValueError, match=text):
            run(m, **kw)
    with pytest.raises(RuntimeError, match="unsupported"):
        run(m, kernel="tc", v_head_dim=256)
    with torch.no_grad():
        run(m, q=m["q"].clone().requires_grad_())


@pytest.mark.parametrize("kernel", KERNELS)
def test_append_then_attend(cuda_device, kernel):
    """A prompt in two chunks, then decode steps: rows (full and compressed) appended with their rotation,
    queries rotated in the same call, attention over what was written.  The attention is held to the
    cache's contents, and the cache's contents to the rows that were put in."""
    D, N1, bs, ratio, K, B = 576, 24, 64, 4, 90, 3
    g = torch.Generator().manual_seed(21)
    rope = rope_table(600, 64)
    lens = [0] * B
    table = torch.randperm(B * 8, generator=g).to(torch.int32).reshape(B, 8)
    cmp_table = torch.randperm(B * 3, generator=g).to(torch.int32).reshape(B, 3)
    ori = torch.zeros((B * 8, bs, 1, D), device="cuda").to(torch.float8_e4m3fn)
    cmp_ = torch.zeros((B * 3, bs, 1, D), device="cuda").to(torch.float8_e4m3fn)
    ori_s, cmp_s = torch.ones((B * 8, 1), device="cuda"), torch.ones((B * 3, 1), device="cuda")
    rows = [[] for _ in range(B)]
    for new in ([200, 13, 0], [60, 1, 300], [1, 1, 1], [1, 1, 1], [2, 2, 2]):
        size = 0.5 if sum(new) > 3 else 0.9  # the decode rows raise the blocks' scales
        old, lens = lens, [a + n for a, n in zip(lens, new)]
        T = sum(new)
        kv = (torch.randn((T, D), generator=g) * size).to(torch.bfloat16)
        q = torch.randn((T, N1, D), generator=g).to(torch.bfloat16)
        cu = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32).cuda()
        seq = torch.tensor(lens, dtype=torch.int32).cuda()
        qr = sharedkv_cache_append(kv.cuda(), cache=ori, cache_scale=ori_s, block_table=table.cuda(), cu_seqlens_q=cu, seqused_kv=seq,
                                   rope_table=rope, q=q.cuda(), check_status=True)
        c_new = [n // ratio - o // ratio for n, o in zip(lens, old)]
        if sum(c_new):
            ckv = (torch.randn((sum(c_new), D), generator=g) * size).to(torch.bfloat16).cuda()
            sharedkv_cache_append(ckv, cache=cmp_, cache_scale=cmp_s, block_table=cmp_table.cuda(),
                                  cu_seqlens_q=torch.tensor([0] + list(np.cumsum(c_new)), dtype=torch.int32).cuda(),
                                  seqused_kv=torch.tensor([n // ratio for n in lens], dtype=torch.int32).cuda(), rope_table=rope,
                                  rope_step=ratio, check_status=True)
        where = ref.positions(new, lens)
        idx = torch.full((T, 1, K), -1, dtype=torch.int32)
        for t, (b, p) in enumerate(where):
            take = torch.randperm((p + 1) // ratio, generator=g)[:K]
            idx[t, 0, :len(take)] = take.to(torch.int32)
            rows[b].append(ref.rotate(kv[t].double(), rope[p].double().cpu(), True))
        m = dict(case=dict(win_left=127, first=2, ratio=ratio, scenario=3), q_lens=new, kv_lens=lens, Dv=512, src="bf16", q=qr, where=where,
                 ori=(ori, ori_s, table.numpy()), cmp=(cmp_, cmp_s, cmp_table.numpy()), idx=idx, sinks=torch.zeros(N1).cuda(), scale=D ** -0.5)
        check(m, *run(m, kernel=kernel, check_status=True), tokens=list(range(0, T, max(1, T // 12))) + [T - 1])
    for b in range(B):  # a value is off by half a step of the scale it was rounded at, twice at most
        got = ref.gather(ori[:, :, 0], ori_s, table[b].numpy(), list(range(lens[b]))).cpu()
        want = torch.stack(rows[b])
        s = ori_s[:, 0].double().cpu()[table[b].long()[torch.arange(lens[b]) // bs]]
        assert ((got - want).abs() <= 2 * (2.0 ** -4 * want.abs() + 2.0 ** -10 * s[:, None]) + 1e-6).all()
