"""sharedkv_cache_append on the GPU against the plain 64-bit implementation."""

import math

import numpy as np
import pytest
import torch

from dsv4_planb_b200.api import sparse_attn_sharedkv
from dsv4_planb_b200.cache import rope_table, sharedkv_cache_append
from tests import _cache_ref as ref

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp8": torch.float8_e4m3fn}
HALF_STEP = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp8": 2.0 ** -4}
TINY = {"bf16": 2.0 ** -134, "fp16": 2.0 ** -25, "fp8": 2.0 ** -10}  # half the step below the smallest normal value


def make(q_lens, kv_lens, *, D=576, bs=128, pool="fp8", src="bf16", heads=0, seed=0, extra_blocks=2, size=0.5, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    rng = np.random.default_rng(seed)
    per = [max(0, math.ceil(n / bs)) for n in kv_lens]
    blocks = sum(per) + extra_blocks
    phys = rng.permutation(blocks).astype(np.int32)
    table = np.full((len(q_lens), max(max(per, default=0), 1)), -1, np.int32)
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = phys[at:at + n]
        at += n
    T = sum(q_lens)
    m = dict(bs=bs, q_lens=q_lens, kv_lens=kv_lens, table=torch.from_numpy(table), pool=pool, src=src)
    m["kv"] = (torch.randn((T, D), generator=g) * size).to(TYPES[src])
    m["q"] = (torch.randn((T, heads, D), generator=g) * size).to(TYPES[src]) if heads else None
    raw = torch.randn((blocks, bs, 1, D), generator=g) * size
    if pool == "fp8":
        m["scale"] = torch.exp2(torch.randint(-12, -4, (blocks, 1), generator=g).float())
        m["cache"] = (raw / m["scale"][:, :, None, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    else:
        m["scale"], m["cache"] = None, raw.to(TYPES[pool])
    cu = np.concatenate([[0], np.cumsum(q_lens)]).astype(np.int32)
    m["cu"], m["seq"] = torch.from_numpy(cu), torch.tensor(kv_lens, dtype=torch.int32)
    m["where"] = ref.positions(q_lens, kv_lens)
    return m


def check(m, cache, scale, rope, interleaved=True, step=1, kv=None, where=None):
    """The cache (on the GPU) after one append of m's rows onto m's cache."""
    values = m["cache"].double()[:, :, 0]
    want, want_scale, written = ref.append((m["kv"] if kv is None else kv).double(), values,
                                           None if m["scale"] is None else m["scale"].double()[:, 0],
                                           m["table"].numpy(), m["where"] if where is None else where,
                                           None if rope is None else rope.double().cpu(), interleaved, step)
    got = cache.cpu()
    g = got.double()[:, :, 0]
    if want_scale is not None:
        assert torch.equal(scale.cpu().double().reshape(-1), want_scale)
    raw, old = (x.view(torch.uint8 if m["pool"] == "fp8" else torch.int16) for x in (got, m["cache"]))
    assert torch.equal(raw[:, :, 0][written == 0], old[:, :, 0][written == 0]), "rows that were not written changed"
    again = written == 2  # code * old / new is exact in 32 bits, so its rounding is one nearest-even step
    assert torch.equal(g[again], want[again].float().to(torch.float8_e4m3fn).double())
    new = written == 1
    e, w = g[new], want[new]
    if m["pool"] == "fp8":
        w = w.clamp(-448, 448)
    nan = torch.isnan(w)
    assert torch.equal(nan, torch.isnan(e))
    # one rounding to the cache's type; the rotation adds two products and a sum in 32 bits, at most
    # 3 * 2^-24 of the pair's |a| + |b| <= 2 max |row|
    tol = HALF_STEP[m["pool"]] * w.abs() + TINY[m["pool"]] + 6 * 2.0 ** -24 * w.nan_to_num(0).abs().amax(dim=1, keepdim=True)
    bad = ((e - w).abs() > tol) & ~nan
    assert not bad.any(), f"{int(bad.sum())} values, worst {(e - w)[bad].abs().max()}"
    R = 0 if rope is None else rope.shape[1]
    if m["pool"] != "fp8":  # what is not rotated is copied
        n = w.shape[1] - R
        assert torch.equal(e[:, :n], w[:, :n])


def run(m, rope, **kw):
    cache, scale = m["cache"].cuda(), None if m["scale"] is None else m["scale"].cuda()
    kv = kw.pop("kv", m["kv"].cuda())
    q = sharedkv_cache_append(kv, cache=cache, cache_scale=scale, block_table=m["table"].cuda(), cu_seqlens_q=m["cu"].cuda(),
                              seqused_kv=m["seq"].cuda(), rope_table=rope, **kw)
    return cache, scale, q


LENGTHS = [
    ([1], [1]),
    ([1], [300]),
    ([1, 1, 1], [128, 129, 257]),           # a block's last row, and the next block's first
    ([0, 5, 0, 1, 3], [7, 5, 0, 400, 130]),  # requests without new rows
    ([700, 1, 130], [900, 1, 130]),
    ([128, 256, 127], [128, 300, 255]),      # whole blocks
    ([2] * 70, [2 + 3 * i for i in range(70)]),
    ([2000], [2600]),
    ([1] * 20 + [128], [5] * 20 + [256]),   # a whole block among single rows
]


@pytest.mark.parametrize("pool,src", [("fp8", "bf16"), ("fp8", "fp16"), ("bf16", "bf16"), ("fp16", "fp16")])
@pytest.mark.parametrize("lens", range(len(LENGTHS)))
def test_append_lengths(cuda_device, lens, pool, src):
    q_lens, kv_lens = LENGTHS[lens]
    m = make(q_lens, kv_lens, pool=pool, src=src, seed=lens)
    rope = rope_table(max(kv_lens) + 1, 64)
    check(m, *run(m, rope, check_status=True)[:2], rope)


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("D,bs,R,step", [(512, 16, 64, 1), (576, 48, 64, 4), (16, 1, 16, 1), (1024, 7, 1024, 1), (64, 128, 32, 3)])
@pytest.mark.parametrize("pool", ["fp8", "bf16"])
def test_append_shapes(cuda_device, D, bs, R, step, interleaved, pool):
    m = make([40, 1, 9], [55, 130, 9], D=D, bs=bs, pool=pool, seed=D + bs)
    rope = rope_table(step * 130 + 1, R)
    got = run(m, rope, rope_interleaved=interleaved, rope_step=step, check_status=True)
    check(m, *got[:2], rope, interleaved, step)


@pytest.mark.parametrize("pool", ["fp8", "fp16"])
def test_append_without_rotation(cuda_device, pool):
    m = make([3, 200], [3, 333], pool=pool, src="fp16", seed=3)
    check(m, *run(m, None, check_status=True)[:2], None)


@pytest.mark.parametrize("grow", [1.0, 4.0, 300.0, 0.0])
def test_scale_grows_and_rounds_old_rows(cuda_device, grow):
    """One row at a time into one block: each step against the cache the step before left."""
    rope = rope_table(300, 64)
    m = make([1], [41], seed=11)
    for step in range(3):
        m["kv"] = torch.randn((1, 576), generator=torch.Generator().manual_seed(step)) * 0.5 * grow ** step
        m["kv"] = m["kv"].to(torch.bfloat16)
        cache, scale, _ = run(m, rope, check_status=True)
        check(m, cache, scale, rope)
        m["cache"], m["scale"] = cache.cpu(), scale.cpu()
        m["kv_lens"] = [m["kv_lens"][0] + 1]
        m["seq"] = m["seq"] + 1
        m["where"] = ref.positions([1], m["kv_lens"])


def test_scale_border(cuda_device):
    """448 * 2^k is the largest value of scale 2^k; the next bf16 value above it takes 2^(k + 1)."""
    for top, k in ((448.0, 0), (450.0, 1), (447.0, 0), (1.75, -8), (1.7578125, -7), (3.0e38, 60), (0.0, -60)):
        m = make([1], [1], seed=1)
        m["kv"].zero_()
        m["kv"][0, 5] = -top
        cache, scale, _ = run(m, None, check_status=True)
        assert float(scale[int(m["table"][0, 0])]) == 2.0 ** k
        check(m, cache, scale, None)


def test_infinities_and_nan(cuda_device):
    m = make([4], [4], seed=2)
    m["kv"][1, 3], m["kv"][1, 4], m["kv"][2, 7] = math.inf, -math.inf, math.nan
    cache, scale, _ = run(m, None)
    check(m, cache, scale, None)
    row = cache[int(m["table"][0, 0]), :, 0].float()
    assert row[1, 3] == 448 and row[1, 4] == -448 and torch.isnan(row[2, 7]) and not torch.isnan(row[3]).any()


@pytest.mark.parametrize("pool", ["fp8", "bf16"])
def test_strided_rows_and_padding(cuda_device, pool):
    """kv as a slice of a wider projection; rows behind the last sequence are not written."""
    m = make([3, 0, 66], [70, 0, 140], pool=pool, seed=5)
    T = 69
    wide = torch.randn((T + 5, 2048), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    view = wide[:, 64:64 + 576]
    view[:T] = m["kv"].cuda()
    rope = rope_table(200, 64)
    check(m, *run(m, rope, kv=view, check_status=True)[:2], rope)
    odd = wide[:, 3:3 + 576]  # starts inside a 16-byte vector: copied
    check(m, *run(m, rope, kv=odd, check_status=True)[:2], rope, kv=odd[:T].cpu())


@pytest.mark.parametrize("pool", ["fp8", "bf16"])
def test_bsnd(cuda_device, pool):
    """BSND with fewer new rows than S per request."""
    S, act = 6, [6, 2, 0, 5]
    seq = [300, 2, 9, 131]
    m = make([S] * 4, [max(s, S) for s in seq], pool=pool, heads=3, seed=6)
    m["seq"] = torch.tensor(seq, dtype=torch.int32)
    where = [(b, seq[b] - act[b] + s) if s < act[b] else None for b in range(4) for s in range(S)]
    cu = torch.tensor([0] + list(np.cumsum(act)), dtype=torch.int32)
    rope = rope_table(400, 64)
    cache, scale = m["cache"].cuda(), None if m["scale"] is None else m["scale"].cuda()
    q = m["q"].cuda().reshape(4, S, 3, 576)
    q2 = sharedkv_cache_append(m["kv"].cuda().reshape(4, S, 1, 576), cache=cache, cache_scale=scale, block_table=m["table"].cuda(),
                               cu_seqlens_q=cu.cuda(), seqused_kv=m["seq"].cuda(), rope_table=rope, layout_q="BSND", q=q,
                               check_status=True)
    check(m, cache, scale, rope, where=where)
    assert torch.equal(q, m["q"].cuda().reshape(q.shape))
    check_q(m["q"], q2.reshape(24, 3, 576), rope, where, True, 1)


def check_q(q, got, rope, where, interleaved, step):
    name = {torch.bfloat16: "bf16", torch.float16: "fp16"}[q.dtype]
    for t, w in enumerate(where):
        if w is None:
            assert torch.equal(got[t].cpu(), q[t])
            continue
        x = ref.rotate(q[t].double(), rope[w[1] * step].double().cpu(), interleaved)
        n = q.shape[2] - rope.shape[1]
        assert torch.equal(got[t, :, :n].cpu(), q[t, :, :n])
        tol = HALF_STEP[name] * x.abs() + TINY[name] + 6 * 2.0 ** -24 * x.abs().amax(dim=1, keepdim=True)
        assert ((got[t].cpu().double() - x).abs() <= tol).all()


@pytest.mark.parametrize("heads", [1, 16, 17, 128])
@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("pool", ["fp8", "bf16"])
def test_queries(cuda_device, heads, interleaved, pool):
    m = make([1, 4, 2], [77, 4, 500], pool=pool, heads=heads, seed=heads)
    rope = rope_table(501, 64)
    cache, scale, q = run(m, rope, q=m["q"].cuda(), rope_interleaved=interleaved, check_status=True)
    check(m, cache, scale, rope, interleaved)
    check_q(m["q"], q, rope, m["where"], interleaved, 1)
    mine = m["q"].cuda()
    assert run(m, rope, q=mine, q_out=mine, rope_interleaved=interleaved)[2] is mine
    assert torch.equal(mine, q)


@pytest.mark.parametrize("pool", ["fp8", "bf16"])
def test_skipped_rows(cuda_device, pool):
    """Unmapped and bad blocks, positions past the table and the angles, positions before 0."""
    m = make([3, 2, 1, 5], [130, 5, 10, 3], pool=pool, seed=8)  # request 3: 5 new rows, length 3
    m["table"][0, 1], m["table"][1, 0] = -1, 10 ** 6
    rope = rope_table(130, 64)
    check(m, *run(m, rope)[:2], rope)
    with pytest.raises(RuntimeError, match="bad_block"):
        run(m, rope, check_status=True)
    m = make([2], [131], pool=pool, seed=9)  # the last position lies past the angles
    check(m, *run(m, rope)[:2], rope)
    with pytest.raises(RuntimeError, match="bad_position"):
        run(m, rope, check_status=True)
    m["table"] = m["table"][:, :1].contiguous()  # and past the block table
    check(m, *run(m, rope)[:2], rope)


@pytest.mark.parametrize("q_lens,kv_lens", [([3], [130]), ([1], [200]), ([600], [700])])
def test_blocks_past_the_angles_stay(cuda_device, q_lens, kv_lens):
    """A block none of whose rows has angles keeps its contents and its scale."""
    m = make(q_lens, kv_lens, seed=10)
    rope = rope_table(128, 64)
    cache, scale, _ = run(m, rope)
    check(m, cache, scale, rope)
    phys = int(m["table"][0, 1])
    assert torch.equal(cache[phys].cpu().view(torch.uint8), m["cache"][phys].view(torch.uint8))
    assert torch.equal(scale.cpu().reshape(-1)[phys], m["scale"].reshape(-1)[phys])


@pytest.mark.parametrize("old", [0.0, -1.0, math.nan, math.inf])
def test_block_without_scale(cuda_device, old):
    m = make([1], [3], seed=4)
    m["scale"][int(m["table"][0, 0])] = old
    cache, scale, _ = run(m, None)
    check(m, cache, scale, None)
    with pytest.raises(RuntimeError, match="bad_scale"):
        run(m, None, check_status=True)


@pytest.mark.parametrize("q_lens", [[1] * 1500, [0, 3] * 400 + [700], [40] * 33, [0] * 40 + [1] + [0] * 70], ids=["1500x1", "gaps", "33x40", "one"])
def test_many_requests(cuda_device, q_lens):
    """Every request's runs are found among many, with requests that bring nothing between them."""
    rng = np.random.default_rng(31)
    m = make(q_lens, [n + int(rng.integers(0, 150)) for n in q_lens], D=64, bs=16, seed=31)
    rope = rope_table(900, 64)
    check(m, *run(m, rope, check_status=True)[:2], rope)


@pytest.mark.parametrize("pool", ["fp8", "bf16"])
def test_rows_before_the_first_request(cuda_device, pool):
    """Flat rows in front of the first request and behind the last belong to none."""
    m = make([60, 2], [100, 300], bs=16, pool=pool, seed=32)
    rope, front = rope_table(300, 64), 35
    kv = torch.full((front + 62 + 9, m["kv"].shape[1]), 7.0, dtype=m["kv"].dtype)
    kv[front:front + 62] = m["kv"]
    m["cu"] += front
    check(m, *run(m, rope, kv=kv.cuda(), check_status=True)[:2], rope)


def test_no_rows(cuda_device):
    m = make([0, 0], [4, 0], seed=4)
    check(m, *run(m, rope_table(8, 64), check_status=True)[:2], None)


def test_other_stream_and_graph(cuda_device):
    """A captured append, replayed on new rows, lengths and tables."""
    m = make([1] * 9, [100 + i for i in range(9)], heads=4, seed=12)
    rope = rope_table(400, 64)
    kv, q, seq = m["kv"].cuda(), m["q"].cuda(), m["seq"].cuda()
    cache, scale, table, cu = m["cache"].cuda(), m["scale"].cuda(), m["table"].cuda(), m["cu"].cuda()

    def step():
        return sharedkv_cache_append(kv, cache=cache, cache_scale=scale, block_table=table, cu_seqlens_q=cu, seqused_kv=seq,
                                     rope_table=rope, q=q)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    check(m, cache, scale, rope)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    m["cache"], m["scale"] = cache.cpu(), scale.cpu()
    m["kv"] = (torch.randn(m["kv"].shape, generator=torch.Generator().manual_seed(5)) * 3).to(torch.bfloat16)
    m["where"] = [(b, p + 1) for b, p in m["where"]]
    kv.copy_(m["kv"])
    seq.add_(1)
    graph.replay()
    torch.cuda.synchronize()
    check(m, cache, scale, rope)
    check_q(m["q"], out, rope, m["where"], True, 1)


def test_rows_past_32_bits(cuda_device):
    """16-bit rows more than 2^32 bytes into the pool."""
    D, bs, blocks = 512, 64, 2 ** 32 // (512 * 64 * 2) + 5
    cache = torch.zeros((blocks, bs, 1, D), dtype=torch.bfloat16, device="cuda")
    kv = torch.randn((90, D), generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).cuda()
    table = torch.tensor([[blocks - 2, blocks - 1]], dtype=torch.int32).cuda()
    sharedkv_cache_append(kv, cache=cache, block_table=table, cu_seqlens_q=torch.tensor([0, 90], dtype=torch.int32).cuda(),
                          seqused_kv=torch.tensor([100], dtype=torch.int32).cuda(), check_status=True)
    assert torch.equal(cache[blocks - 2:].reshape(2 * bs, D)[10:100], kv)
    assert not cache[:blocks - 2].any()


def test_rows_read_by_the_16_bit_attention(cuda_device):
    """Rows appended in two calls are what the attention reads: the same bits laid out by hand in another
    order of blocks give the same result."""
    D, bs, lens = 512, 64, [150, 70]
    g = torch.Generator().manual_seed(4)
    rope = rope_table(200, 64)
    cache = torch.zeros((8, bs, 1, D), dtype=torch.bfloat16, device="cuda")
    table = torch.tensor([[5, 0, 3], [2, 7, -1]], dtype=torch.int32)
    for new, done in (([140, 1], [140, 1]), ([10, 69], lens)):
        cu = torch.tensor([0, new[0], sum(new)], dtype=torch.int32).cuda()
        seq = torch.tensor(done, dtype=torch.int32).cuda()
        kv = torch.randn((sum(new), D), generator=g).to(torch.bfloat16).cuda()
        q = sharedkv_cache_append(kv, cache=cache, block_table=table.cuda(), cu_seqlens_q=cu, seqused_kv=seq, rope_table=rope,
                                  q=torch.randn((sum(new), 16, D), generator=g).to(torch.bfloat16).cuda())
    other = torch.tensor([[1, 6, 4], [3, 2, -1]], dtype=torch.int32)
    moved = torch.zeros_like(cache)
    for b, n in enumerate(lens):
        for i in range((n + bs - 1) // bs):
            moved[other[b, i]] = cache[table[b, i]]
    outs = [sparse_attn_sharedkv(q, ori_kv=c, ori_block_table=t.cuda(), cu_seqlens_q=cu, seqused_kv=seq, sinks=torch.zeros(16).cuda(),
                                 softmax_scale=D ** -0.5, v_head_dim=D) for c, t in ((cache, table), (moved, other))]
    outs = [o[0] if isinstance(o, tuple) else o for o in outs]
    assert outs[0].abs().sum() > 0 and torch.equal(*outs)


def test_compiled(cuda_device):
    m = make([1, 3], [9, 200], heads=2, seed=13)
    rope = rope_table(300, 64)
    f = torch.compile(lambda kv, cache, scale, q: sharedkv_cache_append(
        kv, cache=cache, cache_scale=scale, block_table=table, cu_seqlens_q=cu, seqused_kv=seq, rope_table=rope, q=q),
        fullgraph=True, backend="aot_eager")
    table, cu, seq = m["table"].cuda(), m["cu"].cuda(), m["seq"].cuda()
    cache, scale = m["cache"].cuda(), m["scale"].cuda()
    q = f(m["kv"].cuda(), cache, scale, m["q"].cuda())
    check(m, cache, scale, rope)
    check_q(m["q"], q, rope, m["where"], True, 1)


def test_rope_table(cuda_device):
    t = rope_table(1 << 17, 64, base=500.0).cpu().double()
    i = np.arange(0, 64, 2) / 64
    p = (1 << 17) - 1
    ang = p * 500.0 ** -i
    want = torch.from_numpy(np.concatenate([np.cos(ang), np.sin(ang)]))
    assert (t[p] - want).abs().max() <= 2.0 ** -24 + 1e-9  # one rounding; 64-bit angles are off by 2^17 * 2^-51
    assert torch.equal(t[0], torch.cat([torch.ones(32), torch.zeros(32)]).double())


def test_refusals(cuda_device):
    m = make([1, 3], [9, 200], heads=2, seed=14)
    rope = rope_table(300, 64)
    q = m["q"].cuda()

    def call(**kw):
        a = dict(cache=m["cache"].cuda(), cache_scale=m["scale"].cuda(), block_table=m["table"].cuda(), cu_seqlens_q=m["cu"].cuda(),
                 seqused_kv=m["seq"].cuda(), rope_table=rope, q=q)
        kv = kw.pop("kv", m["kv"].cuda())
        a.update(kw)
        return sharedkv_cache_append(kv, **a)

    bad = [
        (dict(kv=m["kv"].float().cuda()), "bfloat16 or float16"),
        (dict(kv=m["kv"]), "must be on"),
        (dict(kv=m["kv"].cuda()[:, :512]), "one row of 576"),
        (dict(cache=m["cache"].cuda()[:, ::2]), "contiguous"),
        (dict(cache=m["cache"].cuda().float()), "type of kv"),
        (dict(cache=m["cache"].cuda().to(torch.bfloat16)), "float8_e4m3fn cache only"),
        (dict(cache=m["cache"].cuda()[:, :, 0]), "block_size"),
        (dict(cache_scale=None), "cache_scale"),
        (dict(cache_scale=m["scale"].cuda()[1:]), "one entry per block"),
        (dict(block_table=m["table"].cuda()[:1]), "block_table"),
        (dict(seqused_kv=m["seq"].cuda()[:1]), "seqused_kv"),
        (dict(rope_table=rope.double()), "float32"),
        (dict(rope_table=rope_table(300, 24)), "multiple of 16"),
        (dict(rope_table=rope.cpu()), "must be on"),
        (dict(rope_table=torch.empty(300 * 64 + 1, device="cuda")[1:].view(300, 64)), "16-byte"),
        (dict(rope_step=0), "rope_step"),
        (dict(q=q[:1]), "per token"),
        (dict(q=q.half()), "kv's type"),
        (dict(q_out=torch.empty((4, 2, 577), dtype=q.dtype, device="cuda")[:, :, :576]), "contiguous"),
        (dict(q=None, q_out=q), "goes with q"),
        (dict(kv=m["kv"].cuda().requires_grad_()), "no backward"),
    ]
    for kw, text in bad:
        with pytest.raises(ValueError, match=text):
            call(**kw)
    wide = torch.zeros((5, 2, 576), dtype=q.dtype, device="cuda")
    with pytest.raises(ValueError, match="share nothing"):
        call(q=wide[:4], q_out=wide[1:])
    with pytest.raises(AssertionError, match="cu_seqlens_q"):
        call(cu_seqlens_q=None)
