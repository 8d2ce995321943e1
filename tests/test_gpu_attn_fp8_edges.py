"""sparse_attn_sharedkv_fp8 where index rows end at a chunk's border, maxima rise far, and one key dominates."""

import math

import pytest
import torch

from tests import _cache_ref as ref
from tests.test_gpu_attn_fp8 import HALF_STEP, KERNELS, SHAPES, check, ident, make, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kernel", KERNELS)
def test_index_rows_that_begin_with_the_stop(cuda_device, kernel):
    """Thousands of tokens see compressed rows by position, and every second one names none: it gets what the
    window alone gives, to the bit."""
    m = make([4000], [4400], N1=8, K=300, seed=40)
    m["idx"][::2, 0, 0] = -1
    window = make([4000], [4400], N1=8, K=300, scenario=1, seed=40)
    window.update(q=m["q"], ori=m["ori"], sinks=m["sinks"])
    want = run(window, kernel=kernel, check_status=True)
    for _ in range(5):
        out, lse = run(m, kernel=kernel, check_status=True)
        assert torch.equal(out[::2], want[0][::2]) and torch.equal(lse[::2], want[1][::2])
    check(m, out, lse, tokens=[0, 1, 2, 3, 1999, 2000, 3998, 3999])


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("K", [2048, 2049, 4096, 5000])
def test_long_index_rows(cuda_device, K, kernel):
    """Rows of more than 2048 indices, with their stop in front of, at and behind every 2048th."""
    stops = [s for s in (None, 0, 1, 2047, 2048, 2049, 4095, 4096, 4097, K - 1) if s is None or s < K]
    m = make([len(stops)] * 12, [21000 + i for i in range(12)], N1=8, K=K, seed=K)
    for t in range(len(m["where"])):
        s = stops[t % len(stops)]
        if s is not None:
            m["idx"][t, 0, s] = -1
    out, lse = run(m, kernel=kernel, check_status=True)
    check(m, out, lse, tokens=range(3 * len(stops)))
    for _ in range(5):
        again = run(m, kernel=kernel)
        assert torch.equal(again[0], out) and torch.equal(again[1], lse)


@pytest.mark.parametrize("kernel", KERNELS)
def test_long_index_rows_in_pieces(cuda_device, kernel):
    """Few tokens, which run in pieces: the pieces behind an early stop are empty."""
    m = make([3, 2], [21000, 30000], N1=40, K=5000, seed=45)
    for t, s in enumerate((0, 5, 2048, 4096)):
        m["idx"][t, 0, s] = -1
    check(m, *run(m, kernel=kernel, check_status=True))


def far_rise(tokens, N1, rise, seed):
    """Every head's scores lie near 0 except for one late key, which all heads meet at about ``rise`` nats."""
    m = make([1] * tokens, [900] * tokens, N1=N1, scenario=1, win_left=799, seed=seed)
    g = torch.Generator().manual_seed(seed)
    pattern = torch.randint(0, 2, (576,), generator=g).float() * 2 - 1
    m["q"] = (pattern + 0.05 * torch.randn((tokens, N1, 576), generator=g)).to(torch.bfloat16).cuda()
    codes, scale, table = m["ori"]
    scale.fill_(2.0 ** -4)
    codes.copy_((torch.randn(codes.shape, generator=g) * 8).to(codes.dtype).cuda())  # values of size 0.5
    for b in range(tokens):  # position 700: several tiles behind the window's start at 100, not in its last one
        row = pattern * (rise / 24 / 2.0 ** -4)  # q . k / sqrt(576) = rise
        codes[int(table[b, 700 // 128]), 700 % 128, 0] = row.to(codes.dtype).cuda()
    return m


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("N1", [1, 16, 32, 33, 128])
@pytest.mark.parametrize("rise", [60, 110, 250, 600])
def test_one_late_key_far_above(cuda_device, rise, N1, kernel):
    """A maximum that rises by more than 104 nats: the factor of what came before it is 0 in 32 bits."""
    m = far_rise(40, N1, rise, seed=41)
    check(m, *run(m, kernel=kernel, check_status=True), tokens=[0, 7, 39])


# Error of a tensor-core weight: rounded to fp16 (2^-11 of it), then split into an e4m3 term (nearest) and two e5m2
# terms (cut). Where the first is normal it leaves at most 2^-4 of the weight's power of two, the second less than
# 2^-7, the third less than 2^-10. Where the first is subnormal (weights below 2^-6) they leave 2^-10, 2^-13 and 2^-16,
# the smallest step of e5m2. A row's largest weight ends at 2^6 or more (the frame follows rises above 2^2.75, the top
# is 2^8.75), so 2^-16 is 2^-22 of it.
WEIGHT, WEIGHT_OF_TOP = 2.0 ** -10 + 2.0 ** -11 + 2.0 ** -20, 2.0 ** -22


def check_weights(m, out, lse, tokens=None):
    """As ``check``, with the bounds above for the weights."""
    for t in range(len(m["where"])) if tokens is None else tokens:
        b, p = m["where"][t]
        o, l, spread, top, reach = ref.attend(
            m["case"], m["q"][t], p, b, (m["ori"][0][:, :, 0], m["ori"][1], m["ori"][2][b]),
            None if m["cmp"] is None else (m["cmp"][0][:, :, 0], m["cmp"][1], m["cmp"][2][b]),
            None if m["idx"] is None else m["idx"][t, 0].numpy(), m["sinks"], m["scale"], m["Dv"])
        d = (36 * 2.0 ** -22 + 3 * 2.0 ** -24) * reach
        assert ((lse[t].double() - l).abs() <= d + 2.0 ** -20 + 2.0 ** -22 * l.abs()).all()
        tol = (HALF_STEP[m["src"]] * o.abs() + 2.0 ** -24 + spread * (2 * d + 2.0 ** -20 + WEIGHT + 70 * 2.0 ** -22)[:, None]
               + WEIGHT_OF_TOP * top)
        err = (out[t].double() - o).abs()
        assert (err <= tol).all(), (t, float((err - tol).max()), float((err.norm(dim=1) / o.norm(dim=1)).max()))


def one_key_dominates(tokens, N1, mass, spread, mean, seed):
    """The first position, which stays visible, takes ``mass`` of the softmax and has a small value; 2176 other keys
    share the rest, with scores that differ by about ``spread`` nats and values with a common mean."""
    K = 2048
    m = make([1] * tokens, [9000] * tokens, N1=N1, K=K, first=1, seed=seed)
    m["sinks"] = None
    g = torch.Generator().manual_seed(seed)
    pattern = torch.randint(0, 2, (64,), generator=g).float() * 2 - 1
    q = torch.randn((tokens, N1, 576), generator=g) * spread
    q[:, :, 512:] = pattern
    m["q"] = q.to(torch.bfloat16).cuda()
    base = torch.randn(512, generator=g) * mean
    for codes, scale, _ in (m["ori"], m["cmp"]):
        scale.fill_(2.0 ** -5)
        x = base + torch.randn(codes.shape[:-1] + (512,), generator=g)
        codes.copy_(torch.cat([x, torch.zeros(codes.shape[:-1] + (64,))], dim=-1).mul_(32).clamp_(-448, 448).to(codes.dtype).cuda())
    codes, _, table = m["ori"]
    top = math.log(mass / (1 - mass) * 2176) * 24 / 64
    for b in range(tokens):
        row = torch.cat([torch.randn(512, generator=g) * 0.02, pattern * top]) * 32
        codes[int(table[b, 0]), 0, 0] = row.to(codes.dtype).cuda()
    return m


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("tokens", [2, 40])  # in pieces, and whole
@pytest.mark.parametrize("mass,spread,mean", [(0.8, 1.0, 1.0), (0.9, 0.02, 1.0), (0.95, 1.0, 1.0), (0.95, 0.02, 0.0), (0.99, 0.5, 1.0)])
def test_tail_behind_one_key(cuda_device, mass, spread, mean, tokens, kernel):
    """What many small weights add up to is not lost beside one large weight."""
    m = one_key_dominates(tokens, 32, mass, spread, mean, seed=42)
    check_weights(m, *run(m, kernel=kernel, check_status=True), tokens=[0, tokens - 1])


@pytest.mark.parametrize("shape", SHAPES, ids=ident)
def test_weights_of_16_bits(cuda_device, shape):
    m = make(**shape, seed=len(shape["q_lens"]))
    if all(n <= k for n, k in zip(m["q_lens"], m["kv_lens"])):
        check_weights(m, *run(m, kernel="tc", check_status=True))


def test_sharp_scores_and_their_tails(cuda_device):
    """Queries of very different sizes: flat softmaxes, sharp ones and all between."""
    m = make([1] * 40, [3000] * 40, N1=128, seed=43)
    size = torch.exp2(torch.arange(128, device="cuda").float() / 8 - 6)
    m["q"] = (m["q"].float() * size[None, :, None]).to(torch.bfloat16)
    check_weights(m, *run(m, kernel="tc", check_status=True), tokens=[0, 13, 39])


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("q_size,scale", [(24, -9), (30, -9), (100, -9), (0, 20), (0, 40), (0, 60), (-40, 40), (60, 20)])
def test_scores_past_all_digits(cuda_device, q_size, scale, kernel):
    """Scores whose 32-bit steps are whole nats, by large queries or by large scales: each head takes its best key."""
    m = make([1] * 40, [1500] * 40, N1=33, K=300, seed=44)
    m["sinks"] = None
    m["q"] = (m["q"].float() * 2.0 ** q_size).to(torch.bfloat16)
    for _, s, _ in (m["ori"], m["cmp"]):
        s.mul_(2.0 ** (scale + 9))
        s.clamp_(2.0 ** -60, 2.0 ** 60)
    out, lse = run(m, kernel=kernel, check_status=True)
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    if q_size + scale <= 0:  # scores of a hundred nats: no key is clear of the others by 200
        check(m, out, lse, tokens=[0, 20, 39])
        return
    for t in (0, 20, 39):
        b, p = m["where"][t]
        ori, cmp_ = ref.visible(m["case"], b, p, m["idx"][t, 0].numpy())
        k = torch.cat([ref.gather(m["ori"][0][:, :, 0], m["ori"][1], m["ori"][2][b], ori),
                       ref.gather(m["cmp"][0][:, :, 0], m["cmp"][1], m["cmp"][2][b], cmp_)])
        s = m["q"][t].double() @ k.T * m["scale"]
        best = s.topk(2, dim=1)
        reach = (m["q"][t].double().abs() @ k.abs().T * m["scale"]).amax(dim=1)
        clear = best.values[:, 0] - best.values[:, 1] > 2 * 40 * 2.0 ** -22 * reach + 200  # more than scores are off by
        assert clear.sum() > 25
        v = k[best.indices[:, 0], :512]
        assert ((out[t].double() - v).abs() <= 2.0 ** -7 * v.abs())[clear].all()
        assert ((lse[t].double() - best.values[:, 0]).abs() <= 40 * 2.0 ** -22 * reach + 2.0 ** -22 * best.values[:, 0].abs())[clear].all()
