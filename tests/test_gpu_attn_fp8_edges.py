"""sparse_attn_sharedkv_fp8 where index rows end at a chunk's border, maxima rise far, and one key dominates."""

import pytest
import torch

from tests.test_gpu_attn_fp8 import KERNELS, check, make, run

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
