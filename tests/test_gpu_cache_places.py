"""sharedkv_cache_append: queries that stay in place unturned, and rows that have no place."""

import pytest
import torch

from dsv4_planb_b200.cache import rope_table
from tests.test_gpu_cache import check, make, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pool", ["fp8", "bf16"])
@pytest.mark.parametrize("interleaved", [True, False])
def test_queries_without_rotation(cuda_device, interleaved, pool):
    """Without angles queries are copied, or stay where they are."""
    m = make([3, 40], [70, 200], pool=pool, heads=18, seed=61)
    for place in (False, True):
        q = m["q"].cuda()
        cache, scale, out = run(m, None, q=q, q_out=q if place else None, rope_interleaved=interleaved, check_status=True)
        check(m, cache, scale, None)
        assert torch.equal(out.cpu(), m["q"]) and (out is q) == place
