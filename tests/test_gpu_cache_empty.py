"""Rows without a request: the cache append and the 8-bit attention on a batch of none."""

import pytest
import torch

from dsv4_planb_b200.cache import rope_table, sharedkv_cache_append
from tests import test_gpu_attn_fp8 as attn
from tests import test_gpu_cache as cache

pytestmark = pytest.mark.gpu


def tables(names, widths, padded):
    """Block tables and lengths of no request, or of rows kept for requests to come."""
    n = 3 if padded else 0
    t = {name: torch.zeros((n, w), dtype=torch.int32, device="cuda") for name, w in zip(names, widths)}
    return dict(t, seqused_kv=torch.full((n,), 100, dtype=torch.int32, device="cuda"), cu_seqlens_q=torch.zeros(1, dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("padded", [False, True])
@pytest.mark.parametrize("pool", ["fp8", "bf16"])
def test_append(cuda_device, pool, padded):
    m = cache.make([7], [200], pool=pool, heads=17, seed=70)
    c, s = m["cache"].cuda(), None if m["scale"] is None else m["scale"].cuda()
    bits = c.view(torch.uint8).clone()
    kw = dict(cache=c, cache_scale=s, rope_table=rope_table(300, 64), check_status=True, **tables(["block_table"], [2], padded))
    q = m["q"].cuda()
    out = torch.full_like(q, 9.0)
    assert sharedkv_cache_append(m["kv"].cuda(), q=q, q_out=out, **kw) is out
    assert torch.equal(out.cpu(), m["q"]) and torch.equal(q.cpu(), m["q"])
    assert sharedkv_cache_append(m["kv"].cuda(), q=q, q_out=q, **kw) is q and torch.equal(q.cpu(), m["q"])
    assert sharedkv_cache_append(m["kv"].cuda(), **kw) is None
    assert torch.equal(c.view(torch.uint8), bits) and (s is None or torch.equal(s.cpu(), m["scale"]))


@pytest.mark.parametrize("padded", [False, True])
@pytest.mark.parametrize("tokens", [2, 70])
@pytest.mark.parametrize("scenario", [1, 2, 3])
@pytest.mark.parametrize("kernel", attn.KERNELS)
def test_attention(cuda_device, kernel, scenario, tokens, padded):
    m = attn.make([tokens], [200], N1=20, K=30, scenario=scenario, seed=71)
    names = ["ori_block_table"] + (["cmp_block_table"] if scenario >= 2 else [])
    out, lse = torch.full((tokens, 20, 512), 9.0, dtype=torch.bfloat16, device="cuda"), torch.full((tokens, 20), 9.0, device="cuda")
    attn.run(m, kernel=kernel, out=out, lse_out=lse, check_status=True, **tables(names, [2, 2], padded))
    assert not out.any() and not lse.any()
