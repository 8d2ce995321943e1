"""The cache's operators beside autograd: changed tensors are noticed, what would get no gradient is refused."""

import pytest
import torch
from torch.autograd import forward_ad
from torch.utils._python_dispatch import TorchDispatchMode

from dsv4_planb_b200.api import sparse_attn_sharedkv
from tests import test_gpu_attn_fp8 as attn
from tests import test_gpu_cache as cache

pytestmark = pytest.mark.gpu


def append_call(m, **kw):
    a = dict(cache=m["cache"].cuda(), cache_scale=None if m["scale"] is None else m["scale"].cuda(), block_table=m["table"].cuda(),
             cu_seqlens_q=m["cu"].cuda(), seqused_kv=m["seq"].cuda(), rope_table=cache.rope_table(300, 64), kv=m["kv"].cuda(), q=m["q"].cuda())
    a.update(kw)
    return a


def append(a):
    a = dict(a)
    return cache.sharedkv_cache_append(a.pop("kv"), **a)


@pytest.mark.parametrize("inference", [False, True])
@pytest.mark.parametrize("pool", ["fp8", "bf16"])
def test_append_raises_versions(cuda_device, pool, inference):
    m = cache.make([1, 3], [9, 200], pool=pool, heads=2, seed=50)
    with torch.inference_mode(inference):
        a = append_call(m)
        written = [t for t in (a["cache"], a["cache_scale"], a["q"]) if t is not None]
        before = [0 if inference else t._version for t in written]
        append(dict(a, q_out=a["q"]))
        if not inference:
            assert all(t._version > v for t, v in zip(written, before))
        read = [a["kv"], a["rope_table"], a["block_table"]]
        if not inference:
            assert not any(t._version for t in read)


def test_attention_raises_versions(cuda_device):
    m = attn.make([1, 2], [700, 900], N1=32, seed=51)
    out, lse = torch.empty((3, 32, 512), dtype=torch.bfloat16, device="cuda"), torch.empty((3, 32), device="cuda")
    attn.run(m, out=out, lse_out=lse)
    assert out._version > 0 and lse._version > 0 and m["q"]._version == 0


def test_append_into_a_saved_cache_is_noticed(cuda_device):
    """A backward pass over the 16-bit cache refuses once rows have been appended to it."""
    m = cache.make([1, 3], [9, 200], D=512, bs=64, pool="bf16", heads=4, seed=52)
    a = append_call(m)
    q = append(a).requires_grad_()
    out = sparse_attn_sharedkv(q, ori_kv=a["cache"], ori_block_table=a["block_table"], cu_seqlens_q=a["cu_seqlens_q"],
                               seqused_kv=a["seqused_kv"], sinks=torch.zeros(4, device="cuda"), softmax_scale=512 ** -0.5)
    append(a)
    with pytest.raises(RuntimeError, match="inplace"):
        out.float().sum().backward()


class Seen(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.names.append(func.name())
        return func(*args, **(kwargs or {}))


def test_dispatch_modes_see_the_calls(cuda_device):
    m = attn.make([1, 2], [700, 900], N1=32, seed=53)
    want = attn.run(m)
    with Seen() as seen:
        got = attn.run(m)
    assert "sas_b200::sparse_attn_sharedkv_fp8" in seen.names and all(torch.equal(x, y) for x, y in zip(got, want))
    c = cache.make([1, 3], [9, 200], heads=2, seed=53)
    a = append_call(c)
    with Seen() as seen:
        append(a)
    assert "sas_b200::sharedkv_cache_append" in seen.names


@pytest.mark.parametrize("name", ["kv", "cache", "cache_scale", "rope_table", "q"])
def test_append_refuses_tangents(cuda_device, name):
    a = append_call(cache.make([1, 3], [9, 200], pool="bf16" if name == "cache" else "fp8", heads=2, seed=54))
    with forward_ad.dual_level():
        a[name] = forward_ad.make_dual(a[name], torch.ones_like(a[name]))
        with pytest.raises(ValueError, match="no derivative"):
            append(a)


@pytest.mark.parametrize("name", ["q", "ori_kv_scale", "cmp_kv_scale", "sinks"])
def test_attention_refuses_tangents(cuda_device, name):
    m = attn.make([1, 2], [700, 900], N1=32, seed=55)
    kw = dict(attn.kwargs(m), q=m["q"])
    with forward_ad.dual_level():
        kw[name] = forward_ad.make_dual(kw[name], torch.ones_like(kw[name]))
        with pytest.raises(ValueError, match="no derivative"):
            attn.run(m, **kw)
