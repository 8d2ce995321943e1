"""Arguments that no kernel takes, and arguments that require a gradient and get none, are refused before anything is
launched (fake CUDA tensors: no GPU)."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from dsv4_planb_b200.attn_fp8 import sparse_attn_sharedkv_fp8
from dsv4_planb_b200.cache import sharedkv_cache_append

F8 = torch.float8_e4m3fn


def empty(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="cuda")


def append_call(pool):
    a = dict(cache=empty(4, 128, 1, 576, dtype=pool), block_table=empty(1, 4, dtype=torch.int32), cu_seqlens_q=empty(2, dtype=torch.int32),
             seqused_kv=empty(1, dtype=torch.int32), rope_table=empty(300, 64), q=empty(3, 8, 576, dtype=torch.bfloat16))
    if pool is F8:
        a["cache_scale"] = empty(4)
    return a


@pytest.mark.parametrize("pool,name", [(F8, "kv"), (F8, "cache_scale"), (F8, "rope_table"), (F8, "q"), (F8, "q_out"), (torch.bfloat16, "cache")])
def test_append(pool, name):
    with FakeTensorMode():
        kv, a = empty(3, 576, dtype=torch.bfloat16), append_call(pool)
        sharedkv_cache_append(kv, **a)
        a["q_out"] = empty(3, 8, 576, dtype=torch.bfloat16)
        (kv if name == "kv" else a[name]).requires_grad_()
        with pytest.raises(ValueError, match="no backward"):
            sharedkv_cache_append(kv, **a)
        with torch.no_grad():
            sharedkv_cache_append(kv, **a)


@pytest.mark.parametrize("name", ["q", "ori_kv", "ori_kv_scale", "cmp_kv", "cmp_kv_scale", "sinks", "out", "lse_out"])
def test_attention(name):
    with FakeTensorMode():
        i32 = torch.int32
        a = dict(ori_kv=empty(4, 128, 1, 576, dtype=F8), ori_kv_scale=empty(4), cmp_kv=empty(4, 128, 1, 576, dtype=F8), cmp_kv_scale=empty(4),
                 ori_block_table=empty(1, 4, dtype=i32), cmp_block_table=empty(1, 4, dtype=i32), cu_seqlens_q=empty(2, dtype=i32),
                 seqused_kv=empty(1, dtype=i32), sinks=empty(8), softmax_scale=1.0, cmp_ratio=4, v_head_dim=512,
                 out=empty(3, 8, 512, dtype=torch.bfloat16), lse_out=empty(3, 8))
        q = empty(3, 8, 576, dtype=torch.bfloat16)
        sparse_attn_sharedkv_fp8(q, **a)
        (q if name == "q" else a[name]).requires_grad_()
        with pytest.raises(ValueError, match="no backward"):
            sparse_attn_sharedkv_fp8(q, **a)
        with torch.no_grad():
            sparse_attn_sharedkv_fp8(q, **a)


@pytest.mark.parametrize("D,Dv,text", [(576, None, r"up to 512 \(got 576, the head dim: pass v_head_dim"), (576, 528, "multiple of 32 up to 512"),
                                       (576, 500, "multiple of 32"), (256, 288, "up to 256"), (576, 0, "multiple of 32"), (48, None, "up to 48"),
                                       (584, 512, "multiple of 16 up to 1024"), (1040, 512, "multiple of 16 up to 1024")])
def test_value_dims(D, Dv, text):
    """Sizes that no kernel takes are refused by name, the default of v_head_dim among them."""
    with FakeTensorMode():
        i32 = torch.int32
        with pytest.raises(ValueError, match=text):
            sparse_attn_sharedkv_fp8(empty(3, 8, D, dtype=torch.bfloat16), ori_kv=empty(4, 128, 1, D, dtype=F8), ori_kv_scale=empty(4),
                                     ori_block_table=empty(1, 4, dtype=i32), cu_seqlens_q=empty(2, dtype=i32), seqused_kv=empty(1, dtype=i32),
                                     softmax_scale=1.0, v_head_dim=Dv)


@pytest.mark.parametrize("D", [568, 1040])
def test_append_dims(D):
    with FakeTensorMode():
        a = append_call(F8)
        a.update(cache=empty(4, 128, 1, D, dtype=F8), q=None, rope_table=None)
        with pytest.raises(ValueError, match="multiple of 16 up to 1024"):
            sharedkv_cache_append(empty(3, D, dtype=torch.bfloat16), **a)
