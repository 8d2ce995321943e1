"""Argument checks of the cache append and of the attention over an 8-bit cache: the C entries reject
calls outside their contract before touching the device, and the Python entries have no CPU path."""

import ctypes

import pytest
import torch

from dsv4_planb_b200 import _lib, build
from dsv4_planb_b200.attn_fp8 import sparse_attn_sharedkv_fp8
from dsv4_planb_b200.cache import rope_table, sharedkv_cache_append

P = 1 << 20  # a 16-byte aligned address that no rejected call reads


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def append_args(**kw):
    a = _lib.SasAppendArgs(2, 2, 0, 576, 64, 1, 1, 100, 8, 128, 4, 0, _lib.SAS_DTYPE_BF16, _lib.SAS_DTYPE_E4M3, 576)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def append(lib, a, kv=P, q=None, q_out=None, rope=P, table=P, cu=P, act_q=None, act_kv=P, cache=P, scale=P, status=None):
    return lib.sas_cache_append(a, kv, q, q_out, rope, table, cu, act_q, act_kv, cache, scale, status, None)


@pytest.mark.parametrize("field,value,rc", [
    ("batch", -1, 1), ("num_tokens", -1, 1), ("num_heads", -1, 1), ("head_dim", 0, 1), ("rope_dim", -16, 1), ("rope_step", 0, 1),
    ("rope_rows", -1, 1), ("block_num", 0, 1), ("block_size", 0, 1), ("table_len", 0, 1), ("kv_row_stride", 568, 1),
    ("dtype", 2, 1), ("dtype", 7, 1), ("cache_dtype", 1, 2), ("head_dim", 568, 2), ("head_dim", 1040, 2), ("rope_dim", 24, 2),
    ("rope_dim", 592, 2), ("kv_row_stride", 577, 2), ("block_num", 1 << 25, 2),
])
def test_append_rejects(lib, field, value, rc):
    a = append_args()
    if field == "head_dim" and value > 576:
        a.kv_row_stride = value
    setattr(a, field, value)
    assert append(lib, a) == rc


def test_append_rejects_pointers(lib):
    a = append_args()
    for name in ("kv", "rope", "table", "act_kv", "cache", "scale"):
        assert append(lib, a, **{name: None}) == _lib.SAS_ERR_INVALID_ARG, name
    for name in ("kv", "rope", "cache"):
        assert append(lib, a, **{name: P + 8}) == _lib.SAS_ERR_INVALID_ARG, name
    for name in ("table", "cu", "act_kv", "scale", "status"):
        assert append(lib, a, **{name: P + 2}) == _lib.SAS_ERR_INVALID_ARG, name
    assert append(lib, append_args(num_heads=4)) == _lib.SAS_ERR_INVALID_ARG  # no q
    assert append(lib, append_args(num_heads=4), q=P, q_out=P + 4) == _lib.SAS_ERR_INVALID_ARG
    assert append(lib, append_args(max_q_len=3), cu=None) == _lib.SAS_ERR_INVALID_ARG  # 2 x 3 rows are not 2
    a.reserved[2] = 1
    assert append(lib, a) == _lib.SAS_ERR_INVALID_ARG
    assert append(lib, append_args(num_tokens=0), kv=None, cache=None) == _lib.SAS_OK
    assert lib.sas_cache_append(None, *([None] * 12)) == _lib.SAS_ERR_INVALID_ARG


def attn_args(**kw):
    a = _lib.SasFp8Args(2, 2, 0, 128, 576, 512, 8, 128, 4, 8, 128, 4, 256, 4, 3, 127, 0, _lib.SAS_DTYPE_BF16, 0.04, 0)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def size(lib, a):
    n = ctypes.c_size_t(0)
    return lib.sas_kvq_workspace_size(a, n), n.value


@pytest.mark.parametrize("field,value,rc", [
    ("batch", -1, 1), ("num_tokens", -1, 1), ("max_q_len", -1, 1), ("num_heads", 0, 1), ("head_dim", 0, 1), ("v_head_dim", 0, 1),
    ("scenario", 0, 1), ("scenario", 4, 1), ("ori_win_left", -1, 1), ("ori_first", -1, 1), ("topk", -1, 1), ("dtype", 2, 1),
    ("ori_block_num", 0, 1), ("ori_block_size", 0, 1), ("ori_table_len", 0, 1), ("cmp_block_num", 0, 1), ("cmp_ratio", 0, 1),
    ("kernel", 3, 1), ("kernel", -1, 1), ("head_dim", 584, 2), ("head_dim", 1040, 2), ("v_head_dim", 528, 2), ("v_head_dim", 500, 2),
    ("ori_block_num", 1 << 25, 2), ("cmp_block_num", 1 << 25, 2),
])
def test_attention_rejects(lib, field, value, rc):
    assert size(lib, attn_args(**{field: value}))[0] == rc


def attend(lib, a, ws=P, ws_bytes=1 << 30, **kw):
    names = ["q", "ori", "ori_scale", "ori_bt", "cmp", "cmp_scale", "cmp_bt", "idx", "cu", "act_q", "act_kv", "sinks", "out", "lse"]
    at = {n: P for n in names}
    at["act_q"] = None
    at.update(kw)
    return lib.sas_kvq_forward(a, *[at[n] for n in names], ws, ws_bytes, None)


def test_attention_rejects_pointers(lib):
    a = attn_args()
    rc, n = size(lib, a)
    assert rc == 0 and n >= 2 * 256 * 4
    assert attend(lib, a, ws=None) == _lib.SAS_ERR_WORKSPACE
    assert attend(lib, a, ws_bytes=n - 1) == _lib.SAS_ERR_WORKSPACE
    for name in ("q", "ori", "ori_scale", "ori_bt", "cmp", "cmp_scale", "cmp_bt", "idx", "act_kv", "out"):
        assert attend(lib, a, **{name: None}) == _lib.SAS_ERR_INVALID_ARG, name
    for name in ("q", "ori", "cmp", "out", "ws"):
        assert attend(lib, a, **{name: P + 8}) == _lib.SAS_ERR_INVALID_ARG, name
    for name in ("ori_scale", "ori_bt", "cmp_scale", "cmp_bt", "idx", "cu", "act_kv", "sinks", "lse"):
        assert attend(lib, a, **{name: P + 2}) == _lib.SAS_ERR_INVALID_ARG, name
    assert attend(lib, attn_args(max_q_len=3), cu=None) == _lib.SAS_ERR_INVALID_ARG
    assert attend(lib, attn_args(num_tokens=0), q=None, out=None) == _lib.SAS_OK
    a.reserved[0] = 1
    assert size(lib, a)[0] == _lib.SAS_ERR_INVALID_ARG
    assert lib.sas_kvq_workspace_size(None, ctypes.c_size_t()) == _lib.SAS_ERR_INVALID_ARG
    assert lib.sas_kvq_read_status(None, P, ctypes.c_uint32(), None) == _lib.SAS_ERR_INVALID_ARG


def test_struct_sizes():
    assert ctypes.sizeof(_lib.SasAppendArgs) == 14 * 4 + 8 + 16
    assert ctypes.sizeof(_lib.SasFp8Args) == 24 * 4


def test_python_has_no_cpu_path():
    z = torch.zeros
    with pytest.raises(ValueError, match="CUDA"):
        sharedkv_cache_append(z(1, 576), cache=z(1, 128, 1, 576), block_table=z(1, 1), seqused_kv=z(1), cu_seqlens_q=z(2))
    with pytest.raises(ValueError, match="CUDA"):
        sparse_attn_sharedkv_fp8(z(1, 4, 576), ori_kv=z(1), ori_kv_scale=z(1), ori_block_table=z(1, 1), seqused_kv=z(1),
                                 cu_seqlens_q=z(2), softmax_scale=1.0)
    with pytest.raises(AssertionError, match="layout"):
        sparse_attn_sharedkv_fp8(z(1, 4, 576), ori_kv=z(1), ori_kv_scale=z(1), ori_block_table=z(1, 1), seqused_kv=z(1),
                                 softmax_scale=1.0, layout_q="SBND")
    with pytest.raises(ValueError, match="kernel"):
        sparse_attn_sharedkv_fp8(z(1, 4, 576), ori_kv=z(1), ori_kv_scale=z(1), ori_block_table=z(1, 1), seqused_kv=z(1),
                                 softmax_scale=1.0, kernel="fast")


def test_rope_table_arguments():
    t = rope_table(3, 16, device="cpu")
    assert t.shape == (3, 16) and t.dtype == torch.float32
    assert torch.equal(rope_table(3, 4, inv_freq=torch.tensor([1.0, 0.5]), device="cpu")[2, :2],
                       torch.cos(torch.tensor([2.0, 1.0], dtype=torch.float64)).float())
    with pytest.raises(ValueError, match="even"):
        rope_table(3, 15, device="cpu")
    with pytest.raises(ValueError, match="entries"):
        rope_table(3, 16, inv_freq=torch.ones(4), device="cpu")
