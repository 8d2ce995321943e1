"""Sparse shared-KV attention over an 8-bit paged cache.

``sparse_attn_sharedkv_fp8`` is ``sparse_attn_sharedkv`` (same scenarios, layouts, index rules and
results up to the cache's rounding) over ``float8_e4m3fn`` pools with one fp32 scale per block, which
halves the cache and what a decode step reads.  ``ori_first`` keeps the first positions of a sequence
visible next to the sliding window.  The reference has neither.
"""

from __future__ import annotations

import functools
from typing import Optional, Tuple, Union

import torch

from . import _lib
from .api import _dense16, _dtype_code, _pool16, _scenario
from .cache import _current_device, _eager, _int32, _ops, _raw_stream, _refuse_derivatives, _written

KERNELS = {"auto": 0, "simt": 1, "tc": 2}
_INT32 = 2**31 - 1  # no position lies beyond it


@functools.lru_cache(maxsize=512)
def _call_args(*sizes) -> Tuple["_lib.SasFp8Args", int]:
    """The call's sizes as the C struct, and the workspace they need (nothing of the tensors)."""
    args = _lib.SasFp8Args(*sizes)
    n = _lib.ctypes.c_size_t(0)
    _lib.check(_lib.load().sas_kvq_workspace_size(args, n), "sas_kvq_workspace_size")
    return args, n.value


def _launch(q, ori_kv, ori_kv_scale, cmp_kv, cmp_kv_scale, cmp_sparse_indices, ori_block_table, cmp_block_table,
            cu_seqlens_q, seqused_kv, sinks, softmax_scale, cmp_ratio, ori_win_left, ori_first, layout_q, v_head_dim,
            kernel, check_status, out, lse):
    device = q.get_device()
    if device != _current_device():
        with torch.cuda.device(device):
            return _launch(q, ori_kv, ori_kv_scale, cmp_kv, cmp_kv_scale, cmp_sparse_indices, ori_block_table,
                           cmp_block_table, cu_seqlens_q, seqused_kv, sinks, softmax_scale, cmp_ratio, ori_win_left,
                           ori_first, layout_q, v_head_dim, kernel, check_status, out, lse)
    scenario = _scenario(cmp_kv, cmp_sparse_indices)
    cu = act_q = cmp_bt = idx = None
    if cu_seqlens_q is not None:
        cu = _int32(cu_seqlens_q, device)
    if layout_q == "TND":
        T, N1, D = q.shape
        S, B = 0, cu.numel() - 1
    else:
        B, S, N1, D = q.shape
        T = B * S
        if cu is not None:
            cu, act_q = None, (cu[1:] - cu[:-1]).contiguous()
    _pool16(ori_kv, "ori_kv")
    ori_bt, seq = _int32(ori_block_table, device), _int32(seqused_kv, device)
    cb = cs = ct = K = 0
    if scenario >= 2:
        _pool16(cmp_kv, "cmp_kv")
        cmp_bt = _int32(cmp_block_table, device)
        cb, cs, _, _ = cmp_kv.shape
        ct = cmp_bt.shape[1]
    if scenario == 3:
        idx = _int32(cmp_sparse_indices, device)
        K = idx.shape[-1]
    if sinks is not None and (sinks.dtype is not torch.float32 or sinks.get_device() != device or not sinks.is_contiguous()):
        sinks = sinks.to(device=q.device, dtype=torch.float32).contiguous()
    q = _dense16(q)
    ob, obs, _, _ = ori_kv.shape
    args, nbytes = _call_args(B, T, S, N1, D, v_head_dim, ob, obs, ori_bt.shape[1], cb, cs, ct, K, cmp_ratio, scenario,
                              ori_win_left, ori_first, _dtype_code(q.dtype), softmax_scale, KERNELS[kernel])
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)  # from the caching allocator, in stream order
    out_user = None
    if out.data_ptr() % 16:  # a caller's out that starts inside a 16-byte vector
        out_user, out = out, torch.empty_like(out)
    lib = _lib.load()
    stream = _raw_stream(device)
    # (conditions in place: eight calls of _ptr cost 1 us)
    rc = lib.sas_kvq_forward(args, q.data_ptr(), ori_kv.data_ptr(), ori_kv_scale.data_ptr(), ori_bt.data_ptr(),
                             None if cmp_kv is None else cmp_kv.data_ptr(),
                             None if cmp_kv is None else cmp_kv_scale.data_ptr(),
                             None if cmp_bt is None else cmp_bt.data_ptr(), None if idx is None else idx.data_ptr(),
                             None if cu is None else cu.data_ptr(), None if act_q is None else act_q.data_ptr(),
                             seq.data_ptr(), None if sinks is None else sinks.data_ptr(), out.data_ptr(),
                             None if lse is None else lse.data_ptr(), ws.data_ptr(), nbytes, stream)
    if rc:
        _lib.check(rc, "sas_kvq_forward")
    if out_user is not None:
        out_user.copy_(out)
    _written(out, lse)
    if check_status:
        st = _lib.ctypes.c_uint32(0)
        _lib.check(lib.sas_kvq_read_status(args, ws.data_ptr(), st, stream), "sas_kvq_read_status")
        if st.value:
            raise RuntimeError(f"sas_kvq_forward device status: {_lib.status_names(st.value)}")


_SCHEMA = ("(Tensor q, Tensor ori_kv, Tensor ori_kv_scale, Tensor? cmp_kv, Tensor? cmp_kv_scale, "
           "Tensor? cmp_sparse_indices, Tensor ori_block_table, Tensor? cmp_block_table, Tensor? cu_seqlens_q, "
           "Tensor seqused_kv, Tensor? sinks, float softmax_scale, int cmp_ratio, int ori_win_left, int ori_first, "
           "str layout_q, int v_head_dim, str kernel, bool check_status, Tensor(a!) out, Tensor(b!)? lse) -> ()")
_ops.define("sparse_attn_sharedkv_fp8" + _SCHEMA)
_ops.impl("sparse_attn_sharedkv_fp8", _launch, "CUDA")


@torch.library.register_fake("sas_b200::sparse_attn_sharedkv_fp8")
def _fake(*args):
    return None


def _check_pool(name, pool, scale, D, q):
    if pool.dtype is not torch.float8_e4m3fn:
        raise ValueError(f"{name} must be float8_e4m3fn (got {pool.dtype}); 16-bit pools go to sparse_attn_sharedkv")
    shape = pool.shape
    if len(shape) != 4 or shape[2] != 1 or shape[3] != D:
        raise ValueError(f"{name} must be [blocks, block_size, 1, {D}] (got {tuple(shape)})")
    if scale is None or scale.dtype is not torch.float32 or scale.numel() != shape[0] or not scale.is_contiguous():
        raise ValueError(f"{name}_scale must be contiguous float32 with one entry per block of {name}")
    if not pool.get_device() == scale.get_device() == q.get_device():
        raise ValueError(f"{name} and {name}_scale must be on {q.device}")


def sparse_attn_sharedkv_fp8(
    q: torch.Tensor,
    *,
    ori_kv: torch.Tensor,
    ori_kv_scale: torch.Tensor,
    cmp_kv: Optional[torch.Tensor] = None,
    cmp_kv_scale: Optional[torch.Tensor] = None,
    cmp_sparse_indices: Optional[torch.Tensor] = None,
    ori_block_table: torch.Tensor,
    cmp_block_table: Optional[torch.Tensor] = None,
    cu_seqlens_q: Optional[torch.Tensor] = None,
    seqused_kv: torch.Tensor,
    sinks: Optional[torch.Tensor] = None,
    softmax_scale: float,
    cmp_ratio: Optional[int] = None,
    ori_win_left: int = 127,
    ori_first: int = 0,
    layout_q: str = "TND",
    return_softmax_lse: bool = False,
    v_head_dim: Optional[int] = None,
    kernel: str = "auto",
    out: Optional[torch.Tensor] = None,
    lse_out: Optional[torch.Tensor] = None,
    check_status: bool = False,
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Attention over 8-bit pools: the keywords, scenarios and results of ``sparse_attn_sharedkv``.

    ``ori_kv`` / ``cmp_kv`` are ``float8_e4m3fn`` ``[blocks, block_size, 1, D]`` and ``*_scale`` fp32
    ``[blocks]`` or ``[blocks, 1]`` (in [2^-60, 2^60]; ``cache.sharedkv_cache_append`` writes both).  A key
    row is code x scale of its block, and its first ``v_head_dim`` dims are its value.  A token at
    position p sees the window [max(p - ``ori_win_left``, 0), p], the positions below ``ori_first`` that
    lie before it, and the compressed rows that ``sparse_attn_sharedkv`` gives it.  ``sinks`` (``[N1]`` or None) adds
    exp(sink) to the softmax's denominator.  Returns ``out`` in the type and layout of ``q`` (last dim
    ``v_head_dim``) and with ``return_softmax_lse`` the natural-log LSE in fp32.

    ``D`` is a multiple of 16 up to 1024 and ``v_head_dim`` (``D`` when None) one of 32 up to 512, so that
    rows of 576 need it said.  ``kernel``: "tc" (tensor cores: D 512 or 576, ``v_head_dim`` 512, up to 128
    heads, bf16 q), "simt" (CUDA cores: every shape), "auto".

    No host synchronisation (``check_status`` reads the status bits and raises); graph-capturable; no
    backward pass.
    """
    assert layout_q in ("TND", "BSND"), f"unsupported layout_q={layout_q!r}"
    if kernel not in KERNELS:
        raise ValueError(f"kernel must be one of {sorted(KERNELS)}")
    if not q.is_cuda:
        raise ValueError("q must be a CUDA tensor (sas_b200 has no CPU path)")
    _refuse_derivatives("sparse_attn_sharedkv_fp8", q, ori_kv, ori_kv_scale, cmp_kv, cmp_kv_scale, sinks, out, lse_out)
    shape, kind = q.shape, q.dtype
    if layout_q == "TND":
        lead = 1
        assert cu_seqlens_q is not None, "cu_seqlens_q is required for TND"
        B = cu_seqlens_q.numel() - 1
    else:
        lead, B = 2, shape[0]
        if cu_seqlens_q is not None and cu_seqlens_q.numel() != B + 1:
            raise ValueError(f"cu_seqlens_q must have {B + 1} entries (got {cu_seqlens_q.numel()})")
    if len(shape) != lead + 2:
        raise ValueError(f"q must be {'[T, N1, D]' if lead == 1 else '[B, S, N1, D]'} (got {tuple(shape)})")
    N1, D = shape[-2], shape[-1]
    Dv = D if v_head_dim is None else int(v_head_dim)
    if D % 16 or D > 1024:
        raise ValueError(f"the head dim must be a multiple of 16 up to 1024 (got {D})")
    if Dv <= 0 or Dv % 32 or Dv > min(D, 512):
        given = "" if v_head_dim is not None else ", the head dim: pass v_head_dim"
        raise ValueError(f"v_head_dim must be a multiple of 32 up to {min(D, 512)} (got {Dv}{given})")
    _check_pool("ori_kv", ori_kv, ori_kv_scale, D, q)
    if ori_block_table.dim() != 2 or ori_block_table.shape[0] < B:
        raise ValueError(f"ori_block_table must be [B>={B}, table_len] (got {tuple(ori_block_table.shape)})")
    if seqused_kv.numel() < B:
        raise ValueError(f"seqused_kv must have {B} entries (got {seqused_kv.numel()})")
    if cmp_kv is not None:
        assert cmp_ratio is not None, "cmp_ratio is required with cmp_kv"
        _check_pool("cmp_kv", cmp_kv, cmp_kv_scale, D, q)
        if cmp_block_table is None or cmp_block_table.dim() != 2 or cmp_block_table.shape[0] < B:
            raise ValueError(f"cmp_block_table must be [B>={B}, table_len]")
        if cmp_sparse_indices is not None:
            rows = cmp_sparse_indices.shape
            if len(rows) != lead + 2 or rows[:lead] != shape[:lead] or rows[lead] != 1:
                raise ValueError(f"cmp_sparse_indices must hold [1, K] per token (got {tuple(rows)})")
    elif cmp_sparse_indices is not None:
        raise ValueError("cmp_sparse_indices goes with cmp_kv")
    if sinks is not None and sinks.numel() != N1:
        raise ValueError(f"sinks must have {N1} entries (got {sinks.numel()})")
    if ori_win_left < 0 or ori_first < 0:
        raise ValueError("ori_win_left and ori_first must be >= 0")
    tokens = shape[:lead]
    if out is None:
        result = out = q.new_empty((*tokens, N1, Dv))
    else:
        result = out.view((*tokens, N1, Dv)) if out.is_contiguous() and out.numel() == tokens.numel() * N1 * Dv else None
        if result is None or out.dtype is not kind or out.get_device() != q.get_device():
            raise ValueError(f"out must be contiguous {kind} of shape {(*tokens, N1, Dv)} on {q.device}")
    lse = sums = lse_out
    if lse is not None:
        sums = lse.view((*tokens, N1)) if lse.is_contiguous() and lse.numel() == tokens.numel() * N1 else None
        if sums is None or lse.dtype is not torch.float32 or lse.get_device() != q.get_device():
            raise ValueError(f"lse_out must be contiguous float32 of shape {(*tokens, N1)} on {q.device}")
    elif return_softmax_lse:
        lse = sums = q.new_empty((*tokens, N1), dtype=torch.float32)
    call = (q, ori_kv, ori_kv_scale, cmp_kv, cmp_kv_scale, cmp_sparse_indices, ori_block_table, cmp_block_table,
            cu_seqlens_q, seqused_kv, sinks, float(softmax_scale), 4 if cmp_ratio is None else min(int(cmp_ratio), _INT32),
            min(int(ori_win_left), _INT32), min(int(ori_first), _INT32), layout_q, Dv, kernel, bool(check_status), out, lse)
    if _eager(q, ori_kv, cmp_kv, out, lse):
        _launch(*call)
    else:
        torch.ops.sas_b200.sparse_attn_sharedkv_fp8(*call)
    return (result, sums) if return_softmax_lse else result
