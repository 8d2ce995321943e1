"""Writing the paged shared-KV cache that the attention operators read.

``sharedkv_cache_append`` puts the new K = V rows of a batch at their positions in a paged pool (the
full-resolution or the compressed one) and rotates the positional tail of each row on the way; given
query heads it rotates those too, in the same launch.  A pool holds 16-bit rows (``bfloat16`` or
``float16``, what ``sparse_attn_sharedkv`` reads) or ``float8_e4m3fn`` codes with one power-of-two scale
per block (what ``sparse_attn_sharedkv_fp8`` reads).  The reference has no counterpart: its caches come
filled.
"""

from __future__ import annotations

import functools
from typing import Optional

import torch
from torch.autograd import forward_ad

from . import _lib
from .api import _dense16, _dtype_code, _i32, _pool16, _ptr

_CACHE_DTYPES = {torch.bfloat16: _lib.SAS_DTYPE_BF16, torch.float16: _lib.SAS_DTYPE_FP16,
                 torch.float8_e4m3fn: _lib.SAS_DTYPE_E4M3}


def rope_table(positions: int, rope_dim: int, *, base: float = 10000.0, inv_freq: Optional[torch.Tensor] = None,
               device="cuda") -> torch.Tensor:
    """Angles of positions 0 .. ``positions`` - 1 as fp32 ``[positions, rope_dim]``: cos of the
    ``rope_dim`` / 2 frequencies, then sin.  ``inv_freq`` (``[rope_dim / 2]``) replaces
    ``base ** (-2 i / rope_dim)``.  Products and functions are taken in 64 bits: at position 2^17 an
    angle in 32 bits is off by up to 2^-8."""
    if rope_dim % 2:
        raise ValueError(f"rope_dim must be even (got {rope_dim})")
    if inv_freq is None:
        inv_freq = base ** (-torch.arange(0, rope_dim, 2, dtype=torch.float64, device=device) / rope_dim)
    if inv_freq.numel() != rope_dim // 2:
        raise ValueError(f"inv_freq must have {rope_dim // 2} entries (got {inv_freq.numel()})")
    ang = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * inv_freq.to(device, torch.float64)
    return torch.cat([ang.cos(), ang.sin()], dim=1).to(torch.float32)


def _refuse_derivatives(what: str, *tensors: Optional[torch.Tensor]) -> None:
    """Raises where one of the call's floating-point tensors would silently get no gradient or lose its tangent."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError(f"{what} has no backward pass: call it under torch.no_grad() or detach its inputs")
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise ValueError(f"{what} has no derivative: pass tensors without tangents")


_PLAIN = frozenset((torch.Tensor, type(None)))
_is_tracing, _transforms = torch._C._is_tracing, torch._C._are_functorch_transforms_active
_dispatch_modes, _function_modes = torch._C._len_torch_dispatch_stack, torch._C._len_torch_function_stack
_increment_version = torch._C._increment_version  # torch.autograd.graph.increment_version takes half a us more


def _eager(*tensors: Optional[torch.Tensor]) -> bool:
    """Plain tensors outside tracing, modes and transforms: the launch needs no dispatcher (whose Python kernels
    cost about 10 us a call).  Everything else takes the registered op."""
    return not (torch.compiler.is_compiling() or _is_tracing() or _dispatch_modes() or _function_modes()
                or _transforms()) and _PLAIN.issuperset(map(type, tensors))


def _written(*tensors: Optional[torch.Tensor]) -> None:
    """Tells autograd that a launch has changed these tensors."""
    _increment_version([t for t in tensors if t is not None])


def _int32(t: torch.Tensor, device: int) -> torch.Tensor:
    """``_i32`` with a short way for what needs no conversion."""
    if t.dtype is torch.int32 and t.get_device() == device and t.is_contiguous():
        return t
    return _i32(t, torch.device("cuda", device))


# The current stream's handle: torch.cuda.current_stream builds a Stream object first (3 us a call).
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)  # of an initialised CUDA: 1 us less


def _rows2d(kv: torch.Tensor, T: int, D: int) -> torch.Tensor:
    """``kv`` as T rows of D consecutive elements, 16-byte aligned; rows may be further apart (a slice
    of a wider projection), anything else is copied."""
    v = kv
    if kv.dim() != 2:
        try:
            v = kv.view(T, D)
        except RuntimeError:
            v = kv.reshape(T, D)
    row, one = v.stride()
    if one != 1 or (T > 1 and (row % 8 or row < D)) or v.data_ptr() % 16:
        v = v.contiguous()
        if v.data_ptr() % 16:
            v = v.clone()
    return v


def _rows_meet(rows: torch.Tensor, T: int, D: int, at: int, size: int) -> bool:
    """Whether some of the T rows of D 16-bit elements lie within ``size`` bytes from address ``at`` on."""
    row, step = rows.data_ptr(), 2 * rows.stride(0) if T > 1 else 2 * D  # one row may have any stride, 0 too
    if not size or row >= at + size or row + (T - 1) * step + 2 * D <= at:
        return False
    first = max((at - row - 2 * D) // step + 1, 0)  # the first row that ends behind the address
    return first < T and row + first * step < at + size


@functools.lru_cache(maxsize=512)
def _append_args(*sizes) -> "_lib.SasAppendArgs":
    """The call's sizes as the C struct (nothing of the tensors themselves)."""
    return _lib.SasAppendArgs(*sizes)


def _append(kv, cache, cache_scale, block_table, seqused_kv, cu_seqlens_q, rope_table, rope_interleaved, rope_step, q,
            q_out, layout_q, check_status):
    device = cache.get_device()
    if device != _current_device():
        with torch.cuda.device(device):
            return _append(kv, cache, cache_scale, block_table, seqused_kv, cu_seqlens_q, rope_table, rope_interleaved,
                           rope_step, q, q_out, layout_q, check_status)
    _pool16(cache, "cache")
    blocks, bs, _, D = cache.shape
    R = rope_rows = rope_at = 0
    if rope_table is not None:
        rope_at = rope_table.data_ptr()
        rope_rows, R = rope_table.shape
        if rope_at % 16:
            raise ValueError("rope_table must start on a 16-byte boundary")
    cu = act_q = None
    if cu_seqlens_q is not None:
        cu = _int32(cu_seqlens_q, device)
    if layout_q == "TND":
        T, S = kv.shape[0], 0
        B = cu.numel() - 1
    else:
        B, S = kv.shape[0], kv.shape[1]
        T = B * S
        if cu is not None:
            cu, act_q = None, (cu[1:] - cu[:-1]).contiguous()
    rows = _rows2d(kv, T, D)
    rows_at = rows.data_ptr()
    table, seq = _int32(block_table, device), _int32(seqused_kv, device)
    heads = q_at = out_at = 0
    if q_out is not None:
        heads, out_at = q_out.shape[-2], q_out.data_ptr()
        if out_at % 16:
            raise ValueError("q_out must start on a 16-byte boundary")
        n = 2 * q_out.numel()
        if rows_at < out_at + n and _rows_meet(rows, T, D, out_at, n):
            raise ValueError("q_out must share nothing with kv")
        if q is None:
            q = q_out  # turned in place
        else:
            d = q.data_ptr() - out_at
            if -n < d < n and n and not (d == 0 and q.is_contiguous()):
                raise ValueError("q_out must be q itself or share nothing with it")
            q = _dense16(q)
        q_at = q.data_ptr()
    args = _append_args(B, T, heads, D, R, int(rope_interleaved), rope_step, rope_rows, blocks, bs, table.shape[1], S,
                        _dtype_code(kv.dtype), _CACHE_DTYPES[cache.dtype], rows.stride(0) if T > 1 else D)
    word = torch.zeros(1, dtype=torch.int32, device=cache.device) if check_status else None
    rc = _lib.load().sas_cache_append(args, rows_at, q_at, out_at, rope_at, table.data_ptr(), _ptr(cu),
                                      _ptr(act_q), seq.data_ptr(), cache.data_ptr(), _ptr(cache_scale), _ptr(word),
                                      _raw_stream(device))
    if rc:
        _lib.check(rc, "sas_cache_append")
    _written(cache, cache_scale, q_out)
    if check_status:
        bits = int(word.item())
        if bits:
            raise RuntimeError(f"sas_cache_append device status: {_lib.status_names(bits)}")


_ops = torch.library.Library("sas_b200", "FRAGMENT")
_ops.define("sharedkv_cache_append(Tensor kv, Tensor(a!) cache, Tensor(b!)? cache_scale, Tensor block_table, "
            "Tensor seqused_kv, Tensor? cu_seqlens_q, Tensor? rope_table, bool rope_interleaved, int rope_step, "
            "Tensor? q, Tensor(c!)? q_out, str layout_q, bool check_status) -> ()")
_ops.impl("sharedkv_cache_append", _append, "CUDA")


@torch.library.register_fake("sas_b200::sharedkv_cache_append")
def _append_fake(kv, cache, cache_scale, block_table, seqused_kv, cu_seqlens_q, rope_table, rope_interleaved, rope_step,
                 q, q_out, layout_q, check_status):
    return None


def sharedkv_cache_append(
    kv: torch.Tensor,
    *,
    cache: torch.Tensor,
    cache_scale: Optional[torch.Tensor] = None,
    block_table: torch.Tensor,
    seqused_kv: torch.Tensor,
    cu_seqlens_q: Optional[torch.Tensor] = None,
    rope_table: Optional[torch.Tensor] = None,
    rope_interleaved: bool = True,
    rope_step: int = 1,
    q: Optional[torch.Tensor] = None,
    q_out: Optional[torch.Tensor] = None,
    layout_q: str = "TND",
    check_status: bool = False,
) -> Optional[torch.Tensor]:
    """Append the new K = V rows of a batch to a paged cache, rotated on the way.

    ``kv`` ``[T, D]`` (or ``[T, 1, D]``; BSND: ``[B, S, D]`` or ``[B, S, 1, D]``), ``bfloat16`` or
    ``float16``; rows may be strided.  ``cache`` ``[blocks, block_size, 1, D]`` in the type of ``kv`` or in
    ``float8_e4m3fn``, then with ``cache_scale`` ``[blocks]`` or ``[blocks, 1]`` fp32: a code stands for
    code x scale of its block.  ``block_table``, ``seqused_kv`` (lengths with the new rows counted in) and
    ``cu_seqlens_q`` are the attention's: row s of a request's n new rows goes to position
    ``seqused_kv - n + s``.  For the compressed pool pass its block table, the compressed lengths and the
    cumulative counts of new compressed rows, with ``rope_step = cmp_ratio`` where a compressed row takes
    the position of its first token.

    ``rope_table`` (``rope_table()``; fp32 ``[positions, R]``) turns the last R dims: row p x ``rope_step``
    for position p; ``rope_interleaved`` pairs dims (2 i, 2 i + 1), else (i, i + R / 2).  ``q`` (``[T, N1, D]``
    or ``[B, S, N1, D]``) is turned by the same angles into ``q_out`` (new when None; ``q`` itself turns in
    place; it shares nothing with ``kv``), which is returned.

    Writes rows of the call's tokens only: padding rows are skipped, and so are rows that their request has no
    place for (negative positions, positions past the angles or the block table, unmapped blocks).
    ``check_status`` synchronises and raises on the latter and on a block without a valid scale.  In an 8-bit cache a block takes the smallest power-of-two scale that its rows
    need when its first row arrives, and raises it when later rows need more; the rows already there are
    then rounded to the new scale.  A block may take rows of one request, and of one place of its table, per
    call.  No host synchronisation; graph-capturable.  No backward pass.
    """
    assert layout_q in ("TND", "BSND"), f"unsupported layout_q={layout_q!r}"
    if not cache.is_cuda:
        raise ValueError("cache must be a CUDA tensor (sas_b200 has no CPU path)")
    _refuse_derivatives("sharedkv_cache_append", kv, cache, cache_scale, rope_table, q, q_out)
    device, kind = cache.get_device(), kv.dtype
    for t in (kv, cache_scale, rope_table, q, q_out):
        if t is not None and t.get_device() != device:
            raise ValueError(f"kv, cache_scale, rope_table, q and q_out must be on {cache.device}")
    if kind is not torch.bfloat16 and kind is not torch.float16:
        raise ValueError(f"kv must be bfloat16 or float16 (got {kind})")
    if cache.dim() != 4 or cache.shape[2] != 1:
        raise ValueError(f"cache must be [blocks, block_size, 1, D] (got {tuple(cache.shape)})")
    blocks, _, _, D = cache.shape
    if D % 16 or D > 1024:
        raise ValueError(f"the head dim must be a multiple of 16 up to 1024 (got {D})")
    rows = kv.shape
    lead = 1 if layout_q == "TND" else 2
    if len(rows) not in (lead + 1, lead + 2) or rows[-1] != D or (len(rows) == lead + 2 and rows[lead] != 1):
        raise ValueError(f"kv must hold one row of {D} per token in layout {layout_q} (got {tuple(rows)})")
    if cache.dtype is torch.float8_e4m3fn:
        if cache_scale is None or cache_scale.dtype is not torch.float32 or cache_scale.numel() != blocks \
                or not cache_scale.is_contiguous():
            raise ValueError("a float8_e4m3fn cache needs cache_scale: contiguous float32, one entry per block")
    elif cache.dtype is not kind:
        raise ValueError(f"cache must be of the type of kv or float8_e4m3fn (got {cache.dtype})")
    elif cache_scale is not None:
        raise ValueError("cache_scale goes with a float8_e4m3fn cache only")
    if lead == 1:
        assert cu_seqlens_q is not None, "cu_seqlens_q is required for TND"
        B = cu_seqlens_q.numel() - 1
    else:
        B = rows[0]
        if cu_seqlens_q is not None and cu_seqlens_q.numel() != B + 1:
            raise ValueError(f"cu_seqlens_q must have {B + 1} entries (got {cu_seqlens_q.numel()})")
    if block_table.dim() != 2 or block_table.shape[0] < B or block_table.shape[1] < 1:
        raise ValueError(f"block_table must be [B>={B}, table_len] (got {tuple(block_table.shape)})")
    if seqused_kv.numel() < B:
        raise ValueError(f"seqused_kv must have {B} entries (got {seqused_kv.numel()})")
    if rope_step < 1:
        raise ValueError("rope_step must be >= 1")
    if rope_table is not None:
        if rope_table.dtype is not torch.float32 or rope_table.dim() != 2 or not rope_table.is_contiguous():
            raise ValueError("rope_table must be a contiguous float32 [positions, rope_dim]")
        if rope_table.shape[1] % 16 or not 0 < rope_table.shape[1] <= D:
            raise ValueError(f"rope_dim must be a multiple of 16 up to {D} (got {rope_table.shape[1]})")
    if q is not None:
        if q.dtype is not kind or q.dim() != lead + 2 or q.shape[:lead] != rows[:lead] or q.shape[-1] != D:
            raise ValueError(f"q must be of kv's type and hold [N1, {D}] per token (got {q.dtype} {tuple(q.shape)})")
        if q_out is None:
            q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
        elif q_out.shape != q.shape or q_out.dtype is not kind or not q_out.is_contiguous():
            raise ValueError("q_out must be contiguous and of q's shape and type")
    elif q_out is not None:
        raise ValueError("q_out goes with q")
    call = (kv, cache, cache_scale, block_table, seqused_kv, cu_seqlens_q, rope_table, bool(rope_interleaved),
            min(int(rope_step), 2**31 - 1), None if q_out is q else q, q_out, layout_q, bool(check_status))
    if _eager(kv, cache, cache_scale, q, q_out):
        _append(*call)
    else:
        torch.ops.sas_b200.sharedkv_cache_append(*call)
    return q_out
