"""A paged cache held in 4 bits: the prologue that writes it (``append_paged_kv_int4``), the
attention that reads it (``paged_attention_int4``) and what it stands for (``unpack_int4``).
The reference has no cache.

A cache is four tensors (``int4_cache`` makes them): codes ``[pages, page_size, Hk, D/2]`` uint8
and scales ``[pages, page_size, Hk, D/32]`` bfloat16 of K and of V, 72 bytes a row at D = 128
instead of 256. Pages, tables and lengths are those of flash_attn_prologue_b200.paged. A row's
channels are in D/32 groups of 32 (channel c in group (c // 8) % (D/32)), each with a scale s of
five significant bits; a channel is rounded to s times a whole number from -8 to 7.
"""
import ctypes
from typing import Optional, Sequence, Tuple

import torch
from torch.autograd.graph import increment_version

from . import _lib
from .fused_epilogue import _DeviceGuard
from .gqa import MAX_HEADS, axes_of, call_library, eager, readable, refuse_tangents
from .paged import ATTENTION_HEAD_DIMS, LARGEST_SCALE, aligned_rows, append_args, check_step, checked_cache, no_grad


def int4_cache(pages, page_size, kv_heads, dim, device="cuda"):
    """(k_cache, v_cache, k_scale, v_scale) of an empty cache: every slot stands for zeros."""
    if dim not in ATTENTION_HEAD_DIMS:
        raise ValueError(f"head dimension must be one of {ATTENTION_HEAD_DIMS}")
    shape = (pages, page_size, kv_heads)
    codes = [torch.full((*shape, dim // 2), 0x88, dtype=torch.uint8, device=device) for _ in range(2)]
    return (*codes, *(torch.zeros((*shape, dim // 32), dtype=torch.bfloat16, device=device) for _ in range(2)))


def _checked_scales(k_cache, k_scale, v_scale, dim):
    """flash_prologue_scales of a cache's scales."""
    shape, groups, device = k_cache.shape, dim // 32, k_cache.device
    if k_scale.shape != (*shape[:3], groups) or v_scale.shape != k_scale.shape:
        raise ValueError("scales must be matching [pages, page_size, Hk, D / 32] tensors")
    if k_scale.dtype is not torch.bfloat16 or v_scale.dtype is not torch.bfloat16:
        raise ValueError("scales must be bfloat16")
    a, b = k_scale.stride(), v_scale.stride()
    if a[3] != 1 or b[3] != 1:
        raise ValueError("scales must be contiguous along the groups")
    if k_scale.device != device or v_scale.device != device:
        raise ValueError("all tensors must share a device")
    return _lib.SCALES_ARGS.pack(k_scale.data_ptr(), a[0], a[1], a[2], v_scale.data_ptr(), b[0], b[1], b[2])


def _check_rows(q):
    if q.dtype is not torch.bfloat16 and q.dtype is not torch.float16:
        raise ValueError("4-bit caches take BF16 or FP16 rows")
    if q.ndim != 3:
        raise ValueError("q must be packed [T,Hq,D]")
    if q.shape[2] not in ATTENTION_HEAD_DIMS:
        raise ValueError(f"head dimension must be one of {ATTENTION_HEAD_DIMS}")


def _append(q, k, v, rmsnorm_weight, scales, sin, cos, k_cache, v_cache, k_scale, v_scale, page_table, seq_lens,
            cu_seqlens, eps, positions, axes):
    _check_rows(q)
    check_step(q, k, v, rmsnorm_weight, scales, sin, cos, eps)
    cache = checked_cache(q, k.shape[1], k_cache, v_cache, page_table, seq_lens, cu_seqlens, torch.uint8)
    scale_args = _checked_scales(k_cache, k_scale, v_scale, q.shape[2])
    turn = None if positions is None and axes is None else axes_of(axes, positions, q, sin.shape[0])
    q, k, v = readable(q), readable(k), readable(v)
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if q.shape[0]:
        args, _alive = append_args(q, k, v, rmsnorm_weight, scales, sin, cos, cache, q_out, eps)
        call_library("flash_prologue_append_paged_int4", args, q.device, scale_args, turn)
    return q_out


@torch.library.custom_op("flash_prologue::append_paged_kv_int4",
                         mutates_args={"k_cache", "v_cache", "k_scale", "v_scale"})
def append_paged_kv_int4_op(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, rmsnorm_weight: Optional[torch.Tensor],
    scales: Optional[torch.Tensor], sin: torch.Tensor, cos: torch.Tensor, k_cache: torch.Tensor,
    v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, page_table: torch.Tensor,
    seq_lens: torch.Tensor, cu_seqlens: Optional[torch.Tensor] = None, eps: float = 1e-5,
    positions: Optional[torch.Tensor] = None, axes: Optional[Sequence[int]] = None,
) -> torch.Tensor:
    return _append(q, k, v, rmsnorm_weight, scales, sin, cos, k_cache, v_cache, k_scale, v_scale, page_table, seq_lens,
                   cu_seqlens, eps, positions, axes)


@append_paged_kv_int4_op.register_fake
def _append_fake(q, k, v, rmsnorm_weight, scales, sin, cos, k_cache, v_cache, k_scale, v_scale, page_table, seq_lens,
                 cu_seqlens=None, eps=1e-5, positions=None, axes=None):
    return torch.empty(q.shape, dtype=q.dtype, device=q.device)


def append_paged_kv_int4(q, k, v, rmsnorm_weight, scales, sin, cos, k_cache, v_cache, k_scale, v_scale, page_table,
                         seq_lens, cu_seqlens=None, eps=1e-5, positions=None, axes=None):
    """append_paged_kv into a cache held in 4 bits: K and V are rounded to codes and scales.

    BF16 or FP16 rows, D 64 or 128. K is rounded from the FP32 values of the prologue, whose
    statistic is taken in 64 bits here, so codes do not depend on the order of a sum; Q comes
    back as from append_paged_kv. A group of 32 channels that holds an infinity or NaN stands
    for NaN. All else (positions, axes, padding, indices out of range, derivatives) as there;
    counts as an in-place change of the cache's four tensors.
    """
    args = (q, k, v, rmsnorm_weight, scales, sin, cos, k_cache, v_cache, k_scale, v_scale, page_table, seq_lens, cu_seqlens)
    no_grad("append_paged_kv_int4", q, k, v, rmsnorm_weight, scales, sin, cos, k_scale, v_scale)
    if not eager(*args, positions):
        return torch.ops.flash_prologue.append_paged_kv_int4(*args, eps, positions, axes)
    out = _append(*args, eps, positions, axes)
    increment_version((k_cache, v_cache, k_scale, v_scale))
    return out


_WORKSPACE_BYTES = {}


def _workspace_bytes(dim, device):
    out = ctypes.c_size_t(0)
    with _DeviceGuard(device):
        _lib.check(_lib.load().flash_prologue_paged_attention_int4_workspace_size(dim, ctypes.byref(out)),
                   "flash_prologue_paged_attention_int4_workspace_size")
    _WORKSPACE_BYTES[dim, device.index] = int(out.value)
    return int(out.value)


def _attention(q, k_cache, v_cache, k_scale, v_scale, page_table, seq_lens, cu_seqlens, softmax_scale, window, want_lse):
    _check_rows(q)
    tokens, heads, dim = q.shape
    kv_heads = k_cache.shape[2] if k_cache.ndim == 4 else 0
    cache = checked_cache(q, kv_heads, k_cache, v_cache, page_table, seq_lens, cu_seqlens, torch.uint8)
    scale_args = _checked_scales(k_cache, k_scale, v_scale, dim)
    if kv_heads <= 0 or heads <= 0 or heads % kv_heads or heads > MAX_HEADS:
        raise ValueError(f"query heads must be a multiple of the key heads and at most {MAX_HEADS}")
    if not -LARGEST_SCALE < softmax_scale < LARGEST_SCALE:
        raise ValueError("softmax_scale must be finite, and in FP32 too")
    if window < 0:
        raise ValueError("window must be 0 (all keys) or positive")
    device = q.device
    if device.type != "cuda":
        raise ValueError("the attention kernels run on CUDA devices only")
    q = aligned_rows(q, q.stride())
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = q.new_empty((tokens, heads), dtype=torch.float32) if want_lse else None
    if tokens:
        stride = q.stride()
        nbytes = _WORKSPACE_BYTES.get((dim, device.index)) or _workspace_bytes(dim, device)
        workspace = q.new_empty((nbytes + 1) // 2)
        args = _lib.ATTENTION_ARGS.pack(
            q.data_ptr(), 0, stride[1], stride[0], out.data_ptr(), 0, dim, heads * dim,
            lse.data_ptr() if want_lse else 0, *cache, workspace.data_ptr(), nbytes, tokens, heads, kv_heads, dim,
            _lib.DTYPE_CODES[q.dtype], window, softmax_scale)
        call_library("flash_prologue_paged_attention_int4", args, device, scale_args)
    return out, lse


@torch.library.custom_op("flash_prologue::paged_attention_int4", mutates_args=())
def paged_attention_int4_op(
    q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
    page_table: torch.Tensor, seq_lens: torch.Tensor, cu_seqlens: Optional[torch.Tensor] = None,
    softmax_scale: float = 1.0, window: int = 0, want_lse: bool = False,
) -> Tuple[torch.Tensor, torch.Tensor]:
    refuse_tangents("paged_attention_int4", q, k_scale, v_scale)
    out, lse = _attention(q, k_cache, v_cache, k_scale, v_scale, page_table, seq_lens, cu_seqlens, softmax_scale, window,
                          want_lse)
    return out, q.new_empty(0, dtype=torch.float32) if lse is None else lse


@paged_attention_int4_op.register_fake
def _attention_fake(q, k_cache, v_cache, k_scale, v_scale, page_table, seq_lens, cu_seqlens=None, softmax_scale=1.0,
                    window=0, want_lse=False):
    return (torch.empty(q.shape, dtype=q.dtype, device=q.device),
            torch.empty(q.shape[:2] if want_lse else (0,), dtype=torch.float32, device=q.device))


def paged_attention_int4(q, k_cache, v_cache, k_scale, v_scale, page_table, seq_lens, cu_seqlens=None, *,
                         softmax_scale=1.0, window=0, return_lse=False):
    """paged_attention over a cache held in 4 bits, with the exact values that it stands for.

    Arguments, masks, windows, rows without keys, indices out of range and derivatives as in
    paged_attention. A scale that is NaN makes the rows that see its slot NaN (of V: their
    channels of its group), and no others. q has the
    type of the rows that were appended: a cache does not know it, and FP16 rows over one of BF16 rows
    want scales of 2^-20 to 7,936 (chunks are multiplied in FP16, where larger ones overflow). Besides
    the output's rounding there is one of each probability (or probability times scale) to 16 bits; each
    group of channels keeps its own, however large the scales of the others.
    """
    tensors = (q, k_cache, v_cache, k_scale, v_scale, page_table, seq_lens, cu_seqlens)
    no_grad("paged_attention_int4", q, k_scale, v_scale)
    call = _attention if eager(*tensors) else torch.ops.flash_prologue.paged_attention_int4
    out, lse = call(*tensors, softmax_scale, window, return_lse)
    return (out, lse) if return_lse else out


def _packed(t):
    """t, or a copy that is contiguous and starts on 16 bytes."""
    t = t.contiguous()
    return t if not t.data_ptr() & 15 else t.clone()


def _unpack(cache, scale, dtype):
    if cache.ndim < 1 or cache.dtype is not torch.uint8 or scale.dtype is not torch.bfloat16:
        raise ValueError("unpack_int4 takes uint8 codes and bfloat16 scales")
    dim = 2 * cache.shape[-1]
    if dim not in ATTENTION_HEAD_DIMS:
        raise ValueError(f"head dimension must be one of {ATTENTION_HEAD_DIMS}")
    if scale.shape != (*cache.shape[:-1], dim // 32):
        raise ValueError("scales must be [..., D / 32] for codes [..., D / 2]")
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise ValueError("4-bit caches stand for BF16 or FP16 values")
    if scale.device != cache.device:
        raise ValueError("all tensors must share a device")
    if cache.device.type != "cuda":
        raise ValueError("the kernels run on CUDA devices only")
    cache, scale = _packed(cache), _packed(scale)
    device = cache.device
    out = cache.new_empty((*cache.shape[:-1], dim), dtype=dtype)
    args = (cache.data_ptr(), scale.data_ptr(), out.data_ptr(), out.numel() // dim, dim, _lib.DTYPE_CODES[dtype])
    if device.index == torch._C._cuda_getDevice():
        status = _lib.load().flash_prologue_unpack_int4(*args, _lib.raw_stream(device.index))
    else:
        with _DeviceGuard(device):
            status = _lib.load().flash_prologue_unpack_int4(*args, _lib.raw_stream(device.index))
    if status:
        _lib.check(status, "flash_prologue_unpack_int4")
    return out


@torch.library.custom_op("flash_prologue::unpack_int4", mutates_args=())
def unpack_int4_op(cache: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    refuse_tangents("unpack_int4", scale)
    return _unpack(cache, scale, dtype)


@unpack_int4_op.register_fake
def _unpack_fake(cache, scale, dtype):
    return torch.empty((*cache.shape[:-1], 2 * cache.shape[-1]), dtype=dtype, device=cache.device)


def unpack_int4(cache, scale, dtype=torch.bfloat16):
    """The values [..., D] that codes [..., D/2] and scales [..., D/32] stand for, exact in ``dtype``.

    BF16, or FP16 where FP16 rows were appended; for a look at a cache, or to move requests
    into a 16-bit one. Not differentiable.
    """
    no_grad("unpack_int4", scale)
    if eager(cache, scale):
        return _unpack(cache, scale, dtype)
    return torch.ops.flash_prologue.unpack_int4(cache, scale, dtype)
