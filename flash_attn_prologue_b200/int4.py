"""A paged cache held in 4 bits: the prologue that writes it (``append_paged_kv_int4``) and what
it stands for (``unpack_int4``). The reference has no cache.

A cache is four tensors (``int4_cache`` makes them): codes ``[pages, page_size, Hk, D/2]`` uint8
and scales ``[pages, page_size, Hk, D/32]`` bfloat16 of K and of V, 72 bytes a row at D = 128
instead of 256. Pages, tables and lengths are those of flash_attn_prologue_b200.paged. A row's
channels are in D/32 groups of 32 (channel c in group (c // 8) % (D/32)), each with a scale s of
five significant bits; a channel is rounded to s times a whole number from -8 to 7.
"""
from typing import Optional, Sequence

import torch
from torch.autograd.graph import increment_version

from . import _lib
from .fused_epilogue import _DeviceGuard
from .gqa import axes_of, call_library, eager, readable, refuse_tangents
from .paged import ATTENTION_HEAD_DIMS, append_args, check_step, checked_cache, no_grad


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
    cache, scale = (t.contiguous() for t in (cache, scale))
    cache, scale = (t if not t.data_ptr() & 15 else t.clone() for t in (cache, scale))
    out = torch.empty((*cache.shape[:-1], dim), dtype=dtype, device=cache.device)
    device = cache.device
    with _DeviceGuard(device):
        _lib.check(_lib.load().flash_prologue_unpack_int4(
            cache.data_ptr(), scale.data_ptr(), out.data_ptr(), out.numel() // dim, dim, _lib.DTYPE_CODES[dtype],
            _lib.raw_stream(device.index)), "flash_prologue_unpack_int4")
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
