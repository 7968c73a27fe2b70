"""Serving from a paged cache: the prologue on a step's new tokens with K and V
appended to their pages (``append_paged_kv``). The reference ends before
attention and has no cache.

A cache is two tensors ``[pages, page_size, Hk, D]`` (any strides with
contiguous D, so ``[pages, Hk, page_size, D]`` memory is passed transposed) and,
per step, ``page_table [B, max_pages]`` and ``seq_lens [B]`` (int32, the step's
new tokens counted). New tokens of all requests are packed along T in request
order, split by ``cu_seqlens [B + 1]`` (int32); without it each request has one.
Nothing is read back from the GPU, so a step can be captured in a CUDA graph.
"""
from typing import Optional

import torch

from . import _lib
from .fused_epilogue import _DeviceGuard
from .gqa import check_rows, eager, flat_fp32, readable, rotation_of, rows_of


def _check_cache(q, heads, k_cache, v_cache, page_table, seq_lens, cu_seqlens):
    """The cache and its tables, for packed rows q [T, H, D] with ``heads`` key heads."""
    if k_cache.ndim != 4 or v_cache.shape != k_cache.shape or k_cache.shape[3] != q.shape[-1]:
        raise ValueError("caches must be matching [pages, page_size, Hk, D] tensors")
    page_size = k_cache.shape[1]
    if page_size < 8 or page_size & (page_size - 1):
        raise ValueError("page_size must be a power of two, at least 8")
    if k_cache.shape[2] != heads:
        raise ValueError("caches and rows must have the same key heads")
    if k_cache.dtype != q.dtype or v_cache.dtype != q.dtype:
        raise ValueError("caches and rows must share a dtype")
    if k_cache.stride(3) != 1 or v_cache.stride(3) != 1:
        raise ValueError("caches must be contiguous along D")
    if page_table.ndim != 2 or seq_lens.shape != (page_table.shape[0],):
        raise ValueError("page_table must be [B, max_pages] and seq_lens [B]")
    for t in (page_table, seq_lens, cu_seqlens):
        if t is not None and t.dtype != torch.int32:
            raise ValueError("page_table, seq_lens and cu_seqlens must be int32")
    if page_table.shape[1] > 1 and page_table.stride(1) != 1 or not seq_lens.is_contiguous():
        raise ValueError("page_table rows and seq_lens must be contiguous")
    if cu_seqlens is None:
        if q.shape[0] != page_table.shape[0]:
            raise ValueError("without cu_seqlens every request has one token")
    elif cu_seqlens.shape != (page_table.shape[0] + 1,) or not cu_seqlens.is_contiguous():
        raise ValueError("cu_seqlens must be a contiguous [B + 1]")
    for t in (k_cache, v_cache, page_table, seq_lens, cu_seqlens):
        if t is not None and t.device != q.device:
            raise ValueError("all tensors must share a device")


def _cache_of(k_cache, v_cache, page_table, seq_lens, cu_seqlens):
    """flash_prologue_cache."""
    a, b = k_cache.stride(), v_cache.stride()
    return (k_cache.data_ptr(), a[0], a[1], a[2], v_cache.data_ptr(), b[0], b[1], b[2], k_cache.shape[0],
            k_cache.shape[1], page_table.data_ptr(), page_table.stride(0), page_table.shape[1], seq_lens.data_ptr(),
            0 if cu_seqlens is None else cu_seqlens.data_ptr(), page_table.shape[0])


def _no_grad(name, tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError(f"{name} is not differentiable: call it under torch.no_grad()")


def _append(q, k, v, rmsnorm_weight, scales, sin, cos, k_cache, v_cache, page_table, seq_lens, cu_seqlens, eps):
    if q.ndim != 3 or v.shape != k.shape or v.dtype != k.dtype or v.device != k.device:
        raise ValueError("q, k and v must be packed [T,Hq,D], [T,Hk,D], [T,Hk,D]")
    check_rows(q, k, rmsnorm_weight, scales, sin, cos, eps)
    _check_cache(q, k.shape[1], k_cache, v_cache, page_table, seq_lens, cu_seqlens)
    q, k, v = readable(q), readable(k), readable(v)
    q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if q.shape[0]:
        w = None if rmsnorm_weight is None else flat_fp32(rmsnorm_weight)
        s = None if scales is None else scales.contiguous()
        args = _lib.APPEND_ARGS.pack(
            *rows_of(q), *rows_of(k), *rows_of(v), *rows_of(q_out), 0 if w is None else w.data_ptr(),
            0 if s is None else s.data_ptr(), *rotation_of(sin, cos),
            *_cache_of(k_cache, v_cache, page_table, seq_lens, cu_seqlens),
            q.shape[0], q.shape[1], k.shape[1], q.shape[2], _lib.DTYPE_CODES[q.dtype], eps)
        with _DeviceGuard(q.device):
            _lib.check(_lib.load().flash_prologue_append_paged(args, _lib.stream_of(q.device)),
                       "flash_prologue_append_paged")
    return q_out


@torch.library.custom_op("flash_prologue::append_paged_kv", mutates_args={"k_cache", "v_cache"})
def append_paged_kv_op(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, rmsnorm_weight: Optional[torch.Tensor],
    scales: Optional[torch.Tensor], sin: torch.Tensor, cos: torch.Tensor, k_cache: torch.Tensor,
    v_cache: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor,
    cu_seqlens: Optional[torch.Tensor] = None, eps: float = 1e-5,
) -> torch.Tensor:
    return _append(q, k, v, rmsnorm_weight, scales, sin, cos, k_cache, v_cache, page_table, seq_lens, cu_seqlens, eps)


@append_paged_kv_op.register_fake
def _append_fake(q, k, v, rmsnorm_weight, scales, sin, cos, k_cache, v_cache, page_table, seq_lens,
                 cu_seqlens=None, eps=1e-5):
    return torch.empty(q.shape, dtype=q.dtype, device=q.device)


def append_paged_kv(q, k, v, rmsnorm_weight, scales, sin, cos, k_cache, v_cache, page_table, seq_lens,
                    cu_seqlens=None, eps=1e-5):
    """The prologue on a step's new tokens; K and V go to the cache, the Q rows come back.

    q [T,Hq,D], k and v [T,Hk,D] (views of one projection are read in place; BF16, FP16 or
    FP32). Each token is turned by its position in its request, seq_lens - new tokens + its
    index among them, which is also where it is written: slot ``position % page_size`` of page
    ``page_table[request, position // page_size]``. rmsnorm_weight [2,1,D] or None (rotation
    only), scales [Hq,1,1] or None, sin/cos FP32 tables [positions, D/2] as in
    qknorm_rope_scale_gqa. Tokens past the last request come back as zeros and are not
    written; so are tokens whose position, page or table row is out of range, which also set
    the device error word. Not differentiable.
    """
    args = (q, k, v, rmsnorm_weight, scales, sin, cos, k_cache, v_cache, page_table, seq_lens, cu_seqlens)
    _no_grad("append_paged_kv", args)
    call = _append if eager(*args) else torch.ops.flash_prologue.append_paged_kv
    return call(*args, eps)
