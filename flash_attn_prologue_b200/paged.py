"""Serving from a paged cache: the prologue on a step's new tokens with K and V
appended to their pages (``append_paged_kv``), and the attention of those tokens
over the cache (``paged_attention``). The reference ends before attention and
has no cache.

A cache is two tensors ``[pages, page_size, Hk, D]`` (any strides with
contiguous D, so ``[pages, Hk, page_size, D]`` memory is passed transposed) and,
per step, ``page_table [B, max_pages]`` and ``seq_lens [B]`` (int32, the step's
new tokens counted). New tokens of all requests are packed along T in request
order, split by ``cu_seqlens [B + 1]`` (int32); without it each request has one.
Nothing is read back from the GPU, so a step can be captured in a CUDA graph.
"""
import ctypes
import math
from typing import Optional, Sequence, Tuple

import torch
from torch.autograd.graph import increment_version

from . import _lib
from .fused_epilogue import _DeviceGuard
from .gqa import (MAX_HEADS, axes_of, call_library, check_rows, eager, flat_fp32, readable, refuse_tangents, rotation_of,
                  rows_of)


def checked_cache(q, heads, k_cache, v_cache, page_table, seq_lens, cu_seqlens, dtype=None):
    """flash_prologue_cache of the cache and its tables, once they fit the packed rows
    q [T, H, D] with ``heads`` key heads; dtype uint8: codes of 4 bits."""
    ks, device = k_cache.shape, q.device
    if dtype is None:
        dtype, dim = q.dtype, q.shape[2]
    else:
        dim = q.shape[2] // 2
    if len(ks) != 4 or v_cache.shape != ks or ks[3] != dim:
        raise ValueError("caches must be matching [pages, page_size, Hk, D] tensors" if dtype is not torch.uint8
                         else "caches must be matching [pages, page_size, Hk, D / 2] tensors")
    pages, page_size, kv_heads, _ = ks
    if page_size < 8 or page_size & (page_size - 1):
        raise ValueError("page_size must be a power of two, at least 8")
    if kv_heads != heads:
        raise ValueError("caches and rows must have the same key heads")
    if k_cache.dtype is not dtype or v_cache.dtype is not dtype:
        raise ValueError("caches and rows must share a dtype" if dtype is not torch.uint8 else "caches must be uint8")
    a, b = k_cache.stride(), v_cache.stride()
    if a[3] != 1 or b[3] != 1:
        raise ValueError("caches must be contiguous along D")
    table, rows = page_table.shape, page_table.stride()
    if len(table) != 2 or seq_lens.shape != table[:1]:
        raise ValueError("page_table must be [B, max_pages] and seq_lens [B]")
    batch, width = table
    int32 = torch.int32
    if page_table.dtype is not int32 or seq_lens.dtype is not int32:
        raise ValueError("page_table, seq_lens and cu_seqlens must be int32")
    if (width > 1 and rows[1] != 1) or not seq_lens.is_contiguous():
        raise ValueError("page_table rows and seq_lens must be contiguous")
    shared = (k_cache.device == device and v_cache.device == device and page_table.device == device
              and seq_lens.device == device)
    if cu_seqlens is None:
        if q.shape[0] != batch:
            raise ValueError("without cu_seqlens every request has one token")
        starts = 0
    else:
        if cu_seqlens.dtype is not int32:
            raise ValueError("page_table, seq_lens and cu_seqlens must be int32")
        if cu_seqlens.shape != (batch + 1,) or not cu_seqlens.is_contiguous():
            raise ValueError("cu_seqlens must be a contiguous [B + 1]")
        shared = shared and cu_seqlens.device == device
        starts = cu_seqlens.data_ptr()
    if not shared:
        raise ValueError("all tensors must share a device")
    return (k_cache.data_ptr(), a[0], a[1], a[2], v_cache.data_ptr(), b[0], b[1], b[2], pages, page_size,
            page_table.data_ptr(), rows[0], width, seq_lens.data_ptr(), starts, batch)


def no_grad(name, *tensors):
    refuse_tangents(name, *tensors)
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise ValueError(f"{name} is not differentiable: call it under torch.no_grad()")


def append_args(q, k, v, rmsnorm_weight, scales, sin, cos, cache, q_out, eps):
    """flash_prologue_append_args, and the tensors that have to live until the call."""
    tokens, heads, dim = q.shape
    w = None if rmsnorm_weight is None else flat_fp32(rmsnorm_weight)
    s = None if scales is None else scales.contiguous()
    return _lib.APPEND_ARGS.pack(
        *rows_of(q), *rows_of(k), *rows_of(v), q_out.data_ptr(), 0, dim, heads * dim,
        0 if w is None else w.data_ptr(), 0 if s is None else s.data_ptr(), *rotation_of(sin, cos), *cache, tokens,
        heads, k.shape[1], dim, _lib.DTYPE_CODES[q.dtype], eps), (w, s)


def check_step(q, k, v, rmsnorm_weight, scales, sin, cos, eps):
    """The rows of a step's new tokens, and what turns and scales them."""
    if q.ndim != 3 or v.shape != k.shape or v.dtype != k.dtype or v.device != k.device:
        raise ValueError("q, k and v must be packed [T,Hq,D], [T,Hk,D], [T,Hk,D]")
    check_rows(q, k, rmsnorm_weight, scales, sin, cos, eps)


def _append(q, k, v, rmsnorm_weight, scales, sin, cos, k_cache, v_cache, page_table, seq_lens, cu_seqlens, eps,
            positions=None, axes=None):
    check_step(q, k, v, rmsnorm_weight, scales, sin, cos, eps)
    cache = checked_cache(q, k.shape[1], k_cache, v_cache, page_table, seq_lens, cu_seqlens)
    turn = None if positions is None and axes is None else axes_of(axes, positions, q, sin.shape[0])
    q, k, v = readable(q), readable(k), readable(v)
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    if q.shape[0]:
        args, _alive = append_args(q, k, v, rmsnorm_weight, scales, sin, cos, cache, q_out, eps)
        if turn is None:
            call_library("flash_prologue_append_paged", args, q.device)
        else:
            call_library("flash_prologue_append_paged_axes", args, q.device, turn)
    return q_out


@torch.library.custom_op("flash_prologue::append_paged_kv", mutates_args={"k_cache", "v_cache"})
def append_paged_kv_op(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, rmsnorm_weight: Optional[torch.Tensor],
    scales: Optional[torch.Tensor], sin: torch.Tensor, cos: torch.Tensor, k_cache: torch.Tensor,
    v_cache: torch.Tensor, page_table: torch.Tensor, seq_lens: torch.Tensor,
    cu_seqlens: Optional[torch.Tensor] = None, eps: float = 1e-5, positions: Optional[torch.Tensor] = None,
    axes: Optional[Sequence[int]] = None,
) -> torch.Tensor:
    return _append(q, k, v, rmsnorm_weight, scales, sin, cos, k_cache, v_cache, page_table, seq_lens, cu_seqlens, eps,
                   positions, axes)


@append_paged_kv_op.register_fake
def _append_fake(q, k, v, rmsnorm_weight, scales, sin, cos, k_cache, v_cache, page_table, seq_lens,
                 cu_seqlens=None, eps=1e-5, positions=None, axes=None):
    return torch.empty(q.shape, dtype=q.dtype, device=q.device)


def append_paged_kv(q, k, v, rmsnorm_weight, scales, sin, cos, k_cache, v_cache, page_table, seq_lens,
                    cu_seqlens=None, eps=1e-5, positions=None, axes=None):
    """The prologue on a step's new tokens; K and V go to the cache, the Q rows come back.

    q [T,Hq,D], k and v [T,Hk,D] (views of one projection are read in place; BF16, FP16 or
    FP32). Each token is turned by its position in its request, seq_lens - new tokens + its
    index among them, which is also where it is written: slot ``position % page_size`` of page
    ``page_table[request, position // page_size]``. rmsnorm_weight [2,1,D] or None (rotation
    only), scales [Hq,1,1] or None, sin/cos FP32 tables [positions, D/2] as in
    qknorm_rope_scale_gqa. ``positions`` [T] turns tokens by other positions than those they are
    written at, and with ``axes`` (as in qknorm_rope_scale_gqa) positions are [axes,T].
    Tokens past the last request, or before the first where cu_seqlens
    begin above 0, come back as zeros and are not written; so are tokens whose position, page or table row is out of range, which also set
    the device error word. Counts as an in-place change of both caches. Not differentiable:
    tensors that require gradients (where they are enabled) or carry tangents are refused.
    """
    args = (q, k, v, rmsnorm_weight, scales, sin, cos, k_cache, v_cache, page_table, seq_lens, cu_seqlens)
    no_grad("append_paged_kv", q, k, v, rmsnorm_weight, scales, sin, cos, k_cache, v_cache)
    if not eager(*args, positions):
        return torch.ops.flash_prologue.append_paged_kv(*args, eps, positions, axes)
    out = _append(*args, eps, positions, axes)
    increment_version((k_cache, v_cache))  # as the registered op: autograd refuses what it saved of the caches before
    return out


ATTENTION_HEAD_DIMS = (64, 128)
LARGEST_SCALE = 2.0 ** 127  # times log2(e) it is still an FP32 number
_WORKSPACE_BYTES = {}


def _workspace_bytes(dim, device):
    out = ctypes.c_size_t(0)
    with _DeviceGuard(device):
        _lib.check(_lib.load().flash_prologue_paged_attention_workspace_size(dim, ctypes.byref(out)),
                   "flash_prologue_paged_attention_workspace_size")
    _WORKSPACE_BYTES[dim, device.index] = int(out.value)
    return int(out.value)


def aligned_rows(q, stride):
    """q, or a copy whose rows start on 16 bytes and are contiguous along D."""
    if stride[2] == 1 and not (stride[0] | stride[1]) & 7 and not q.data_ptr() & 15:
        return q
    return q.contiguous().clone()


def _attention(q, k_cache, v_cache, page_table, seq_lens, cu_seqlens, softmax_scale, window, want_lse):
    shape, dtype = q.shape, q.dtype
    if len(shape) != 3:
        raise ValueError("q must be packed [T,Hq,D]")
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise ValueError("paged attention takes BF16 or FP16")
    tokens, heads, dim = shape
    if dim not in ATTENTION_HEAD_DIMS:
        raise ValueError(f"head dimension must be one of {ATTENTION_HEAD_DIMS}")
    kv_heads = k_cache.shape[2] if k_cache.ndim == 4 else 0
    cache = checked_cache(q, kv_heads, k_cache, v_cache, page_table, seq_lens, cu_seqlens)
    if kv_heads <= 0 or heads <= 0 or heads % kv_heads or heads > MAX_HEADS:
        raise ValueError(f"query heads must be a multiple of the key heads and at most {MAX_HEADS}")
    if not -LARGEST_SCALE < softmax_scale < LARGEST_SCALE:
        raise ValueError("softmax_scale must be finite, and in FP32 too")
    if window < 0:
        raise ValueError("window must be 0 (all keys) or positive")
    device = q.device
    if device.type != "cuda":
        raise ValueError("the attention kernels run on CUDA devices only")
    stride = q.stride()
    q = aligned_rows(q, stride)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = q.new_empty((tokens, heads), dtype=torch.float32) if want_lse else None
    if tokens:
        stride = q.stride()
        nbytes = _WORKSPACE_BYTES.get((dim, device.index)) or _workspace_bytes(dim, device)
        workspace = q.new_empty((nbytes + 1) // 2)
        args = _lib.ATTENTION_ARGS.pack(
            q.data_ptr(), 0, stride[1], stride[0], out.data_ptr(), 0, dim, heads * dim,
            lse.data_ptr() if want_lse else 0, *cache, workspace.data_ptr(), nbytes, tokens, heads, kv_heads, dim,
            _lib.DTYPE_CODES[dtype], window, softmax_scale)
        call_library("flash_prologue_paged_attention", args, device)
    return out, lse


@torch.library.custom_op("flash_prologue::paged_attention", mutates_args=())
def paged_attention_op(
    q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
    seq_lens: torch.Tensor, cu_seqlens: Optional[torch.Tensor] = None, softmax_scale: float = 1.0, window: int = 0,
    want_lse: bool = False,
) -> Tuple[torch.Tensor, torch.Tensor]:
    refuse_tangents("paged_attention", q, k_cache, v_cache)
    out, lse = _attention(q, k_cache, v_cache, page_table, seq_lens, cu_seqlens, softmax_scale, window, want_lse)
    return out, q.new_empty(0, dtype=torch.float32) if lse is None else lse


@paged_attention_op.register_fake
def _attention_fake(q, k_cache, v_cache, page_table, seq_lens, cu_seqlens=None, softmax_scale=1.0, window=0,
                    want_lse=False):
    return (torch.empty(q.shape, dtype=q.dtype, device=q.device),
            torch.empty(q.shape[:2] if want_lse else (0,), dtype=torch.float32, device=q.device))


def paged_attention(q, k_cache, v_cache, page_table, seq_lens, cu_seqlens=None, *, softmax_scale=1.0, window=0,
                    return_lse=False):
    """Attention of a step's new tokens over a paged cache that holds them already.

    q [T,Hq,D] (BF16 or FP16, D 64 or 128; Hq a multiple of the cache's heads): the new tokens
    of all requests as append_paged_kv returns them. A token at position p of its request
    attends to the cached positions 0 .. p, or p - window + 1 .. p with a window; query head h
    reads key head h // (Hq / Hk). softmax_scale multiplies the scores: 1 by default, since the
    prologue's exp(scales) has scaled Q (it has to be finite in FP32). Returns the rows [T,Hq,D] in q's type and, with
    return_lse, the scores' log-sum-exp [T,Hq] in FP32. A token that sees no key, padding on
    either side of the requests included, gets zeros (lse -inf); one whose page is outside the
    cache gets NaN, as may tokens of its request near it, and the device error word is set.
    What lies in slots that a token does not see never reaches it. Not differentiable: as
    append_paged_kv.
    """
    tensors = (q, k_cache, v_cache, page_table, seq_lens, cu_seqlens)
    no_grad("paged_attention", q, k_cache, v_cache)
    call = _attention if eager(*tensors) else torch.ops.flash_prologue.paged_attention
    out, lse = call(*tensors, softmax_scale, window, return_lse)
    return (out, lse) if return_lse else out
