"""The page tables of a serving step, built on the GPU from the requests' lengths: ``plan_paged_step``.

What append_paged_kv and paged_attention read of a step (page_table, seq_lens, cu_seqlens), and
each new token's request, position and slot, without a word from the host: a captured graph can
plan, append and attend, step after step. The reference has no cache.
"""
from typing import NamedTuple, Optional, Tuple

import torch
from torch.autograd.graph import increment_version

from . import _lib
from .gqa import call_library, eager

MAX_REQUESTS = 8192


class PagedStep(NamedTuple):
    """What plan_paged_step returns, int32 but for the slots (int64)."""
    seq_lens: torch.Tensor    # [B] tokens held after the step
    cu_seqlens: torch.Tensor  # [B + 1] where the requests' new tokens begin
    positions: torch.Tensor   # [tokens] each new token's position in its request
    slots: torch.Tensor       # [tokens] its slot: page * page_size + slot in the page
    requests: torch.Tensor    # [tokens] its request
    free_count: torch.Tensor  # [1] pages left on the stack


def _plan(page_table, seq_lens, new_lens, free_pages, free_count, page_size, tokens, keep):
    device, int32, lens, shape = page_table.device, torch.int32, seq_lens.shape, page_table.shape
    if len(shape) != 2 or lens != shape[:1] or new_lens.shape != lens:
        raise ValueError("page_table must be [B, max_pages], seq_lens and new_lens [B]")
    if free_pages.ndim != 1 or free_count.shape != (1,):
        raise ValueError("free_pages must be a stack [pages] and free_count [1]")
    if keep is not None and keep.shape != lens:
        raise ValueError("keep must be [B]")
    batch, width = shape
    stride = page_table.stride()
    right, shared = page_table.dtype is int32, True
    packed = width <= 1 or stride[1] == 1
    for t in (seq_lens, new_lens, free_pages, free_count) if keep is None else (seq_lens, new_lens, free_pages, free_count, keep):
        right, shared, packed = right and t.dtype is int32, shared and t.device == device, packed and t.is_contiguous()
    if not right:
        raise ValueError("tables, lengths, free_pages and free_count must be int32")
    if not shared:
        raise ValueError("all tensors must share a device")
    if not packed:
        raise ValueError("page_table rows, lengths and free_pages must be contiguous")
    if batch > 1 and width > 0 and stride[0] < width:
        raise ValueError("page_table rows must not share memory")
    if page_size < 8 or page_size & (page_size - 1):
        raise ValueError("page_size must be a power of two, at least 8")
    if batch > MAX_REQUESTS:
        raise ValueError(f"at most {MAX_REQUESTS} requests a step")
    if tokens < 0:
        raise ValueError("tokens must not be negative")
    if device.type != "cuda":
        raise ValueError("the planning kernel runs on CUDA devices only")
    new = seq_lens.new_empty
    out = PagedStep(new(batch), new(batch + 1), new(tokens), new(tokens, dtype=torch.int64), new(tokens), new(1))
    args = _lib.PLAN_ARGS.pack(
        page_table.data_ptr(), stride[0], width, seq_lens.data_ptr(), new_lens.data_ptr(),
        0 if keep is None else keep.data_ptr(), free_pages.data_ptr(), free_pages.shape[0], free_count.data_ptr(),
        out.seq_lens.data_ptr(), out.cu_seqlens.data_ptr(), out.free_count.data_ptr(), out.positions.data_ptr(),
        out.slots.data_ptr(), out.requests.data_ptr(), tokens, batch, page_size)
    call_library("flash_prologue_plan_paged_step", args, device)
    return out


@torch.library.custom_op("flash_prologue::plan_paged_step", mutates_args={"page_table", "free_pages"})
def plan_paged_step_op(
    page_table: torch.Tensor, seq_lens: torch.Tensor, new_lens: torch.Tensor, free_pages: torch.Tensor,
    free_count: torch.Tensor, page_size: int, tokens: int, keep: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    return tuple(_plan(page_table, seq_lens, new_lens, free_pages, free_count, page_size, tokens, keep))


@plan_paged_step_op.register_fake
def _plan_fake(page_table, seq_lens, new_lens, free_pages, free_count, page_size, tokens, keep=None):
    return (torch.empty_like(seq_lens), seq_lens.new_empty(seq_lens.shape[0] + 1), seq_lens.new_empty(tokens),
            seq_lens.new_empty(tokens, dtype=torch.int64), seq_lens.new_empty(tokens), torch.empty_like(free_count))


def plan_paged_step(page_table, seq_lens, new_lens, free_pages, free_count, page_size, tokens, keep=None):
    """Plans a step: pages for the requests that grow, back from those that ended. Returns a PagedStep.

    page_table [B, max_pages], seq_lens [B] tokens held so far, new_lens [B] tokens that join in
    this step, or -1 for a request that has ended; free_pages [pages] is a stack of free pages and
    free_count [1] how many it holds (all int32). First the pages of ended requests go on top of
    the stack, request by request, and these requests are empty; the first ``keep[r]`` of them stay
    out (pages that another request shares). Then requests take the pages they grow by from its
    top, in order, into page_table. Both are changed in place, lengths and count come back as new
    tensors, so a call with the same lengths and count does the same again. ``tokens``: the packed
    new tokens of the step, as many as the rows that the model runs on; rows behind the requests'
    tokens (padding) have request -1, slot -1 and position 0.

    page_size is a power of two, at least 8; at most 8,192 requests. Nothing is read back from the
    GPU. Where free pages run out the table gets -1 (append_paged_kv then leaves such tokens out, and
    their attention is NaN) and so do the tokens' slots. Lengths count such tokens all the same, and
    the entries stay -1 until the request ends, which returns the pages that it has and no other
    entry (nor any that a caller set below 0). A shortage, lengths out of range, and pages that
    the stack has no room for set the device error word.
    """
    args = (page_table, seq_lens, new_lens, free_pages, free_count, page_size, tokens, keep)
    if not eager(page_table, seq_lens, new_lens, free_pages, free_count, keep):
        return PagedStep(*torch.ops.flash_prologue.plan_paged_step(*args))
    out = _plan(*args)
    increment_version((page_table, free_pages))
    return out
