"""The prologue with grouped-query heads and a position per token.

``qknorm_rope_scale_gqa``: RMSNorm of Q (Hq heads) and K (Hk heads, Hq a
multiple of Hk), the split-half rotation of each token's position, Q multiplied
by exp(scales), with its backward; registered as
``flash_prologue::qknorm_rope_scale_gqa`` / ``_gqa_backward``. The reference's
prologue has equal Q and K heads and takes sin/cos rows in token order
(flash_attn_prologue/functional.py:29-70); the arithmetic and the layouts are
its own. The kernels (csrc/gqa_fwd.cu, csrc/gqa_bwd.cu) read strided views in
place. With ``axes`` each rotation pair is turned by the position on an axis of
its own (time, height and width of images and video); ``rotary_axes`` lays out
the usual patterns.
"""
import ctypes
import functools
import math
from typing import Optional, Sequence, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib
from .distributed import active_peer_group
from .fused_epilogue import _DeviceGuard, _grad_view
from .functional import SUPPORTED_CUTE_HEAD_DIMS, _recorded

MAX_HEADS = 512


def check_rows(q, k, rmsnorm_weight, scales, sin, cos, eps):
    """Types, heads, devices and tables that the prologue on rows q/k [..., D] takes.

    q and k are packed [T, H, D] or dense [B, H, N, D] and agree in everything
    but the head count; rmsnorm_weight and scales may be None where the caller
    allows it."""
    qs, ks, dtype = q.shape, k.shape, q.dtype
    if len(qs) not in (3, 4) or len(ks) != len(qs):
        raise ValueError("q/k must both be packed [T,H,D] or dense [B,H,N,D]")
    hq, hk, d = qs[1], ks[1], qs[-1]
    if qs[0] != ks[0] or qs[2:] != ks[2:]:
        raise ValueError("q/k may differ in their head count only")
    if dtype not in _lib.DTYPE_CODES or k.dtype != dtype:
        raise ValueError("q/k must share BF16, FP16, or FP32 dtype")
    if d not in SUPPORTED_CUTE_HEAD_DIMS:
        raise ValueError(f"head dimension must be one of {SUPPORTED_CUTE_HEAD_DIMS}")
    if hk <= 0 or hq <= 0 or hq % hk or hq > MAX_HEADS:
        raise ValueError(f"query heads must be a multiple of the key heads and at most {MAX_HEADS}")
    if not 0 < eps < math.inf:
        raise ValueError("eps must be finite and positive")
    float32 = torch.float32
    device = q.device
    shared = k.device == device and sin.device == device and cos.device == device
    fp32 = sin.dtype is float32 and cos.dtype is float32
    if rmsnorm_weight is not None:
        if rmsnorm_weight.shape != (2, 1, d):
            raise ValueError("weight must be [2,1,D]")
        shared, fp32 = shared and rmsnorm_weight.device == device, fp32 and rmsnorm_weight.dtype is float32
    if scales is not None:
        if scales.shape != (hq, 1, 1):
            raise ValueError("log-scales must be [Hq,1,1]")
        shared, fp32 = shared and scales.device == device, fp32 and scales.dtype is float32
    if sin.ndim != 2 or sin.shape != cos.shape or sin.shape[1] != d // 2:
        raise ValueError("sin/cos must be matching tables [positions, D/2]")
    if not fp32:
        raise ValueError("weights, log-scales, and sin/cos must be FP32")
    if sin.requires_grad or cos.requires_grad:
        raise ValueError("gradients of sin/cos are not implemented")
    if not shared:
        raise ValueError("all tensors must share a device")
    if device.type != "cuda":
        raise ValueError("the prologue kernels run on CUDA devices only")


MAX_AXES = 4


def rotary_axes(sections, interleaved=False):
    """The axis of each rotation pair, for ``axes=``: sections[a] of the D / 2 pairs turn by axis a.

    In blocks (all pairs of axis 0, then those of axis 1, ...), or interleaved: the axes in
    turn, 0, 1, 2, 0, 1, 2, ..., each as long as it has pairs left."""
    sections = [int(n) for n in sections]
    if not 1 <= len(sections) <= MAX_AXES or min(sections) < 0:
        raise ValueError(f"sections must be 1 to {MAX_AXES} counts of pairs")
    if not interleaved:
        return tuple(a for a, n in enumerate(sections) for _ in range(n))
    left, out = list(sections), []
    while any(left):
        for a, n in enumerate(left):
            if n:
                out.append(a)
                left[a] -= 1
    return tuple(out)


def _axis_bytes(axes):
    """The axes' numbers, a byte each: patterns are kept by these, never by objects whose value may change."""
    if not isinstance(axes, torch.Tensor):
        try:
            return bytes(axes if type(axes) is tuple else tuple(axes))
        except TypeError:
            pass
        except ValueError:
            raise ValueError(f"axes must be in 0 .. {MAX_AXES - 1}") from None
    raise ValueError("axes must be a sequence of whole numbers")


@functools.lru_cache(maxsize=64)
def _packed_axes(axes, half):
    """``pairs`` of flash_prologue_axes, and one more than the last axis."""
    if len(axes) != half:
        raise ValueError("axes must name the axis of each of the D / 2 rotation pairs")
    if max(axes) >= MAX_AXES:
        raise ValueError(f"axes must be in 0 .. {MAX_AXES - 1}")
    words = [0] * 4
    for j, a in enumerate(axes):
        words[j // 32] |= a << 2 * (j % 32)
    return tuple(words), max(axes) + 1


def axes_of(axes, positions, q, rows):
    """flash_prologue_axes of rows q packed [T, H, D] or dense [B, H, N, D] and tables of ``rows`` rows; axes None:
    all pairs by the one position a token that positions has."""
    half = q.shape[-1] // 2
    if positions is None:
        raise ValueError("axes take positions")
    dtype, shape, st = positions.dtype, positions.shape, positions.stride()
    if dtype is not torch.int32 and dtype is not torch.int64:
        raise ValueError("positions must be int32 or int64")
    tokens = q.shape[:1] if q.ndim == 3 else (q.shape[0], q.shape[2])
    if axes is None:
        words, count, named = (0, 0, 0, 0), 1, 1
        shape, st = (1, *shape), (0, *st)
    else:
        words, named = _packed_axes(_axis_bytes(axes), half)
        count = shape[0] if shape else 0
    if shape[1:] != tokens and shape[1:] != tokens[1:] or not named <= count <= MAX_AXES or len(shape) < 2:
        raise ValueError("positions must be [axes,T] for packed rows, [axes,N] or [axes,B,N] for dense rows")
    if positions.device != q.device:
        raise ValueError("all tensors must share a device")
    if rows >= 1 << 31:
        raise ValueError("sin/cos tables of several axes must have fewer than 2^31 rows")
    return _lib.AXES_ARGS.pack(positions.data_ptr(), st[0], st[1] if len(st) == 3 else 0, st[-1],
                               64 if dtype is torch.int64 else 32, count, *words)


def _check_positions(positions, q, sin):
    n = q.shape[0] if q.ndim == 3 else q.shape[2]
    if positions is None:
        if sin.shape[0] < n:
            raise ValueError("sin/cos have fewer rows than there are tokens")
        return
    if positions.dtype not in (torch.int32, torch.int64):
        raise ValueError("positions must be int32 or int64")
    if positions.shape != (n,) and (q.ndim == 3 or positions.shape != (q.shape[0], n)):
        raise ValueError("positions must be [T] for packed rows, [N] or [B,N] for dense rows")
    if positions.device != q.device:
        raise ValueError("all tensors must share a device")


def eager(*tensors) -> bool:
    """An eager call on plain tensors, parameters or None (functional._plain_eager, which takes no parameters)."""
    if _recorded():
        return False
    for t in tensors:
        if t is not None and type(t) is not torch.Tensor and type(t) is not torch.nn.Parameter:
            return False
    return True


def refuse_tangents(name, *tensors):
    """Forward-mode derivatives would be lost without a word: neither the kernels nor a
    registered operator (without a rule for them) hands tangents on."""
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError(f"{name} has no forward-mode derivative")


def call_library(name, args, device, *more):
    """Calls entry point ``name`` on ``device``'s current stream, with the device current."""
    function = getattr(_lib.load(), name)
    if device.index == torch._C._cuda_getDevice():
        status = function(args, *more, _lib.raw_stream(device.index))
    else:
        with _DeviceGuard(device):
            status = function(args, *more, _lib.raw_stream(device.index))
    if status:
        _lib.check(status, name)


def readable(t):
    """t itself when the kernels can read its rows in place (d stride 1), else a copy."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def rows_of(t):
    """flash_prologue_rows of a packed [T, H, D] or dense [B, H, N, D] tensor."""
    st = t.stride()
    return (t.data_ptr(), 0, st[1], st[0]) if len(st) == 3 else (t.data_ptr(), st[0], st[1], st[2])


def rotation_of(sin, cos):
    """flash_prologue_rotation of two [positions, D/2] tables."""
    a, b = sin.stride(), cos.stride()
    return (sin.data_ptr(), a[0], a[1], cos.data_ptr(), b[0], b[1], sin.shape[0])


def flat_fp32(t):
    """A parameter as the contiguous, 16-byte aligned array the kernels read."""
    t = t.contiguous()
    return t if not t.data_ptr() & 15 else t.clone()


def _call(name, q, k, w, s, sin, cos, positions, eps, axes, rows, grads=(0, 0), workspace=(0, 0), peers=(0, 0)):
    B, N = (1, q.shape[0]) if q.ndim == 3 else (q.shape[0], q.shape[2])
    if positions is None or axes is not None:
        where = (0, 0, 0, 64)
    else:
        st = positions.stride()
        where = (positions.data_ptr(), st[0] if len(st) == 2 else 0, st[-1],
                 64 if positions.dtype == torch.int64 else 32)
    args = _lib.GQA_ARGS.pack(
        *rows_of(q), *rows_of(k), *rows, w.data_ptr(), s.data_ptr(), *rotation_of(sin, cos), *where, *grads,
        *workspace, *peers, B, N, q.shape[1], k.shape[1], q.shape[-1], _lib.DTYPE_CODES[q.dtype], eps)
    if axes is None:
        call_library(name, args, q.device)
    else:
        call_library(name + "_axes", args, q.device, axes)


def _in_place_rows(t):
    """As ``readable``, with expanded (stride-0) activations made contiguous too."""
    if t.is_contiguous():
        return t
    if t.stride(-1) != 1 or any(n > 1 and st == 0 for n, st in zip(t.shape, t.stride())):
        return t.contiguous()
    return t


def _turned(axes, positions, q, sin):
    """flash_prologue_axes, or None where the one-axis call takes the (checked) positions."""
    if axes is None:
        _check_positions(positions, q, sin)
        return None
    return axes_of(axes, positions, q, sin.shape[0])


def gqa_forward(q, k, rmsnorm_weight, scales, sin, cos, positions, eps, axes=None):
    check_rows(q, k, rmsnorm_weight, scales, sin, cos, eps)
    turn = _turned(axes, positions, q, sin)
    q, k = _in_place_rows(q), _in_place_rows(k)
    q_out, k_out = torch.empty_like(q), torch.empty_like(k)  # dense, in the inputs' memory order
    if q.numel():
        _call("flash_prologue_gqa_fwd", q, k, flat_fp32(rmsnorm_weight), scales.contiguous(), sin, cos, positions, eps,
              turn, (*rows_of(q_out), *rows_of(k_out), *_lib.NO_ROWS, *_lib.NO_ROWS, *_lib.NO_ROWS, *_lib.NO_ROWS))
    return q_out, k_out


_WORKSPACE_BYTES = {}


def _workspace_bytes(heads, dim, device):
    nbytes = _WORKSPACE_BYTES.get((heads, dim, device))
    if nbytes is None:
        out = ctypes.c_size_t(0)
        with _DeviceGuard(device):
            _lib.check(_lib.load().flash_prologue_gqa_bwd_workspace_size(heads, dim, ctypes.byref(out)),
                       "flash_prologue_gqa_bwd_workspace_size")
        nbytes = _WORKSPACE_BYTES[(heads, dim, device)] = int(out.value)
    return nbytes


def gqa_backward(q, k, rmsnorm_weight, scales, sin, cos, positions, grad_q_out, grad_k_out, eps, checked=False,
                 axes=None):
    """``checked``: the arguments but the gradients went through gqa_forward."""
    turn = None
    if not checked:
        check_rows(q, k, rmsnorm_weight, scales, sin, cos, eps)
        turn = _turned(axes, positions, q, sin)
    elif axes is not None:
        turn = axes_of(axes, positions, q, sin.shape[0])
    if grad_q_out.shape != q.shape or grad_k_out.shape != k.shape:
        raise ValueError("upstream gradients must have the shapes of q and k")
    q, k = _in_place_rows(q), _in_place_rows(k)
    grad_q, grad_k = torch.empty_like(q), torch.empty_like(k)
    grad_w = torch.empty_like(rmsnorm_weight, memory_format=torch.contiguous_format)
    grad_s = torch.empty_like(scales, memory_format=torch.contiguous_format)
    gq, gk = _grad_view(grad_q_out, q), _grad_view(grad_k_out, k)
    workspace = grad_w.new_empty(_workspace_bytes(q.shape[1], q.shape[-1], q.device) // 4)
    group = active_peer_group(q.device)
    peers = (0, 0) if group is None else (ctypes.addressof(group.desc), group.next_epoch())
    _call("flash_prologue_gqa_bwd", q, k, flat_fp32(rmsnorm_weight), scales.contiguous(), sin, cos, positions, eps,
          turn, (*_lib.NO_ROWS, *_lib.NO_ROWS, *rows_of(gq), *rows_of(gk), *rows_of(grad_q), *rows_of(grad_k)),
          (grad_w.data_ptr(), grad_s.data_ptr()), (workspace.data_ptr(), 4 * workspace.numel()), peers)
    return grad_q, grad_k, grad_w, grad_s


def _forward(q, k, rmsnorm_weight, scales, sin, cos, positions, eps, axes):
    args = (q, k, rmsnorm_weight, scales, sin, cos, positions, eps)
    return gqa_forward(*args) if axes is None else gqa_forward(*args, axes=axes)


class _GqaEager(torch.autograd.Function):
    """The op for eager calls, without the custom-op dispatch layers (as _CuteEager)."""

    @staticmethod
    def forward(ctx, q, k, rmsnorm_weight, scales, sin, cos, positions, eps, axes):
        ctx.save_for_backward(q, k, rmsnorm_weight, scales, sin, cos, positions)
        ctx.eps, ctx.axes = eps, None if axes is None else tuple(_axis_bytes(axes))  # a list may change until the backward
        return _forward(q, k, rmsnorm_weight, scales, sin, cos, positions, eps, axes)

    @staticmethod
    def backward(ctx, grad_q, grad_k):
        if torch.is_grad_enabled():  # create_graph: the registered op, which refuses second derivatives
            dq, dk, dw, ds = qknorm_rope_scale_gqa_backward_op(*ctx.saved_tensors, grad_q, grad_k, ctx.eps, ctx.axes)
        else:
            more = {} if ctx.axes is None else {"axes": ctx.axes}
            dq, dk, dw, ds = gqa_backward(*ctx.saved_tensors, grad_q, grad_k, ctx.eps, checked=True, **more)
        return dq, dk, dw, ds, None, None, None, None, None


@torch.library.custom_op("flash_prologue::qknorm_rope_scale_gqa", mutates_args=())
def qknorm_rope_scale_gqa_op(
    q: torch.Tensor, k: torch.Tensor, rmsnorm_weight: torch.Tensor, scales: torch.Tensor, sin: torch.Tensor,
    cos: torch.Tensor, positions: Optional[torch.Tensor] = None, eps: float = 1e-5,
    axes: Optional[Sequence[int]] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    refuse_tangents("qknorm_rope_scale_gqa", q, k, rmsnorm_weight, scales, sin, cos)
    return _forward(q, k, rmsnorm_weight, scales, sin, cos, positions, eps, axes)


@qknorm_rope_scale_gqa_op.register_fake
def _gqa_fake(q, k, rmsnorm_weight, scales, sin, cos, positions=None, eps=1e-5, axes=None):
    return torch.empty_like(_in_place_rows(q)), torch.empty_like(_in_place_rows(k))


@torch.library.custom_op("flash_prologue::qknorm_rope_scale_gqa_backward", mutates_args=())
def qknorm_rope_scale_gqa_backward_op(
    q: torch.Tensor, k: torch.Tensor, rmsnorm_weight: torch.Tensor, scales: torch.Tensor, sin: torch.Tensor,
    cos: torch.Tensor, positions: Optional[torch.Tensor], grad_q_out: torch.Tensor, grad_k_out: torch.Tensor,
    eps: float = 1e-5, axes: Optional[Sequence[int]] = None,
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    refuse_tangents("qknorm_rope_scale_gqa_backward", q, k, rmsnorm_weight, scales, sin, cos, grad_q_out, grad_k_out)
    more = {} if axes is None else {"axes": axes}
    return gqa_backward(q, k, rmsnorm_weight, scales, sin, cos, positions, grad_q_out, grad_k_out, eps, **more)


@qknorm_rope_scale_gqa_backward_op.register_fake
def _gqa_backward_fake(q, k, rmsnorm_weight, scales, sin, cos, positions, grad_q_out, grad_k_out, eps=1e-5, axes=None):
    return (torch.empty_like(_in_place_rows(q)), torch.empty_like(_in_place_rows(k)),
            torch.empty_like(rmsnorm_weight, memory_format=torch.contiguous_format),
            torch.empty_like(scales, memory_format=torch.contiguous_format))


def _setup_context(ctx, inputs, output):
    ctx.save_for_backward(*inputs[:7])
    ctx.eps, ctx.axes = inputs[7:]


def _backward(ctx, grad_q, grad_k):
    dq, dk, dw, ds = qknorm_rope_scale_gqa_backward_op(*ctx.saved_tensors, grad_q, grad_k, ctx.eps, ctx.axes)
    return dq, dk, dw, ds, None, None, None, None, None


torch.library.register_autograd("flash_prologue::qknorm_rope_scale_gqa", _backward, setup_context=_setup_context)


def qknorm_rope_scale_gqa(q, k, rmsnorm_weight, scales, sin, cos, positions=None, eps=1e-5, axes=None):
    """qknorm_rope_scale with Hq query heads on Hk key heads and a position per token.

    q/k: packed [T,Hq,D] / [T,Hk,D] or dense [B,Hq,N,D] / [B,Hk,N,D], BF16/FP16/FP32,
    D in (32, 64, 128, 256), Hq a multiple of Hk (at most 512). rmsnorm_weight [2,1,D]
    and scales [Hq,1,1]: FP32. sin/cos: FP32 tables [positions, D/2]; ``positions``
    (int32 or int64; [T], or [N] / [B,N] for dense rows) names each token's row, and
    without it token n has row n. A position outside the tables gives NaN rows and sets
    the device error word. All arithmetic through the final cast is FP32. Differentiable
    in q, k, rmsnorm_weight and scales, once: second and forward-mode derivatives are refused.
    Outputs and gradients keep the inputs' memory order.

    ``axes``: up to four positions a token ([axes,T], [axes,N] or [axes,B,N]), and axes[j], a
    number in 0 .. 3, says which of them turns rotation pair j (channels j and j + D/2) of every
    head; rotary_axes makes the usual patterns. A token with any of its positions outside the
    tables gives NaN rows.
    """
    refuse_tangents("qknorm_rope_scale_gqa", q, k, rmsnorm_weight, scales, sin, cos)
    if eager(q, k, rmsnorm_weight, scales, sin, cos, positions):
        if not torch.is_grad_enabled() or not (q.requires_grad or k.requires_grad or rmsnorm_weight.requires_grad
                                               or scales.requires_grad):
            return _forward(q, k, rmsnorm_weight, scales, sin, cos, positions, eps, axes)
        return _GqaEager.apply(q, k, rmsnorm_weight, scales, sin, cos, positions, eps, axes)
    return torch.ops.flash_prologue.qknorm_rope_scale_gqa(q, k, rmsnorm_weight, scales, sin, cos, positions, eps, axes)
