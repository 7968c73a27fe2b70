"""Eager calls without the dispatcher's layers mean what the registered operators mean.

The kernels are replaced by plain functions where only the host's path matters, so most of
this runs on the CPU."""
import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode

import flash_attn_prologue_b200 as fap
from flash_attn_prologue_b200 import functional, fused_epilogue, gqa, paged
from tests._paged import tables

OPS = torch.ops.flash_prologue


def _rows(device="cpu", heads=4, kv_heads=2):
    g = torch.Generator().manual_seed(0)
    q, k = (torch.randn(3, h, 64, generator=g).to(device) for h in (heads, kv_heads))
    return q, k, torch.ones(2, 1, 64, device=device), torch.zeros(heads, 1, 1, device=device), *tables(3, 64, device)


@pytest.fixture
def plain_gqa(monkeypatch):
    """qknorm_rope_scale_gqa with q^2 and 3 k in place of the kernels' results."""
    monkeypatch.setattr(gqa, "gqa_forward", lambda q, k, w, s, sin, cos, positions, eps: (q * q, 3 * k))

    def backward(q, k, w, s, sin, cos, positions, grad_q, grad_k, eps, checked=False):
        return 2 * q * grad_q, 3 * grad_k, torch.zeros_like(w), torch.zeros_like(s)

    monkeypatch.setattr(gqa, "gqa_backward", backward)


def _step(device="cpu"):
    """append_paged_kv's arguments, and paged_attention's."""
    q, k, w, s, _, _ = _rows(device)
    sin, cos = tables(16, 64, device)
    g = torch.Generator().manual_seed(1)
    caches = [torch.randn(4, 16, 2, 64, generator=g).to(device) for _ in range(2)]
    table = torch.arange(3, dtype=torch.int32, device=device)[:, None]
    lens = torch.full((3,), 9, dtype=torch.int32, device=device)
    return [q, k, k.clone(), w, s, sin, cos, *caches, table, lens, None], [q, *caches, table, lens, None]


@pytest.fixture
def plain_step(monkeypatch):
    """append_paged_kv and paged_attention with 2 q in place of the kernels' results."""
    monkeypatch.setattr(paged, "_append", lambda q, *rest: 2 * q)
    monkeypatch.setattr(paged, "_attention", lambda q, *rest: (2 * q, None))


def _differentiate_twice(call, q):
    out = call(q)[0]
    first = torch.autograd.grad(out.sum(), q, create_graph=True)[0]
    return torch.autograd.grad(first.square().sum() + call(q)[0].sum(), q)


@pytest.mark.parametrize("call", [
    fap.qknorm_rope_scale_gqa,
    lambda *a: OPS.qknorm_rope_scale_gqa(*a, None, 1e-5),
])
def test_second_derivatives_are_refused(call, plain_gqa):
    q, *rest = _rows()
    with pytest.raises(RuntimeError, match="differentiate twice|no autograd formula"):
        _differentiate_twice(lambda q: call(q, *rest), q.requires_grad_())


@pytest.mark.parametrize("call", [
    functional._CuteEager.apply,
    OPS.qknorm_rope_scale_cute,
])
def test_second_derivatives_of_equal_heads_are_refused(call, monkeypatch):
    monkeypatch.setattr(fused_epilogue, "cute_forward", lambda q, k, w, s, sin, cos, eps: (q * q, 3 * k))
    monkeypatch.setattr(fused_epilogue, "cute_backward", lambda q, k, w, s, sin, cos, gq, gk, eps:
                        (2 * q * gq, 3 * gk, torch.zeros_like(w), torch.zeros_like(s)))
    q, k, *rest = _rows(heads=2)
    with pytest.raises(RuntimeError, match="differentiate twice|no autograd formula"):
        _differentiate_twice(lambda q: call(q, k[None], *rest, 1e-5), q[None].requires_grad_())


@pytest.mark.gpu
def test_second_derivatives_on_the_gpu():
    q, *rest = _rows("cuda")
    for call in (lambda q: fap.qknorm_rope_scale_gqa(q, *rest), lambda q: OPS.qknorm_rope_scale_gqa(q, *rest, None, 1e-5),
                 lambda q: fap.qknorm_rope_scale(q, rest[0].repeat_interleave(2, 1), *rest[1:], backend="cute")):
        leaf = q.clone().requires_grad_()
        first = torch.autograd.grad(call(leaf)[0].sum(), leaf)[0]
        again = torch.autograd.grad(call(leaf)[0].sum(), leaf, create_graph=True)[0]
        assert torch.equal(first, again)
        with pytest.raises(RuntimeError, match="differentiate twice|no autograd formula"):
            _differentiate_twice(call, leaf)


def _refuses_tangents(call, args, at):
    with forward_ad.dual_level():
        duals = list(args)
        duals[at] = forward_ad.make_dual(args[at], torch.ones_like(args[at]))
        with pytest.raises(NotImplementedError, match="forward"):
            call(*duals)
        call(*args)  # no tangents in a call: nothing to lose


@pytest.mark.parametrize("at", range(6))
@pytest.mark.parametrize("needs_grad", [False, True])
@pytest.mark.parametrize("call", [fap.qknorm_rope_scale_gqa, lambda *a: OPS.qknorm_rope_scale_gqa(*a, None, 1e-5)])
def test_forward_mode_is_refused(call, needs_grad, at, plain_gqa):
    args = list(_rows())
    if needs_grad:
        args[2 if at != 2 else 3].requires_grad_()
    _refuses_tangents(call, args, at)


@pytest.mark.parametrize("at", range(9))
def test_forward_mode_is_refused_by_the_append(at, plain_step):
    args = _step()[0]
    with torch.no_grad():
        _refuses_tangents(fap.append_paged_kv, args, at)
    _refuses_tangents(fap.append_paged_kv, args, at)


@pytest.mark.parametrize("at", [0, 1, 2])
@pytest.mark.parametrize("call", [fap.paged_attention, OPS.paged_attention])
def test_forward_mode_is_refused_by_the_attention(call, at, plain_step):
    _refuses_tangents(call, _step()[1], at)


def test_forward_mode_transform_is_refused(plain_gqa, plain_step):
    q, *rest = _rows()
    with pytest.raises(NotImplementedError, match="forward"):
        torch.func.jvp(lambda q: fap.qknorm_rope_scale_gqa(q, *rest), (q,), (torch.ones_like(q),))
    q, *rest = _step()[1]
    with pytest.raises(NotImplementedError, match="forward"):
        torch.func.jvp(lambda q: fap.paged_attention(q, *rest), (q,), (torch.ones_like(q),))


class _Names(TorchDispatchMode):
    """Notes the operators called under it."""

    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.names.append(func.name())
        return func(*args, **(kwargs or {}))


def _calls(device):
    rows = _rows(device)
    cute = [rows[0], rows[1].repeat_interleave(2, 1), *rows[2:]]
    append, attend = _step(device)
    if device == "cuda":
        append, attend = ([t.bfloat16() if t is not None and t.ndim >= 3 and t.shape[-1] == 64 and t.shape[0] > 2 else t
                           for t in args] for args in (append, attend))
    return [("qknorm_rope_scale_gqa", fap.qknorm_rope_scale_gqa, rows),
            ("qknorm_rope_scale_cute", lambda *a: fap.qknorm_rope_scale(*a, backend="cute"), cute),
            ("append_paged_kv", fap.append_paged_kv, append), ("paged_attention", fap.paged_attention, attend)]


@pytest.mark.parametrize("which", [0, 2, 3])
def test_dispatch_modes_and_traces_see_the_operators(which, plain_gqa, plain_step):
    name, call, args = _calls("cpu")[which]
    with _Names() as seen:
        call(*args)
    assert f"flash_prologue::{name}" in seen.names
    graph = make_fx(lambda *a: call(*a))(*args)
    assert name in graph.code


@pytest.mark.gpu
@pytest.mark.parametrize("which", range(4))
def test_a_trace_of_real_tensors_replays(which):
    """make_fx on real tensors records the operator, and its graph computes new results from new inputs."""
    name, call, args = _calls("cuda")[which]
    fresh = lambda: [t.clone() if t is not None else None for t in args]  # noqa: E731
    graph = make_fx(lambda *a: call(*a))(*fresh())
    assert name in graph.code
    args = [args[0] * 2 + 1, *args[1:]]
    a, b = call(*fresh()), graph(*fresh())
    for x, y in zip(a if isinstance(a, tuple) else (a,), b if isinstance(b, tuple) else (b,)):
        assert torch.equal(x, y) and x.any()


@pytest.mark.parametrize("call", [fap.append_paged_kv, lambda *a: OPS.append_paged_kv(*a, 1e-5)])
def test_an_append_counts_as_a_change_of_the_caches(call, plain_step):
    args = _step()[0]
    caches = args[7:9]
    weight = torch.ones(64, requires_grad=True)
    saved = [(c * weight).sum() for c in caches]  # the caches are kept for the backward
    with torch.no_grad():
        call(*args)
    assert [c._version for c in caches] == [1, 1]
    for loss in saved:
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    with torch.inference_mode():
        args = _step()[0]
        call(*args)  # inference tensors have no version to count


@pytest.mark.gpu
def test_an_append_on_the_gpu_counts_as_a_change():
    _, call, args = _calls("cuda")[2]
    weight = torch.ones(64, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    loss = (args[8][1:] * weight).sum()  # a view's counter is its base's
    call(*args)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        call(*[t.clone() if t is not None else None for t in args])


class _Noting(torch.Tensor):
    """A tensor subclass that notes the operators called with it."""

    names = []

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        cls.names.append(str(func))
        return super().__torch_function__(func, types, args, kwargs or {})


@pytest.mark.parametrize("which,at", [(w, i) for w, n in ((0, 6), (2, 12), (3, 6)) for i in range(n)])
def test_a_tensor_subclass_in_any_place_takes_the_operator(which, at, plain_gqa, plain_step):
    name, call, args = _calls("cpu")[which]
    args = list(args)
    if args[at] is None:  # cu_seqlens
        args[at] = torch.arange(4, dtype=torch.int32)
    args[at] = args[at].as_subclass(_Noting)
    _Noting.names.clear()
    call(*args)
    assert any(f"flash_prologue.{name}" in n for n in _Noting.names)
