"""Eager calls without the dispatcher's layers mean what the registered operators mean.

The kernels are replaced by plain functions where only the host's path matters, so most of
this runs on the CPU."""
import pytest
import torch

import flash_attn_prologue_b200 as fap
from flash_attn_prologue_b200 import functional, fused_epilogue, gqa
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
