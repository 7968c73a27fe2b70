"""What may name the axes of the rotation pairs."""
import numpy as np
import pytest
import torch

import flash_attn_prologue_b200 as fap
from flash_attn_prologue_b200 import _lib
from flash_attn_prologue_b200.gqa import axes_of
from tests._paged import tables

ROWS, POSITIONS = torch.zeros(5, 8, 64), torch.zeros(3, 5, dtype=torch.int32)


def _words(axes):
    return _lib.AXES_ARGS.unpack(axes_of(axes, POSITIONS, ROWS, 10))[-4:]


def test_numbers_of_any_whole_type():
    axes = [j % 3 for j in range(32)]
    want = (sum(a << 2 * j for j, a in enumerate(axes)), 0, 0, 0)
    for same in (axes, tuple(axes), np.array(axes), np.array(axes, dtype=np.int8), [np.int64(a) for a in axes], range(0)):
        if len(same):
            assert _words(same) == want


@pytest.mark.parametrize("axes", [
    [0.5] * 32, [1.0] * 32, ["0"] * 32, "0" * 32, [None] * 32, 32, torch.zeros(32, dtype=torch.int64), torch.zeros(32),
    [torch.tensor(0.0)] * 32, [0] * 31 + [torch.tensor(1.0)],
])
def test_nothing_else(axes):
    with pytest.raises(ValueError, match="whole numbers"):
        _words(axes)


def test_numbers_that_change_are_followed():
    """No pattern is kept by the objects that held it."""
    one = torch.tensor(0)
    for axes in (np.zeros(32, dtype=np.int64), [0] * 32, [0, one] + [0] * 30, (0, one) + (0,) * 30):
        one.zero_()
        assert _words(axes)[0] == 0
        if axes[1] is one:
            one.fill_(2)
        else:
            axes[1] = 2
        assert _words(axes)[0] == 2 << 2


def test_numbers_out_of_range():
    for wrong in (-1, 4, 255, 256, 2 ** 70):
        with pytest.raises(ValueError, match="in 0 .. 3"):
            _words([0] * 31 + [wrong])


@pytest.mark.gpu
def test_a_list_that_changes_before_the_backward():
    g = torch.Generator(device="cuda").manual_seed(0)
    q, k = (torch.randn(5, h, 64, generator=g, device="cuda").requires_grad_() for h in (4, 2))
    w, s = torch.ones(2, 1, 64, device="cuda"), torch.zeros(4, 1, 1, device="cuda")
    positions = torch.randint(0, 30, (3, 5), generator=g, device="cuda")
    up = [torch.randn(t.shape, generator=g, device="cuda") for t in (q, k)]
    axes = [j % 3 for j in range(32)]
    grads = []
    for change in (False, True):
        out = fap.qknorm_rope_scale_gqa(q, k, w, s, *tables(30, 64), positions, axes=axes)
        if change:
            axes[:] = [0] * 32
        grads.append(torch.autograd.grad(out, (q, k), up))
    assert all(torch.equal(a, b) for a, b in zip(*grads))
