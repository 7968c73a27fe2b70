"""paged_attention_int4 with splits that are none: what valid requests get, and no row outside the output."""
import math

import pytest
import torch

import flash_attn_prologue_b200 as fap
from flash_attn_prologue_b200 import _lib, int4
from tests._int4 import Requests4
from tests.test_int4_attention import SCORE, _bound

BF16 = torch.bfloat16
OUT = 4  # the output's address among the packed arguments, behind q's address and strides


def _guarded(monkeypatch, req, q, cu):
    """The call with its rows in the middle of a larger tensor, whose other rows have to stay."""
    T, H, D = q.shape
    room = torch.full((T + 64, H, D), 3.0, dtype=q.dtype, device="cuda")
    call = int4.call_library

    def redirected(name, args, device, scales):
        fields = list(_lib.ATTENTION_ARGS.unpack(args))
        assert fields[OUT + 2:OUT + 4] == [D, H * D]
        fields[OUT] = room[32:].data_ptr()
        call(name, _lib.ATTENTION_ARGS.pack(*fields), device, scales)

    with monkeypatch.context() as m:
        m.setattr(int4, "call_library", redirected)
        _, lse = fap.paged_attention_int4(q, *req.cache, req.table, req.seq_lens, torch.tensor(cu, dtype=torch.int32, device="cuda"),
                                          softmax_scale=0.1, return_lse=True)
    assert (room[:32] == 3).all() and (room[T + 32:] == 3).all()
    return room[32:T + 32], lse


@pytest.mark.gpu
@pytest.mark.parametrize("news", [[20, 20], [1, 1], [100, 60]])
@pytest.mark.parametrize("D", [64, 128])
def test_splits_that_leave_the_rows(news, D, monkeypatch):
    """Starts are cut to the rows, and a request that ends before it begins has none."""
    req = Requests4(news, [150, 170], 8, 2, D, 16, BF16)
    q = req.q.to(BF16)
    T = sum(news)
    for wrong, right in (([0, T + 20, T + 60], [0, T, T]), ([0, -5, T], [0, 0, T]), ([-3, news[0], T + 1], [0, news[0], T]),
                         ([0, 0, 0], [0, 0, 0]), ([2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1], [T, T, T])):
        got, lse = _guarded(monkeypatch, req, q, wrong)
        want, want_lse = _guarded(monkeypatch, req, q, right)
        sure = slice(0, 0) if wrong[0] > T else slice(None)  # (there rows are both in front of the requests and request 1's)
        assert torch.equal(got[sure], want[sure]) and torch.equal(lse[sure], want_lse[sure])
    # rows that only one request has
    half = T // 2
    req.news = [0, T - half]
    got, lse = _guarded(monkeypatch, req, q, [half, half, T])
    exact, bound, exact_lse = _bound(req, q[half:], 0.1, 0)
    assert ((got[half:].double() - exact).abs() <= bound).all() and ((lse[half:].double() - exact_lse).abs() <= SCORE).all()
    assert not got[:half].any() and (lse[:half] == -math.inf).all()


@pytest.mark.gpu
def test_rows_of_one_request_beside_a_split_that_runs_backwards(monkeypatch):
    req = Requests4([20, 20], [50, 50], 8, 2, 64, 16, BF16)
    q = req.q.to(BF16)
    got, lse = _guarded(monkeypatch, req, q, [30, 10, 40])  # rows 30 .. 39 are request 1's alone, 0 .. 9 nobody's
    req.news = [0, 30]
    exact, bound, exact_lse = _bound(req, q[10:], 0.1, 0)
    assert ((got[30:].double() - exact[20:]).abs() <= bound[20:]).all()
    assert ((lse[30:].double() - exact_lse[20:]).abs() <= SCORE).all()
    assert not got[:10].any()
