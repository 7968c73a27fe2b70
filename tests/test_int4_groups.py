"""paged_attention_int4 over V whose groups of channels have scales far apart: each group is right to its own."""
import pytest
import torch

from tests._int4 import Requests4, groups, values64
from tests.test_int4_attention import _attend, _bound

BF16, FP16 = torch.bfloat16, torch.float16


def _spread(req, top, ratio, seed=0):
    """Scales of V of five significant bits within a factor of two in each group, group g's 2^(ratio g / (G - 1)) below
    the first one's."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    shape = req.scales[1].shape
    size = torch.randint(16, 32, shape, generator=g, device="cuda").double() / 16
    sign = torch.randint(0, 2, shape, generator=g, device="cuda").double() * 2 - 1
    power = torch.exp2(torch.tensor([top - ratio * i // (shape[-1] - 1) for i in range(shape[-1])], device="cuda").double())
    req.scales[1][:] = torch.where(req.scales[1].isnan(), float("nan"), size * sign * power).to(BF16)
    req.v = values64(req.codes[1], req.scales[1])


@pytest.mark.gpu
@pytest.mark.parametrize("news", [[1, 1], [2, 1], [3, 2], [60, 40]])  # tiles of 8, 8, 16 and 128 rows
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype,top,ratio", [(BF16, 20, 12), (BF16, 20, 21), (BF16, 20, 32), (BF16, 100, 180), (FP16, 11, 12),
                                             (FP16, 11, 31)])
def test_small_groups_keep_their_bits(dtype, top, ratio, D, news):
    """The bound of every row, for each group by itself. A weight (probability times scale, 2^7 times as large beside
    the power of two above its group's largest scale) is off by 2^-25 where it is an FP16 subnormal: 2^-32 of that power,
    for codes of up to 8 and sums of probabilities of 1/2 at least, so 2^-27 of the group's largest scale for each key."""
    req = Requests4(news, [500, 700], 8, 2, D, 16, dtype)
    _spread(req, top, ratio)
    q = req.q.to(dtype)
    for scale, window in ((0.1, 0), (0.5, 200)):
        out = _attend(req, q, softmax_scale=scale, window=window)
        exact, bound, _ = _bound(req, q, scale, window)
        largest = req.scales[1].double().abs().nan_to_num(0.0).amax((0, 1, 2))[groups(D)]
        keys = window or 700
        tiny = 2.0 ** -25 if dtype is FP16 else 2.0 ** -134  # half the output's own least step
        off = (out.double() - exact).abs() / (bound + keys * 2.0 ** -27 * largest + tiny)
        assert float(off.max()) <= 1, float(off.max())


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("news", [[2, 1], [4, 4], [60, 40]])
def test_scales_of_later_tokens_leave_no_trace(news, D):
    """A row's bits go by the keys that it sees, however large the scales of those behind it."""
    req = Requests4(news, [300, 90], 8, 2, D, 16, BF16)
    q = req.q.to(BF16)
    clean = _attend(req, q, softmax_scale=0.1)
    for value in (2.0 ** 60, 2.0 ** 120, 0.0):
        for g in (0, D // 32 - 1):
            kept = req.scales[1].clone()
            req.scales[1][(*req.places(0, 299, 300), slice(None), g)] = value
            got = _attend(req, q, softmax_scale=0.1)
            req.scales[1].copy_(kept)
            rows = [i for i in range(sum(news)) if i != news[0] - 1]
            assert torch.equal(got[rows], clean[rows])
            other = groups(D) != g
            assert torch.equal(got[news[0] - 1][:, other], clean[news[0] - 1][:, other])


@pytest.mark.gpu
@pytest.mark.parametrize("news,totals", [([1], [3000]), ([1, 1], [40000, 5]), ([3, 2], [9000, 30])])
def test_groups_that_grow_along_the_keys(news, totals):
    """Largest scales that move late, group by group, in caches that several CTAs share."""
    req = Requests4(news, totals, 16, 4, 128, 64, BF16)
    for r, total in enumerate(totals):
        at = torch.arange(total, device="cuda")
        where = req.places(r, 0, total)
        for g in range(4):
            power = torch.exp2(((at // (61 + 40 * g)) % 23 - 40 + 9 * g).double())
            req.scales[1][(*where, slice(None), g)] = power[:, None].to(BF16)
    req.v = values64(req.codes[1], req.scales[1])
    q = req.q.to(BF16)
    out = _attend(req, q, softmax_scale=0.05)
    exact, bound, _ = _bound(req, q, 0.05, 0)
    largest = req.scales[1].double().abs().nan_to_num(0.0).amax((0, 1, 2))[groups(128)]
    off = (out.double() - exact).abs() / (bound + max(totals) * 2.0 ** -27 * largest)
    assert float(off.max()) <= 1, float(off.max())
