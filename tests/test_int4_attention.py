"""paged_attention_int4 against plain attention in 64 bits over the values that the cache stands for.

Bounds as for 16-bit caches: one cast of the output, one of each probability (or probability
times scale) to the rows' type or FP16, FP32 scores of exact products. Where codes are added up
as code + 8 and 8 sum p s is taken off again, the sums are as large as LIFT = 8 sum p |s| whatever
the codes: a warp adds the products of at most 128 steps of 16 keys in sequence at these sizes, and
each addition is off by at most 2^-23 of the sum (one rounding, one cut inside the product), 2^-16
of LIFT in all.
"""
import math

import pytest
import torch

import flash_attn_prologue_b200 as fap
from flash_attn_prologue_b200 import _lib
from tests._int4 import Requests4, groups, values64
from tests._paged import HALF_ULP, tables
from tests.test_paged_attention import SCORE, _exact

BF16, FP16 = torch.bfloat16, torch.float16


class _Lifted:
    """The same requests with 8 |s| in place of every value."""

    def __init__(self, req):
        self.news, self.totals, self.k, self.places = req.news, req.totals, req.k, req.places
        self.v = 8 * req.scales[1].double().abs()[..., groups(req.k.shape[-1])]


def _bound(req, q, scale, window, rows=None):
    """(exact rows, their bound, exact lse)."""
    exact, size, lse = _exact(req, q, scale, window, rows)
    lift = _exact(_Lifted(req), q, scale, window, rows)[0]
    u = HALF_ULP[q.dtype]
    return exact, u * exact.abs() + (u + SCORE) * size + 2.0 ** -16 * lift + 1e-30, lse


def _attend(req, q, decode=False, **more):
    return fap.paged_attention_int4(q, *req.cache, req.table, req.seq_lens, None if decode else req.cu, **more)


def _check(req, q, scale=None, window=0, decode=False, rows=None):
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    out, lse = _attend(req, q, decode, softmax_scale=scale, window=window, return_lse=True)
    assert out.shape == q.shape and out.dtype == q.dtype and lse.shape == q.shape[:2]
    exact, bound, exact_lse = _bound(req, q, scale, window, rows)
    pick = slice(None) if rows is None else rows
    off = ((out.double() - exact).abs() / bound)[pick]
    assert not off.numel() or float(off.max()) <= 1, float(off.max())
    far = torch.where(exact_lse.isinf(), (lse != exact_lse).double(), (lse.double() - exact_lse).abs())[pick]
    assert not far.numel() or float(far.max()) <= SCORE
    return out, lse


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hk", [(8, 8), (32, 8), (16, 1), (40, 2), (7, 1)])
@pytest.mark.parametrize("page,window", [(8, 0), (32, 0), (16, 100), (128, 1)])
def test_single_tokens(Hq, Hk, page, window, D, dtype):
    totals = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 500, 1000]
    req = Requests4([1] * len(totals), totals, Hq, Hk, D, page, dtype, page == 32, seed=page)
    _check(req, req.q.to(dtype), window=window, decode=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hk", [(8, 2), (4, 4), (15, 5), (7, 1), (32, 1), (48, 2)])
@pytest.mark.parametrize("page,hnd,window", [(16, False, 0), (8, True, 50), (64, True, 0), (256, False, 17)])
def test_chunks(Hq, Hk, page, hnd, window, D, dtype):
    req = Requests4([1, 0, 7, 33, 2, 20], [1, 12, 7, 300, 130, 70], Hq, Hk, D, page, dtype, hnd, seed=page)
    _check(req, req.q.to(dtype), window=window)


@pytest.mark.gpu
@pytest.mark.parametrize("news,totals", [
    ([1] * 9, [1, 64, 100, 128, 129, 192, 200, 255, 256]),
    ([2, 0, 1, 3], [200, 256, 1, 3]),
    ([1] * 400, [1 + i % 250 for i in range(400)]),
])
@pytest.mark.parametrize("Hq,Hk,D,window", [(8, 2, 128, 0), (16, 16, 64, 70), (48, 2, 64, 0)])
def test_short_caches(news, totals, Hq, Hk, D, window):
    req = Requests4(news, totals, Hq, Hk, D, 64, FP16)
    assert req.table.shape[1] * 64 <= 256
    _check(req, req.q.half(), window=window, rows=list(range(0, sum(news), 1 + sum(news) // 60)))


@pytest.mark.gpu
@pytest.mark.parametrize("news,totals", [
    ([1], [40000]),
    ([1, 1], [70001, 3]),
    ([5], [20000]),
    ([300], [5000]),
    ([1000, 1, 0, 40], [1000, 9000, 5, 2040]),
    ([1] * 300, [1 + 7 * (i % 40) for i in range(300)]),
    ([i % 3 for i in range(290)], [3 + i for i in range(290)]),
    ([3, 0, 5, 1], [20000, 7000, 12345, 5]),
    ([2, 1, 0, 3] * 35, [300 + 9 * i for i in range(140)]),
])
@pytest.mark.parametrize("window", [0, 777])
def test_long_and_many(news, totals, window):
    req = Requests4(news, totals, 16, 4, 128, 16, BF16)
    rows = None if sum(news) <= 350 else list(range(0, sum(news), 61))
    _check(req, req.q.to(BF16), window=window, rows=rows)


@pytest.mark.gpu
@pytest.mark.parametrize("news,totals", [
    ([900, 0, 1300, 5], [900, 40, 2000, 1100]),
    ([1] * 300 + [1500], [9] * 300 + [1500]),
    ([40, 3, 25, 1], [3000, 2500, 2900, 900]),
])
@pytest.mark.parametrize("Hq,Hk,D,dtype,window", [(32, 2, 64, FP16, 0), (32, 2, 128, BF16, 100), (12, 4, 128, FP16, 0)])
def test_many_and_few_tiles(news, totals, Hq, Hk, D, dtype, window):
    req = Requests4(news, totals, Hq, Hk, D, 16, dtype)
    rows = None if sum(news) <= 350 else list(range(0, sum(news), 37)) + [sum(news) - 1]
    _check(req, req.q.to(dtype), window=window, rows=rows)


@pytest.mark.gpu
@pytest.mark.parametrize("news,totals", [([4, 3], [2, 5]), ([6, 2], [0, 2]), ([40], [10]), ([200], [30])])
def test_rows_without_keys_are_zero(news, totals):
    req = Requests4(news, totals, 8, 2, 64, 8, BF16)
    out, lse = _check(req, req.q.to(BF16))
    empty = max(0, news[0] - totals[0])
    assert not out[:empty].any() and (lse[:empty] == -math.inf).all()


@pytest.mark.gpu
@pytest.mark.parametrize("chunk", [1, 12, 200])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_unseen_scales_never_reach_a_row(value, D, chunk):
    """A NaN or infinite scale of a later token, or of one before the window, changes nothing; one that is seen
    makes its group NaN (V) or the row (K)."""
    req = Requests4([chunk, 3], [chunk + 90, 30], 8, 2, D, 16, FP16)
    q, window = req.q.half(), 64

    def call():
        return _attend(req, q, softmax_scale=0.1, window=window)

    clean = call()
    lost = {chunk + 90 - 4, 5, 90 + chunk // 2 - 1}
    position = torch.arange(90, 90 + chunk, device="cuda")
    sees = torch.zeros(chunk, dtype=torch.bool, device="cuda")
    for at in lost:
        sees |= (position >= at) & (position - window < at)
    hidden = torch.cat((~sees, torch.ones(3, dtype=torch.bool, device="cuda")))
    for which, cache in enumerate(req.scales):
        kept = cache.clone()
        for at in lost:
            where = req.places(0, at, at + 1)
            cache[(*where, slice(None), 0)] = value
        got = call()
        assert torch.equal(got[hidden], clean[hidden])
        mine = groups(D) == 0
        if which == 1:
            assert got[:chunk][sees][..., mine].isnan().all()
            other = (got[:chunk][sees][..., ~mine].double() - clean[:chunk][sees][..., ~mine].double()).abs()
            assert not other.numel() or float(other.max()) < 2.0 ** -8 * float(clean.double().abs().max())
        elif math.isnan(value):  # (infinite scales are not of the format: only unseen ones mean something)
            assert got[:chunk][sees].isnan().all()
        cache.copy_(kept)


@pytest.mark.gpu
@pytest.mark.parametrize("news", [[1, 1], [3, 40], [1, 300]])
@pytest.mark.parametrize("D", [64, 128])
def test_scales_of_many_sizes(news, D):
    """Scales of V from 2^-90 to 2^60 and zeros, in one cache: the largest carry the output, each row is right to them."""
    req = Requests4(news, [500, 700], 8, 2, D, 16, BF16)
    g = torch.Generator(device="cuda").manual_seed(3)
    shape = req.scales[1].shape
    for low, high in ((-90, -60), (-12, 12), (40, 60)):
        power = torch.randint(low, high + 1, shape, generator=g, device="cuda")
        req.scales[1][:] = torch.where(req.scales[1].isnan(), math.nan, torch.exp2(power.double())).to(BF16)
        req.scales[1][torch.rand(shape, generator=g, device="cuda") < 0.1] = 0.0
        req.v = values64(req.codes[1], req.scales[1])
        q = req.q.to(BF16)
        out = _attend(req, q, softmax_scale=0.1)
        exact, bound, _ = _bound(req, q, 0.1, 0)
        size = _exact(req, q, 0.1, 0)[1]
        # weights below 2^-14 of the largest scale's keep less than FP16's bits: 2^-25 of its row's sum of |v|
        assert ((out.double() - exact).abs() <= bound + 2.0 ** -24 * size.amax(-1, keepdim=True)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("news", [[1, 1], [3, 40], [1, 300]])
@pytest.mark.parametrize("size", [2.0 ** -100, 2.0 ** -20, 2.0 ** 30, 2.0 ** 100])
def test_queries_of_any_size(news, size):
    """Rows of Q far from 1, the scale taking scores back; a row of zeros, and one with a value 2^12 times the others."""
    req = Requests4(news, [200, 400], 8, 2, 128, 16, BF16)
    q = req.q.clone()
    q[0, 1] = 0
    q[-1, 2, 5] *= 2.0 ** 6
    _check(req, (q * size).to(BF16), scale=0.05 / size)


@pytest.mark.gpu
@pytest.mark.parametrize("news", [[1, 1], [3, 40], [2, 300]])
def test_large_scores_pick_one_key_and_scales(news):
    req = Requests4(news, [200, 400], 8, 2, 64, 16, BF16)
    q = req.q.to(BF16)
    # the largest score's lead makes it the only term; scores up to 2^13 are exact to 2^-11 of one
    out = _attend(req, q, softmax_scale=100.0)
    exact, size, _ = _exact(req, q, 100.0, 0)
    assert ((out.double() - exact).abs() <= 2.0 ** -8 * exact.abs() + 2.0 ** -5 * size.amax(-1, keepdim=True)).all()
    for scale in (0.0, -0.2, 1e-50, 1e-44, 1e-39, -1e-50):
        _check(req, q, scale=scale)


@pytest.mark.gpu
def test_queries_that_are_not_finite():
    """They are lost, and no other row."""
    for news in ([1, 1], [30, 20]):
        req = Requests4(news, [100, 90], 8, 2, 64, 16, BF16)
        q = req.q.to(BF16)
        clean = _attend(req, q)
        q[0, 3, 7], q[1, 5, 1] = math.nan, math.inf
        got = _attend(req, q)
        lost = torch.zeros(q.shape[:2], dtype=torch.bool, device="cuda")
        lost[0, 3] = lost[1, 5] = True
        assert not got[lost].isfinite().any() and torch.equal(got[~lost], clean[~lost])


@pytest.mark.gpu
def test_requests_share_pages_and_strided_rows():
    req = Requests4([1, 1, 50], [40, 33, 90], 8, 2, 128, 16, BF16, share=True)
    wide = torch.randn(52, 14, 128, device="cuda").to(BF16)
    _check(req, wide[:, 3:11])
    odd = torch.randn(52 * 8 * 128 + 3, device="cuda").to(BF16)[3:].view(52, 8, 128)  # copied to alignment
    _check(req, odd)
    # codes and scales inside wider tensors
    pages, page, Hk = req.codes[0].shape[:3]
    for i in range(2):
        codes = torch.zeros(pages, page, Hk + 1, 80, dtype=torch.uint8, device="cuda")
        scales = torch.zeros(pages, page + 2, Hk, 8, dtype=BF16, device="cuda")
        codes[:, :, 1:, 16:] = req.codes[i]
        scales[:, :page, :, 4:] = req.scales[i]
        req.codes[i], req.scales[i] = codes[:, :, 1:, 16:], scales[:, :page, :, 4:]
    _check(req, wide[:, :8])


@pytest.mark.gpu
@pytest.mark.parametrize("news", [[1, 1, 1], [40, 30, 50], [200, 30, 60]])
def test_pages_out_of_range_give_nan_and_the_error_word(news):
    req = Requests4(news, [max(100, news[0]), 60, 70], 8, 2, 64, 16, BF16)
    q = req.q.to(BF16)
    clean = _attend(req, q)
    _lib.device_error()
    for wrong in (-1, 10 ** 6):
        table = req.table.clone()
        table[1, 1] = wrong
        got = fap.paged_attention_int4(q, *req.cache, table, req.seq_lens, req.cu)
        assert _lib.device_error() == 2
        assert got[news[0] + news[1] - 1].isnan().all()
        assert torch.equal(got[:news[0]], clean[:news[0]]) and torch.equal(got[-news[2]:], clean[-news[2]:])
    lens = req.seq_lens.clone()
    lens[1] = 10 ** 6  # more tokens than its pages hold
    got = fap.paged_attention_int4(q, *req.cache, req.table, lens, req.cu)
    assert _lib.device_error() == 2
    assert got[news[0]:-news[2]].isnan().all()
    # other lengths move the borders at which the work is cut, and with them the order of sums: right, not equal
    exact, bound, _ = _bound(req, q, 1.0, 0)
    assert ((got[:news[0]].double() - exact[:news[0]]).abs() <= bound[:news[0]]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("news,totals,window", [
    ([700, 0, 900, 5], [900, 40, 2000, 1100], 0),   # whole tiles, more than the GPU holds at once
    ([70, 3, 25], [6000, 2500, 2900], 0),           # keys shared out
])
@pytest.mark.parametrize("D", [64, 128])
def test_waits_that_run_out(news, totals, window, D, monkeypatch):
    """Tiles given up come out as NaN with the error word set, shares of a tile included; the rest has its bits."""
    req = Requests4(news, totals, 32, 4, D, 16, BF16)
    other = Requests4(news, totals, 32, 4, D, 16, BF16, seed=1)

    def call(r):
        return _attend(r, r.q.to(BF16), softmax_scale=0.1, window=window, return_lse=True)

    def bounded(cycles):
        def run(name, args, device, scales):
            status = _lib.load().flash_prologue_selftest_attention_int4_waits(args, scales, cycles,
                                                                              _lib.raw_stream(device.index))
            _lib.check(status, "flash_prologue_selftest_attention_int4_waits")
        return run

    clean, clean_lse = call(req)
    _lib.device_error()
    given_up = 0
    for cycles in (1, 200, 600, 1000, 2000, 4000, 8000, 20000, 100000, 2 ** 32):
        call(other)  # leaves other rows and shares where this call's may come to lie
        torch.cuda.synchronize()
        with monkeypatch.context() as m:
            m.setattr(fap.int4, "call_library", bounded(cycles))
            got, lse = call(req)
        error = _lib.device_error()
        lost = got.isnan().all(-1)
        assert torch.equal(got.isnan().any(-1), lost) and torch.equal(lse.isnan(), lost)
        assert torch.equal(got[~lost], clean[~lost]) and torch.equal(lse[~lost], clean_lse[~lost])
        assert error == 1 if lost.any() else error in (0, 1)
        given_up += int(lost.sum())
    assert error == 0 and not lost.any()  # the limit of a call
    assert given_up
    assert all(torch.equal(a, b) for a, b in zip(call(req), (clean, clean_lse)))


@pytest.mark.gpu
@pytest.mark.parametrize("news,totals,ahead", [
    ([1, 0, 1, 3, 1, 1], [40, 9, 1, 250, 66, 130], 5),
    ([2, 1, 0, 1, 1, 1], [3000, 70, 4, 900, 64, 333], 7),
    ([60, 2], [90, 9], 5),
    ([70, 2], [1500, 2], 300),
])
@pytest.mark.parametrize("D,window", [(64, 0), (128, 50)])
def test_rows_outside_the_requests_are_zero(news, totals, ahead, D, window):
    req = Requests4(news, totals, 8, 2, D, 16, BF16)
    q = torch.cat((torch.ones(ahead, 8, D, device="cuda"), req.q, torch.ones(2, 8, D, device="cuda"))).to(BF16)
    torch.full((4, *q.shape), math.nan, dtype=BF16, device="cuda")  # what an unwritten output may come to lie in
    scale = D ** -0.5
    out, lse = fap.paged_attention_int4(q, *req.cache, req.table, req.seq_lens, req.cu + ahead, softmax_scale=scale,
                                        window=window, return_lse=True)
    for rows in (slice(0, ahead), slice(-2, None)):
        assert (out[rows] == 0).all() and (lse[rows] == -math.inf).all()
    exact, bound, exact_lse = _bound(req, q[ahead:-2], scale, window)
    assert ((out[ahead:-2].double() - exact).abs() <= bound).all()
    assert ((lse[ahead:-2].double() - exact_lse).abs() <= SCORE).all()


@pytest.mark.gpu
def test_wrong_splits_stay_inside_the_rows():
    req = Requests4([20, 20], [50, 50], 8, 2, 64, 16, BF16)
    q = req.q.to(BF16)
    for cu in ([0, 60, 100], [0, -5, 40], [30, 10, 40], [0, 0, 0]):
        out = fap.paged_attention_int4(q, *req.cache, req.table, req.seq_lens,
                                       torch.tensor(cu, dtype=torch.int32, device="cuda"))
        assert out.shape == q.shape
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_offsets_past_32_bits():
    pages, page, Hk, D = 300_000, 16, 8, 128  # 2.5 GB of codes a cache
    cache = [torch.empty(pages, page, Hk, D // 2, dtype=torch.uint8, device="cuda") for _ in range(2)]
    cache += [torch.empty(pages, page, Hk, D // 32, dtype=BF16, device="cuda") for _ in range(2)]
    table = torch.tensor([[pages - 1, 0, pages - 7], [pages - 3, 131072, 5]], dtype=torch.int32, device="cuda")
    for news in ([1, 1], [30, 37], [40, 48]):
        small = Requests4(news, [40, 48], 16, Hk, D, page, BF16)
        for r in range(2):
            for c in range(3):
                for big, little in zip(cache, small.cache):
                    big[table[r, c]] = little[small.table[r, c]]
        q = small.q.to(BF16)
        got = fap.paged_attention_int4(q, *cache, table, small.seq_lens, small.cu, softmax_scale=0.1)
        assert torch.equal(got, _attend(small, q, softmax_scale=0.1))


@pytest.mark.gpu
@pytest.mark.parametrize("news,totals", [([1] * 5, [4000, 3, 900, 77, 2000]), ([9, 400, 0, 3], [900, 2500, 5, 3])])
def test_repeats_bit_for_bit_and_on_another_stream(news, totals):
    req = Requests4(news, totals, 16, 4, 128, 16, BF16)
    q = req.q.to(BF16)
    first = _attend(req, q, return_lse=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = _attend(req, q, return_lse=True)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(first, again):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("news,totals", [([1, 1], [3000, 50]), ([40, 200], [2000, 400])])
def test_two_captured_graphs_follow_their_buffers(news, totals):
    reqs = [Requests4(news, totals, 16, 4, 64, 16, BF16, seed=s) for s in (0, 5)]
    qs = [r.q.to(BF16) for r in reqs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _attend(reqs[0], qs[0])
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for r, q in zip(reqs, qs):  # of one memory pool, as a server's graphs
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            outs.append(_attend(r, q))
        graphs.append(graph)
    for r in reqs:
        r.seq_lens -= 1
    for i in (0, 1, 0):
        graphs[i].replay()
        assert torch.equal(outs[i], _attend(reqs[i], qs[i]))


@pytest.mark.gpu
def test_opcheck_and_compiled():
    req = Requests4([2, 1], [10, 5], 8, 2, 64, 16, BF16)
    args = (req.q.to(BF16), *req.cache, req.table, req.seq_lens, req.cu)
    result = torch.library.opcheck(torch.ops.flash_prologue.paged_attention_int4.default, (*args, 0.5, 0, True),
                                   test_utils=("test_schema", "test_faketensor"))
    assert set(result.values()) == {"SUCCESS"}, result
    compiled = torch.compile(fap.paged_attention_int4, fullgraph=True)(*args, softmax_scale=0.5)
    assert torch.equal(compiled, fap.paged_attention_int4(*args, softmax_scale=0.5))


@pytest.mark.gpu
@pytest.mark.parametrize("D,dtype", [(128, BF16), (64, FP16)])
def test_serving_steps(D, dtype):
    """Plan, append and attend, step after step, against attention over all tokens' rows so far; in a captured graph too."""
    B, Hq, Hk, page, width, pool = 4, 8, 2, 16, 12, 40
    g = torch.Generator(device="cuda").manual_seed(2)
    cache = fap.int4_cache(pool, page, Hk, D)
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    free = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    lens, count = torch.zeros(B, dtype=torch.int32, device="cuda"), torch.tensor([pool], dtype=torch.int32, device="cuda")
    w, s = torch.ones(2, 1, D, device="cuda"), torch.full((Hq, 1, 1), math.log(D ** -0.5), device="cuda")
    sin, cos = tables(256, D)
    axes = fap.rotary_axes((D // 4, D // 8, D // 8), interleaved=True)
    kept = {r: [] for r in range(B)}  # rows of K and V as the cache holds them
    _lib.device_error()
    for news in ([50, 0, 17, 3], [1, 1, 1, 1], [1, 30, -1, 1], [-1, 1, 8, 1], [20, 1, 1, 1]):
        T = sum(max(n, 0) for n in news)
        new = torch.tensor(news, dtype=torch.int32, device="cuda")
        step = fap.plan_paged_step(table, lens, new, free, count, page, T + 2)  # two rows of padding
        lens, count = step.seq_lens, step.free_count
        q, k, v = (torch.randn(T + 2, h, D, generator=g, device="cuda").to(dtype) for h in (Hq, Hk, Hk))
        positions = torch.stack((step.positions, step.positions // 2, step.positions % 5))
        q = fap.append_paged_kv_int4(q, k, v, w, s, sin, cos, *cache, table, lens, step.cu_seqlens, positions=positions,
                                     axes=axes)
        out = fap.paged_attention_int4(q, *cache, table, lens, step.cu_seqlens)
        assert _lib.device_error() == 0
        assert not out[T:].any() and not q[T:].any()
        slots = step.slots[:T]
        rows = [fap.unpack_int4(cache[i].flatten(0, 1)[slots], cache[i + 2].flatten(0, 1)[slots], dtype).double()
                for i in range(2)]
        begin = 0
        for r, n in enumerate(news):
            if n < 0:
                kept[r] = []
                continue
            kept[r] += [(rows[0][i], rows[1][i]) for i in range(begin, begin + n)]
            assert len(kept[r]) == int(lens[r])
            for i in range(n):
                seen = kept[r][:len(kept[r]) - n + i + 1]
                keys, values = (torch.stack([x[j] for x in seen], 1).repeat_interleave(Hq // Hk, 0) for j in range(2))
                p = torch.einsum("hd,hjd->hj", q[begin + i].double(), keys).softmax(1)
                exact, size = (torch.einsum("hj,hjd->hd", p, x) for x in (values, values.abs()))
                u = HALF_ULP[dtype]
                # (LIFT: the largest value of a group is 8 s)
                bound = u * exact.abs() + (u + SCORE) * size + 2.0 ** -16 * size.amax(-1, keepdim=True) * 32 + 1e-30
                assert ((out[begin + i].double() - exact).abs() <= bound).all()
            begin += n


def _cpu(T=3, Hq=8, Hk=2, D=64, page=16):
    caches = fap.int4_cache(4, page, Hk, D, "cpu")
    return dict(q=torch.zeros(T, Hq, D, dtype=BF16), **dict(zip(("k_cache", "v_cache", "k_scale", "v_scale"), caches)),
                page_table=torch.zeros(3, 1, dtype=torch.int32), seq_lens=torch.ones(3, dtype=torch.int32))


@pytest.mark.parametrize("change,text", [
    (dict(q=torch.zeros(1, 3, 8, 64, dtype=BF16)), "must be packed"),
    (dict(q=torch.zeros(3, 8, 64)), "BF16 or FP16"),
    (dict(q=torch.zeros(3, 8, 32, dtype=BF16)), "head dimension"),
    (dict(q=torch.zeros(3, 7, 64, dtype=BF16)), "multiple of the key heads"),
    (dict(k_cache=torch.zeros(4, 16, 2, 64, dtype=torch.uint8)), "matching"),
    (dict(k_cache=torch.zeros(4, 16, 2, 32), v_cache=torch.zeros(4, 16, 2, 32)), "uint8"),
    (dict(k_scale=torch.zeros(4, 16, 2, 4, dtype=BF16)), "scales must be matching"),
    (dict(v_scale=torch.zeros(4, 16, 2, 2)), "scales must be bfloat16"),
    (dict(page_table=torch.zeros(3, 1, dtype=torch.int64)), "must be int32"),
    (dict(softmax_scale=math.inf), "softmax_scale"),
    (dict(softmax_scale=math.nan), "softmax_scale"),
    (dict(window=-1), "window"),
    (dict(q=torch.zeros(3, 8, 64, dtype=BF16, requires_grad=True)), "not differentiable"),
    (dict(), "CUDA devices only"),
])
def test_refusals(change, text):
    with pytest.raises(ValueError, match=text):
        fap.paged_attention_int4(**{**_cpu(), **change})


@pytest.mark.gpu
def test_refused_layouts():
    args = {n: t.cuda() for n, t in _cpu().items()}
    for name, bad in (("k_cache", torch.zeros(4 * 16 * 2 * 32 + 8, dtype=torch.uint8, device="cuda")[8:].view(4, 16, 2, 32)),
                      ("v_scale", torch.zeros(4 * 16 * 2 * 2 + 1, dtype=BF16, device="cuda")[1:].view(4, 16, 2, 2)),
                      ("k_scale", torch.zeros(4, 16, 2, 3, dtype=BF16, device="cuda")[..., :2])):
        with pytest.raises(ValueError, match="align"):
            fap.paged_attention_int4(**{**args, name: bad})


@pytest.mark.gpu
@pytest.mark.parametrize("D,dtype", [(64, FP16), (128, BF16)])
@pytest.mark.parametrize("Hq,Hk,news,totals", [
    (16, 2, [1, 1], [50001, 333]),
    (12, 6, [2, 1, 1], [9000, 65, 64]),
    (8, 1, [1], [30011]),
    (9, 3, [1, 1, 0, 1], [4097, 31, 9, 20000]),
    (5, 5, [1, 2], [70, 6001]),
])
@pytest.mark.parametrize("page,hnd,window", [(32, False, 0), (64, True, 0), (64, False, 1000), (128, True, 65)])
def test_few_key_heads(Hq, Hk, news, totals, page, hnd, window, D, dtype):
    req = Requests4(news, totals, Hq, Hk, D, page, dtype, hnd, seed=Hk)
    _check(req, req.q.to(dtype), window=window)


@pytest.mark.gpu
@pytest.mark.parametrize("Hk", [1, 2, 4])
def test_pages_of_whole_steps_out_of_range(Hk):
    req = Requests4([1, 1, 1], [700, 200, 900], 8, Hk, 128, 64, BF16)
    q = req.q.to(BF16)
    clean = _attend(req, q, decode=True)
    _lib.device_error()
    for wrong in (-1, 10 ** 6):
        table = req.table.clone()
        table[1, 1] = wrong
        got = fap.paged_attention_int4(q, *req.cache, table, req.seq_lens)
        assert _lib.device_error() == 2
        assert got[1].isnan().all() and torch.equal(got[::2], clean[::2])
