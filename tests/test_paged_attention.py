"""paged_attention against plain attention in 64 bits.

Bounds: one cast of the output (half an ulp of it) and one of each probability (half an ulp of
its share of the sum), plus FP32 scores: with |q| |k| sums up to 2^6 and D <= 128 products added
in FP32 a score is off by less than 2^-12, and so is each probability, relatively.
"""
import math

import pytest
import torch

import flash_attn_prologue_b200 as fap
from flash_attn_prologue_b200 import _lib
from tests._paged import HALF_ULP, Requests, tables

BF16, FP16 = torch.bfloat16, torch.float16
SCORE = 2.0 ** -12


def _exact(req, q, scale, window, rows=None):
    """(out, sum of p |v|, lse) of every new token in 64 bits; only keys a token sees are touched."""
    T, Hq, D = q.shape
    out = torch.zeros(T, Hq, D, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(out)
    lse = torch.full((T, Hq), -math.inf, dtype=torch.float64, device="cuda")
    begin = 0
    for r, (new, total) in enumerate(zip(req.news, req.totals)):
        k_all, v_all = (c[req.places(r, 0, total)].double() for c in (req.k, req.v))
        G = Hq // k_all.shape[1]
        k_all, v_all = (t.repeat_interleave(G, 1) for t in (k_all, v_all))
        for i in range(new):
            last = total - new + i + 1
            first = max(0, last - window) if window else 0
            if last <= 0 or (rows is not None and begin + i not in rows):
                continue
            k, v = k_all[first:last], v_all[first:last]
            s = torch.einsum("hd,jhd->hj", q[begin + i].double(), k) * scale
            lse[begin + i] = s.logsumexp(1)
            p = s.softmax(1)
            out[begin + i] = torch.einsum("hj,jhd->hd", p, v)
            size[begin + i] = torch.einsum("hj,jhd->hd", p, v.abs())
        begin += new
    return out, size, lse


def _check(req, q, scale=None, window=0, decode=False, rows=None):
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    out, lse = fap.paged_attention(q, req.k, req.v, req.table, req.seq_lens, None if decode else req.cu,
                                   softmax_scale=scale, window=window, return_lse=True)
    assert out.shape == q.shape and out.dtype == q.dtype and lse.shape == q.shape[:2]
    exact, size, exact_lse = _exact(req, q, scale, window, rows)
    pick = slice(None) if rows is None else rows
    u = HALF_ULP[q.dtype]
    bound = u * exact.abs() + (u + SCORE) * size + 1e-30
    off = ((out.double() - exact).abs() / bound)[pick]
    assert not off.numel() or float(off.max()) <= 1, float(off.max())
    far = torch.where(exact_lse.isinf(), (lse != exact_lse).double(), (lse.double() - exact_lse).abs())[pick]
    assert not far.numel() or float(far.max()) <= SCORE
    return out, lse


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hk", [(8, 2), (4, 4), (15, 5), (7, 1), (32, 1), (48, 2)])
@pytest.mark.parametrize("page,hnd,window", [(16, False, 0), (8, True, 50), (64, True, 0), (256, False, 17)])
def test_chunks(Hq, Hk, page, hnd, window, D, dtype):
    req = Requests([1, 0, 7, 33, 2, 20], [1, 12, 7, 300, 130, 70], Hq, Hk, D, page, dtype, hnd, seed=page)
    _check(req, req.q.to(dtype), window=window)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hk", [(8, 8), (32, 8), (16, 1), (40, 2)])
@pytest.mark.parametrize("page,window", [(8, 0), (32, 0), (16, 100), (128, 1)])
def test_single_tokens(Hq, Hk, page, window, D, dtype):
    totals = [1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 500, 1000]
    req = Requests([1] * len(totals), totals, Hq, Hk, D, page, dtype, page == 32, seed=page)
    _check(req, req.q.to(dtype), window=window, decode=True)


@pytest.mark.gpu
@pytest.mark.parametrize("news,totals", [
    ([1] * 9, [1, 64, 100, 128, 129, 192, 200, 255, 256]),
    ([2, 0, 1, 3], [200, 256, 1, 3]),
    ([1] * 400, [1 + i % 250 for i in range(400)]),
])
@pytest.mark.parametrize("Hq,Hk,D,window", [(8, 2, 128, 0), (16, 16, 64, 70), (48, 2, 64, 0)])
def test_short_caches(news, totals, Hq, Hk, D, window):
    """Caches that one CTA an item reads whole."""
    req = Requests(news, totals, Hq, Hk, D, 64, FP16)
    assert req.table.shape[1] * 64 <= 256
    _check(req, req.q.half(), window=window, rows=list(range(0, sum(news), 1 + sum(news) // 60)))


@pytest.mark.gpu
@pytest.mark.parametrize("news,totals", [
    ([1], [40000]),                      # split over the whole GPU
    ([1, 1], [70001, 3]),
    ([5], [20000]),
    ([300], [5000]),                     # many row tiles
    ([1000, 1, 0, 40], [1000, 9000, 5, 2040]),
    ([1] * 300, [1 + 7 * (i % 40) for i in range(300)]),  # more requests than threads
    ([i % 3 for i in range(290)], [3 + i for i in range(290)]),
])
@pytest.mark.parametrize("window", [0, 777])
def test_long_and_many(news, totals, window):
    req = Requests(news, totals, 16, 4, 128, 16, BF16)
    rows = None if sum(news) <= 350 else list(range(0, sum(news), 61))
    _check(req, req.q.to(BF16), window=window, rows=rows)


@pytest.mark.gpu
@pytest.mark.parametrize("news,totals", [
    ([1, 1, 1], [9000, 30, 20001]),
    ([3, 0, 5, 1], [20000, 7000, 12345, 5]),
    ([1] * 140, [300 + 7 * i for i in range(140)]),  # more requests than threads
    ([2, 1, 0, 3] * 35, [300 + 9 * i for i in range(140)]),
])
@pytest.mark.parametrize("Hq,Hk,D,window", [(8, 2, 64, 0), (3, 1, 128, 0), (4, 1, 64, 5000), (12, 4, 128, 300)])
def test_few_items_over_many_ctas(news, totals, Hq, Hk, D, window):
    """Key heads times row tiles are fewer than a full GPU's CTAs, or about as many."""
    req = Requests(news, totals, Hq, Hk, D, 32, BF16)
    _check(req, req.q.to(BF16), window=window)


@pytest.mark.gpu
@pytest.mark.parametrize("news,totals", [
    ([900, 0, 1300, 5], [900, 40, 2000, 1100]),   # more tiles than the GPU holds at once
    ([1] * 300 + [1500], [9] * 300 + [1500]),     # most of them of other requests than the last
    ([40, 3, 25, 1], [3000, 2500, 2900, 900]),    # few, of uneven requests: keys shared out
])
@pytest.mark.parametrize("Hq,Hk,D,dtype,window", [(32, 2, 64, FP16, 0), (32, 2, 128, BF16, 100), (12, 4, 128, FP16, 0)])
def test_many_and_few_tiles(news, totals, Hq, Hk, D, dtype, window):
    req = Requests(news, totals, Hq, Hk, D, 16, dtype)
    rows = None if sum(news) <= 350 else list(range(0, sum(news), 37)) + [sum(news) - 1]
    _check(req, req.q.to(dtype), window=window, rows=rows)


@pytest.mark.gpu
@pytest.mark.parametrize("news,totals", [([4, 3], [2, 5]), ([6, 2], [0, 2]), ([40], [10])])
def test_rows_without_keys_are_zero(news, totals):
    req = Requests(news, totals, 8, 2, 64, 8, BF16)
    out, lse = _check(req, req.q.to(BF16))
    empty = max(0, news[0] - totals[0])
    assert not out[:empty].any() and (lse[:empty] == -math.inf).all()


@pytest.mark.gpu
@pytest.mark.parametrize("chunk", [12, 200])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_unseen_keys_never_reach_a_row(value, chunk):
    """A non-finite K or V of a later token, or of one before the window, changes nothing."""
    req = Requests([chunk, 3], [chunk + 90, 30], 8, 2, 128, 16, FP16)
    q = req.q.half()
    window = 64

    def call():
        return fap.paged_attention(q, req.k, req.v, req.table, req.seq_lens, req.cu, softmax_scale=0.1, window=window)

    clean = call()
    for cache in (req.k, req.v):
        kept = cache.clone()
        for at in (chunk + 90 - 4, 5, 90 + chunk // 2):
            where = req.places(0, at, at + 1)
            cache[where] = value
        got = call()
        position = torch.arange(90, 90 + chunk, device="cuda")
        sees = torch.zeros(chunk, dtype=torch.bool, device="cuda")
        for at in (chunk + 90 - 4, 5, 90 + chunk // 2):
            sees |= (position >= at) & (position - window < at)
        hidden = torch.cat((~sees, torch.ones(3, dtype=torch.bool, device="cuda")))
        assert hidden.any() and sees.any()
        assert torch.equal(got[hidden], clean[hidden])
        if cache is req.v:
            assert not got[:chunk][sees].isfinite().any()
            if math.isinf(value):  # two infinities of one sign, or one, and no key of weight 0
                assert (got[:chunk][sees] == value).all()
        cache.copy_(kept)


@pytest.mark.gpu
def test_large_scores_pick_one_key_and_scales():
    req = Requests([3, 40], [200, 400], 8, 2, 64, 16, BF16)
    q = req.q.to(BF16)
    # the largest score's lead makes it the only term; scores up to 2^13 are exact to 2^-11 of one
    out = fap.paged_attention(q, req.k, req.v, req.table, req.seq_lens, req.cu, softmax_scale=100.0)
    exact, size, _ = _exact(req, q, 100.0, 0)
    assert ((out.double() - exact).abs() <= 2.0 ** -8 * exact.abs() + 2.0 ** -5 * size.amax(-1, keepdim=True)).all()
    _check(req, q, scale=0.0)
    _check(req, q, scale=-0.2)


@pytest.mark.gpu
@pytest.mark.parametrize("news", [[3, 1], [40, 3]])
@pytest.mark.parametrize("scale", [1e-50, 1e-44, 1e-39, 1e-37, -1e-50])
def test_scales_that_vanish_in_fp32(scale, news):
    """Equal weights, whether the scale rounds to 0, to a subnormal number or to a very small one."""
    req = Requests(news, [45, 400], 8, 2, 64, 16, BF16)
    _check(req, req.q.to(BF16), scale=scale)


@pytest.mark.gpu
def test_requests_share_pages_and_strided_rows():
    req = Requests([1, 1, 50], [40, 33, 90], 8, 2, 128, 16, BF16, share=True)
    wide = torch.randn(52, 14, 128, device="cuda").to(BF16)
    _check(req, wide[:, 3:11])
    odd = torch.randn(52 * 8 * 128 + 3, device="cuda").to(BF16)[3:].view(52, 8, 128)  # copied to alignment
    _check(req, odd)
    _check(req, torch.randn(52, 128, 8, device="cuda").to(BF16).transpose(1, 2))


@pytest.mark.gpu
@pytest.mark.parametrize("news", [[1, 1, 1], [40, 30, 50]])
def test_pages_out_of_range_give_nan_and_the_error_word(news):
    req = Requests(news, [100, 60, 70], 8, 2, 64, 16, BF16)
    q = req.q.to(BF16)
    clean = fap.paged_attention(q, req.k, req.v, req.table, req.seq_lens, req.cu)
    _lib.device_error()
    for wrong in (-1, 10 ** 6):
        table = req.table.clone()
        table[1, 1] = wrong
        got = fap.paged_attention(q, req.k, req.v, table, req.seq_lens, req.cu)
        assert _lib.device_error() == 2
        assert got[news[0] + news[1] - 1].isnan().all()
        assert torch.equal(got[:news[0]], clean[:news[0]]) and torch.equal(got[-news[2]:], clean[-news[2]:])
    lens = req.seq_lens.clone()
    lens[1] = 10 ** 6  # more tokens than its pages hold
    got = fap.paged_attention(q, req.k, req.v, req.table, lens, req.cu)
    assert _lib.device_error() == 2
    assert got[news[0]:-news[2]].isnan().all() and torch.equal(got[:news[0]], clean[:news[0]])


@pytest.mark.gpu
@pytest.mark.parametrize("news,totals,window", [
    ([700, 0, 900, 5], [900, 40, 2000, 1100], 0),   # whole tiles, more than the GPU holds at once
    ([1500, 40], [1500, 4000], 300),
    ([70, 3, 25], [6000, 2500, 2900], 0),           # keys shared out
])
@pytest.mark.parametrize("D", [64, 128])
def test_waits_that_run_out(news, totals, window, D, monkeypatch):
    """Tiles given up come out as NaN with the error word set, shares of a tile included; the rest has its bits."""
    req = Requests(news, totals, 32, 4, D, 16, BF16)
    other = Requests(news, totals, 32, 4, D, 16, BF16, seed=1)

    def call(r):
        return fap.paged_attention(r.q.to(BF16), r.k, r.v, r.table, r.seq_lens, r.cu, softmax_scale=0.1, window=window,
                                   return_lse=True)

    def bounded(cycles):
        def run(name, args, device):
            status = _lib.load().flash_prologue_selftest_attention_waits(args, cycles, _lib.raw_stream(device.index))
            _lib.check(status, "flash_prologue_selftest_attention_waits")
        return run

    clean, clean_lse = call(req)
    _lib.device_error()
    given_up = 0
    for cycles in (1, 200, 600, 1000, 2000, 4000, 8000, 20000, 100000, 2 ** 32):
        call(other)  # leaves other rows and shares where this call's may come to lie
        torch.cuda.synchronize()
        with monkeypatch.context() as m:
            m.setattr(fap.paged, "call_library", bounded(cycles))
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
@pytest.mark.parametrize("chunk", [1, 60])
def test_padding_rows_are_zero(chunk):
    req = Requests([chunk, 2], [chunk + 30, 9], 8, 2, 64, 16, BF16)
    q = torch.cat((req.q, torch.ones(5, 8, 64, device="cuda"))).to(BF16)
    out, lse = fap.paged_attention(q, req.k, req.v, req.table, req.seq_lens, req.cu, return_lse=True)
    assert not out[-5:].any() and (lse[-5:] == -math.inf).all() and out[:-5].any(-1).all()
    assert torch.equal(out[:-5], fap.paged_attention(q[:-5], req.k, req.v, req.table, req.seq_lens, req.cu))


@pytest.mark.gpu
@pytest.mark.parametrize("news,totals,ahead", [
    ([1, 0, 1, 3, 1, 1], [40, 9, 1, 250, 66, 130], 5),      # single-token kernel, short caches
    ([2, 1, 0, 1, 1, 1], [3000, 70, 4, 900, 64, 333], 7),   # split over CTAs
    ([60, 2], [90, 9], 5),                                  # 128-row tiles
    ([70, 2], [1500, 2], 300),                              # keys shared out
])
@pytest.mark.parametrize("D,window", [(64, 0), (128, 50)])
def test_rows_before_the_first_request_are_zero(news, totals, ahead, D, window):
    """cu_seqlens that begin behind 0, as append_paged_kv takes them."""
    req = Requests(news, totals, 8, 2, D, 16, BF16)
    q = torch.cat((torch.ones(ahead, 8, D, device="cuda"), req.q, torch.ones(2, 8, D, device="cuda"))).to(BF16)
    torch.full((4, *q.shape), math.nan, dtype=BF16, device="cuda")  # what an unwritten output may come to lie in
    scale = D ** -0.5
    out, lse = fap.paged_attention(q, req.k, req.v, req.table, req.seq_lens, req.cu + ahead, softmax_scale=scale,
                                   window=window, return_lse=True)
    for rows in (slice(0, ahead), slice(-2, None)):
        assert (out[rows] == 0).all() and (lse[rows] == -math.inf).all()
    exact, size, exact_lse = _exact(req, q[ahead:-2], scale, window)
    u = HALF_ULP[BF16]
    assert ((out[ahead:-2].double() - exact).abs() <= u * exact.abs() + (u + SCORE) * size + 1e-30).all()
    assert ((lse[ahead:-2].double() - exact_lse).abs() <= SCORE).all()


@pytest.mark.gpu
def test_wrong_splits_stay_inside_the_rows():
    """cu_seqlens that run backwards or past the rows are cut to them; nothing faults."""
    req = Requests([20, 20], [50, 50], 8, 2, 64, 16, BF16)
    q = req.q.to(BF16)
    for cu in ([0, 60, 100], [0, -5, 40], [30, 10, 40], [0, 0, 0]):
        out = fap.paged_attention(q, req.k, req.v, req.table, req.seq_lens,
                                  torch.tensor(cu, dtype=torch.int32, device="cuda"))
        assert out.shape == q.shape
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_offsets_past_32_bits():
    pages, page, Hk, D = 140_000, 16, 8, 128  # 2.3 G elements a cache
    k, v = (torch.empty(pages, page, Hk, D, dtype=BF16, device="cuda") for _ in range(2))
    table = torch.tensor([[pages - 1, 0, pages - 7], [pages - 3, 131072, 5]], dtype=torch.int32, device="cuda")
    for p in table.flatten().tolist():
        k[p], v[p] = torch.randn(2, page, Hk, D, device="cuda").to(BF16)
    for news in ([1, 1], [30, 37]):
        small = Requests(news, [48, 40], 16, Hk, D, page, BF16)
        q = small.q.to(BF16)
        far = fap.paged_attention(q, k, v, table, small.seq_lens, small.cu)
        near_table = torch.arange(6, dtype=torch.int32, device="cuda").view(2, 3)
        near = fap.paged_attention(q, k[table.flatten().long()], v[table.flatten().long()], near_table,
                                   small.seq_lens, small.cu)
        assert torch.equal(far, near)


@pytest.mark.gpu
@pytest.mark.parametrize("news", [[1, 1], [70, 3]])
def test_repeats_bit_for_bit_on_streams_and_in_graphs(news):
    req = Requests(news, [3000, 800], 16, 2, 128, 16, BF16)
    q = req.q.to(BF16)
    call = lambda: fap.paged_attention(q, req.k, req.v, req.table, req.seq_lens, req.cu)  # noqa: E731
    first = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(call(), first)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for _ in range(3):
        graph.replay()
        assert torch.equal(out, first)
    req.seq_lens -= 100
    graph.replay()
    assert torch.equal(out, call()) and not torch.equal(out, first)


@pytest.mark.gpu
def test_append_then_attend_is_causal_attention():
    """A prompt in chunks and then token by token gives the rows of the whole prompt at once."""
    T, Hq, Hk, D, page = 150, 8, 2, 64, 16
    g = torch.Generator(device="cuda").manual_seed(3)
    qkv = torch.randn(T, Hq + 2 * Hk, D, generator=g, device="cuda").to(BF16)
    w = 1 + 0.1 * torch.randn(2, 1, D, generator=g, device="cuda")
    s = torch.full((Hq, 1, 1), math.log(D ** -0.5), device="cuda")
    sin, cos = tables(T, D)

    def serve(splits):
        k, v = (torch.full((12, page, Hk, D), math.nan, dtype=BF16, device="cuda") for _ in range(2))
        table = torch.randperm(12, generator=g, device="cuda")[None, :10].to(torch.int32).contiguous()
        out, done = [], 0
        for n in splits:
            rows = qkv[done:done + n]
            done += n
            lens = torch.tensor([done], dtype=torch.int32, device="cuda")
            cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
            q = fap.append_paged_kv(rows[:, :Hq], rows[:, Hq:Hq + Hk], rows[:, Hq + Hk:], w, s, sin, cos, k, v, table,
                                    lens, cu)
            out.append(fap.paged_attention(q, k, v, table, lens, cu))
        return torch.cat(out).float()

    whole = serve([T])
    for splits in ([100, 50], [1] * T, [3, 64, 80, 3]):
        # both are within one cast of the output and one of the probabilities (|v| <= 5 here)
        assert (serve(splits) - whole).abs().max() <= 2 * 2 * 2.0 ** -8 * 5


@pytest.mark.gpu
def test_opcheck_and_compiled():
    req = Requests([2, 1], [10, 5], 8, 2, 64, 16, BF16)
    args = (req.q.to(BF16), req.k, req.v, req.table, req.seq_lens, req.cu)
    result = torch.library.opcheck(torch.ops.flash_prologue.paged_attention.default, (*args, 0.5, 0, True),
                                   test_utils=("test_schema", "test_faketensor"))
    assert set(result.values()) == {"SUCCESS"}, result
    assert torch.equal(torch.compile(fap.paged_attention, fullgraph=True)(*args), fap.paged_attention(*args))


@pytest.mark.gpu
def test_no_tokens():
    req = Requests([0, 0], [5, 0], 8, 2, 64, 16, BF16)
    out, lse = fap.paged_attention(req.q.to(BF16), req.k, req.v, req.table, req.seq_lens, req.cu, return_lse=True)
    assert out.shape == (0, 8, 64) and lse.shape == (0, 8)


def _cpu_call(**change):
    args = dict(q=torch.zeros(3, 8, 64, dtype=BF16), k_cache=torch.zeros(4, 16, 2, 64, dtype=BF16),
                v_cache=torch.zeros(4, 16, 2, 64, dtype=BF16), page_table=torch.zeros(3, 1, dtype=torch.int32),
                seq_lens=torch.ones(3, dtype=torch.int32))
    return fap.paged_attention(**{**args, **change})


@pytest.mark.parametrize("change,text", [
    (dict(q=torch.zeros(8, 64, dtype=BF16)), "packed"),
    (dict(q=torch.zeros(3, 8, 64)), "BF16 or FP16"),
    (dict(q=torch.zeros(3, 8, 32, dtype=BF16)), "head dimension"),
    (dict(q=torch.zeros(3, 7, 64, dtype=BF16)), "multiple of the key heads"),
    (dict(q=torch.zeros(3, 1024, 64, dtype=BF16)), "at most 512"),
    (dict(q=torch.zeros(3, 8, 64, dtype=torch.float16)), "share a dtype"),
    (dict(q=torch.zeros(4, 8, 64, dtype=BF16)), "one token"),
    (dict(k_cache=torch.zeros(4, 16, 2, 32, dtype=BF16)), "matching"),
    (dict(k_cache=torch.zeros(4, 24, 2, 64, dtype=BF16), v_cache=torch.zeros(4, 24, 2, 64, dtype=BF16)), "power of two"),
    (dict(seq_lens=torch.ones(3, dtype=torch.int64)), "int32"),
    (dict(cu_seqlens=torch.zeros(3, dtype=torch.int32)), "cu_seqlens must be"),
    (dict(softmax_scale=math.nan), "softmax_scale"),
    (dict(window=-1), "window"),
    (dict(q=torch.zeros(3, 8, 64, dtype=BF16, requires_grad=True)), "not differentiable"),
    (dict(), "CUDA devices only"),
])
def test_refusals(change, text):
    with pytest.raises(ValueError, match=text):
        _cpu_call(**change)


def test_c_abi_refusals():
    """Arguments that the library turns away before it touches the device."""
    lib = _lib.load()

    def call(ptr=64, n=512, T=3, Hq=8, Hk=2, D=64, dtype=0, window=0, scale=1.0, page=16, slot=128, batch=3, cu=0, k=64):
        cache = (k, 2048, slot, 64, 64, 2048, 128, 64, 4, page, 64, 1, 1, 64, cu, batch)
        return lib.flash_prologue_paged_attention(_lib.ATTENTION_ARGS.pack(
            ptr, 0, 64, n, ptr, 0, 64, n, 0, *cache, 0, 0, T, Hq, Hk, D, dtype, window, scale), None)

    assert call(T=0, batch=0, ptr=0) == _lib.OK
    for wrong, status in ((dict(dtype=2), 2), (dict(D=32), 2), (dict(Hk=3), 1), (dict(Hk=0), 1), (dict(Hq=1024), 2),
                          (dict(window=-1), 1), (dict(scale=math.inf), 1), (dict(page=24), 1), (dict(page=4), 1),
                          (dict(slot=129), _lib.ERR_ALIGNMENT), (dict(k=72), _lib.ERR_ALIGNMENT), (dict(k=0), 1),
                          (dict(batch=2), 1), (dict(ptr=0), 1), (dict(ptr=68), _lib.ERR_ALIGNMENT),
                          (dict(n=513), _lib.ERR_ALIGNMENT), (dict(T=-1), 1), (dict(batch=-1, cu=64), 1)):
        assert call(**wrong) == status, wrong


@pytest.mark.parametrize("scale", [3e38, -1e300, math.nan, math.inf])
def test_scales_that_fp32_cannot_hold_are_refused(scale):
    with pytest.raises(ValueError, match="softmax_scale"):
        _cpu_call(softmax_scale=scale)
    cache = (64, 2048, 128, 64, 64, 2048, 128, 64, 4, 16, 64, 1, 1, 64, 0, 3)
    args = _lib.ATTENTION_ARGS.pack(64, 0, 64, 512, 64, 0, 64, 512, 0, *cache, 0, 0, 3, 8, 2, 64, 0, 0, scale)
    assert _lib.load().flash_prologue_paged_attention(args, None) == 1


@pytest.mark.parametrize("cycles", [0, -1, 10 ** 10])
def test_wait_limits_that_are_refused(cycles):
    assert _lib.load().flash_prologue_selftest_attention_waits(bytes(_lib.ATTENTION_ARGS.size), cycles, None) == 1
