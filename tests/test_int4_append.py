"""append_paged_kv_int4 and unpack_int4 against the 4-bit format's definition in 64 bits."""
import pytest
import torch

import flash_attn_prologue_b200 as fap
from flash_attn_prologue_b200 import _lib
from tests._int4 import Requests4, codes_of, cut, encode64, groups, pack, values64
from tests._paged import BAND, assert_within, rotate64, tables

BF16, FP16 = torch.bfloat16, torch.float16


def _inputs(req, Hq, Hk, D, dtype, norm=True, odd=False, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    T = sum(req.news)

    def rand(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if odd:
        q, k, v = (rand(T * h * D + 1).to(dtype)[1:].view(T, h, D) for h in (Hq, Hk, Hk))
    else:
        buf = rand(T, Hq + 2 * Hk, D).to(dtype)
        q, k, v = buf[:, :Hq], buf[:, Hq:Hq + Hk], buf[:, Hq + Hk:]
    w = 1 + 0.2 * rand(2, 1, D) if norm else None
    s = 0.3 * rand(Hq, 1, 1) if norm else None
    return q, k, v, w, s, *tables(max([1] + req.totals), D)


def _check_codes(packed, scale, rows, size, half, name):
    """Codes and scales of FP32 rows that are within BAND * size of ``rows``."""
    D = rows.shape[-1]
    off, s = BAND * size, scale.double()
    # a scale is another than the exact row's only where the extreme is that near a border (the two agree elsewhere)
    near, sums = torch.zeros_like(s), torch.zeros_like(s)
    for g in range(D // 32):
        mine = groups(D, rows.device) == g
        near[..., g] = off[..., mine].amax(-1)
        sums[..., g] = rows[..., mine].amax(-1) + rows[..., mine].amin(-1)
    low, high = (_moved_scale(rows, near, sign, half) for sign in (-1, 1))
    assert ((s.abs() >= low - 1e-300) & (s.abs() <= high)).all(), name
    assert ((s * sums <= 0) | (sums.abs() <= 2 * near)).all(), name  # the largest magnitude has code -8
    # a code is the nearest one, but where x / s is that near a half
    s = s[..., groups(D, rows.device)]
    x = rows / torch.where(s == 0, 1, s)
    far = (codes_of(packed).double() - torch.clamp(torch.round(x), -8, 7)).abs()
    border = ((x - torch.floor(x)) - 0.5).abs() * s.abs() <= 2 * off
    assert ((far == 0) | (border & (far == 1))).all(), name


def _moved_scale(rows, near, sign, half):
    """Least and largest magnitudes of the scale when the extreme moves by ``near``."""
    D = rows.shape[-1]
    out = []
    for g in range(D // 32):
        part = rows[..., groups(D, rows.device) == g].abs().amax(-1)
        out.append(cut((part + sign * near[..., g]).clamp(min=0), half).abs())
    return torch.stack(out, -1)


def _check(req, args, decode=False, **turn):
    q, k, v, w, s, sin, cos = args
    half = q.dtype is FP16
    before = [t.clone() for t in req.cache]
    _lib.device_error()
    got = fap.append_paged_kv_int4(*args, *req.cache, req.table, req.seq_lens, None if decode else req.cu, **turn)
    assert _lib.device_error() == 0
    assert got.shape == q.shape and got.is_contiguous()
    at = torch.cat([torch.arange(t - n, t, device="cuda") for n, t in zip(req.news, req.totals)])
    sn, cs = sin[at][:, None], cos[at][:, None]
    gain = 1.0 if s is None else s.double().exp().view(-1, 1)
    assert_within(got, *rotate64(q, None if w is None else w[0], sn, cs, gain), "q")
    k_rows, k_size = rotate64(k, None if w is None else w[1], sn, cs, 1.0)
    begin = 0
    for r, (n, t) in enumerate(zip(req.news, req.totals)):
        where = req.places(r, t - n, t)
        _check_codes(req.codes[0][where], req.scales[0][where], k_rows[begin:begin + n], k_size[begin:begin + n], half, "k")
        codes, scales = encode64(v[begin:begin + n], half)  # V is exact: so are its codes
        assert torch.equal(codes_of(req.codes[1][where]).double(), codes)
        assert torch.equal(req.scales[1][where].double(), scales)
        for was, now in zip(before, req.cache):
            was[where] = now[where]
        begin += n
    for was, now in zip(before, req.cache):  # nothing else of the cache has changed
        assert torch.equal(was.view(torch.uint8) if was.dtype == torch.uint8 else was.nan_to_num(77.0),
                           now.view(torch.uint8) if now.dtype == torch.uint8 else now.nan_to_num(77.0))
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq,Hk,page,hnd,norm,odd", [
    (8, 2, 16, False, True, False), (15, 5, 8, True, True, False), (4, 4, 64, False, False, False),
    (6, 1, 128, True, True, True),
])
def test_chunks(Hq, Hk, page, hnd, norm, odd, D, dtype):
    req = Requests4([3, 0, 40, 1, 17], [3, 9, 140, 1, 64], Hq, Hk, D, page, dtype, hnd)
    _check(req, _inputs(req, Hq, Hk, D, dtype, norm, odd))


@pytest.mark.gpu
@pytest.mark.parametrize("totals", [[1], [8, 9, 7, 1], list(range(1, 200, 2))])
def test_single_tokens(totals):
    req = Requests4([1] * len(totals), totals, 32, 8, 128, 8, BF16)
    _check(req, _inputs(req, 32, 8, 128, BF16), decode=True)


@pytest.mark.gpu
def test_long_chunk_and_empty_step():
    req = Requests4([1500, 0, 711], [1500, 30, 2000], 32, 8, 128, 64, BF16)
    _check(req, _inputs(req, 32, 8, 128, BF16))
    req = Requests4([0, 0], [5, 0], 8, 2, 64, 16, BF16)
    _check(req, _inputs(req, 8, 2, 64, BF16))


@pytest.mark.gpu
def test_same_queries_as_the_16_bit_cache():
    req = Requests4([50], [50], 8, 2, 64, 16, BF16)
    args = _inputs(req, 8, 2, 64, BF16)
    got = fap.append_paged_kv_int4(*args, *req.cache, req.table, req.seq_lens, req.cu)
    caches = [torch.zeros(req.codes[0].shape[:3] + (64,), dtype=BF16, device="cuda") for _ in range(2)]
    assert torch.equal(got, fap.append_paged_kv(*args, *caches, req.table, req.seq_lens, req.cu))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("D", [64, 128])
def test_values_at_the_edges(D, dtype):
    """Rows of V: zeros, ties, equal extremes of both signs, the type's largest and smallest, infinities and NaN."""
    info, T = torch.finfo(dtype), 12
    req = Requests4([T], [T], 4, 1, D, 16, dtype)
    q, k, v, w, s, sin, cos = _inputs(req, 4, 1, D, dtype)
    v = v.clone()
    v[0] = 0
    v[1] = torch.arange(D, device="cuda").view(1, D) % 33 - 16  # steps of a half: ties
    v[1, 0, groups(D) >= 0] *= 0.5
    v[2, 0, ::2], v[2, 0, 1::2] = 3.0, -3.0
    v[3, 0, ::2], v[3, 0, 1::2] = -5.0, 4.75
    v[4] = info.max
    v[5] = -info.max
    v[6] = info.tiny * torch.randn(1, D, device="cuda")
    v[7, 0, 3] = float("inf")
    v[8, 0, 9] = float("nan")
    v[9, 0, 17] = -float("inf")
    v[10] = 1e-6 * torch.randn(1, D, device="cuda")
    fap.append_paged_kv_int4(q, k, v, w, s, sin, cos, *req.cache, req.table, req.seq_lens, req.cu)
    where = req.places(0, 0, T)
    codes, scales = encode64(v, dtype is FP16)
    got_s = req.scales[1][where]
    assert torch.equal(got_s.isnan(), scales.isnan())
    assert torch.equal(got_s.double().nan_to_num(0.0), scales.nan_to_num(0.0))
    assert torch.equal(codes_of(req.codes[1][where]).double(), codes)
    out = fap.unpack_int4(req.codes[1][where], got_s, dtype)
    exact = codes * scales[..., groups(D)]
    assert torch.equal(out.isnan(), exact.isnan())
    assert torch.equal(out.double().nan_to_num(0.0), exact.nan_to_num(0.0))  # exact in the rows' type


@pytest.mark.gpu
def test_large_and_lost_keys():
    """Keys beyond FP16 stand for the largest values, keys of infinities for NaN."""
    req = Requests4([3], [3], 2, 1, 64, 8, FP16)
    q, k, v, _, _, sin, cos = _inputs(req, 2, 1, 64, FP16, norm=False)
    k = k.clone()
    k[0] = 60000.0
    k[1, 0, 5] = float("inf")
    w = torch.full((2, 1, 64), 4.0, device="cuda")
    fap.append_paged_kv_int4(q, k, v, None, None, sin, cos, *req.cache, req.table, req.seq_lens, req.cu)
    where = req.places(0, 0, 3)
    out = fap.unpack_int4(req.codes[0][where], req.scales[0][where], FP16)
    assert out[0].isfinite().all() and out[2].isfinite().all()
    lost = groups(64) == 5 // 8 % 2
    assert out[1, 0, lost].isnan().all() and out[1, 0, ~lost].isfinite().all()
    fap.append_paged_kv_int4(q, k, v, w, None, sin, cos, *req.cache, req.table, req.seq_lens, req.cu)
    # 1 / sqrt(infinity) is 0: the infinity times 0 is NaN, all other channels are zeros
    out = fap.unpack_int4(req.codes[0][where], req.scales[0][where], FP16)
    assert out[1, 0, lost].isnan().all() and not out[1, 0, ~lost].any()


@pytest.mark.gpu
def test_indices_out_of_range_and_padding_write_nothing():
    for change, lost in ((lambda r: r.table[0].fill_(-1), {0, 1, 2, 3}), (lambda r: r.table[2].fill_(10 ** 6), {7}),
                         (lambda r: r.seq_lens.copy_(torch.tensor([20, 1, 9])), {4, 5}), (lambda r: None, set())):
        req = Requests4([4, 3, 1], [20, 3, 9], 8, 2, 64, 8, BF16)
        args = _inputs(req, 8, 2, 64, BF16)
        args = tuple(torch.cat((t, t[:2])) for t in args[:3]) + args[3:]  # two rows of padding
        change(req)
        before = [t.clone() for t in req.cache]
        _lib.device_error()
        got = fap.append_paged_kv_int4(*args, *req.cache, req.table, req.seq_lens, req.cu)
        assert (_lib.device_error() == 2) == bool(lost)
        assert (got == 0).flatten(1).all(1).tolist() == [i in lost or i >= 8 for i in range(10)]
        for was, now in zip(before, req.cache):
            changed = (was.float().nan_to_num(7e7) != now.float().nan_to_num(7e7)).flatten(2).any(2)
            assert int(changed.sum()) <= 8 - len(lost)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_positions_of_several_axes(dtype):
    D, req = 128, Requests4([3, 20], [3, 30], 8, 2, 128, 16, dtype)
    args = _inputs(req, 8, 2, D, dtype)
    pos = torch.randint(0, 30, (3, 23), device="cuda")
    axes = fap.rotary_axes((16, 24, 24), interleaved=True)
    got = fap.append_paged_kv_int4(*args, *req.cache, req.table, req.seq_lens, req.cu, positions=pos, axes=axes)
    plain = [torch.zeros(req.codes[0].shape[:3] + (D,), dtype=dtype, device="cuda") for _ in range(2)]
    assert torch.equal(got, fap.append_paged_kv(*args, *plain, req.table, req.seq_lens, req.cu, positions=pos, axes=axes))
    for r, (n, t) in enumerate(zip(req.news, req.totals)):
        where = req.places(r, t - n, t)
        near = values64(req.codes[0][where], req.scales[0][where]) - plain[0][where].double()
        step = req.scales[0][where].double()[..., groups(D)].abs()
        # half a step, a step and a half where the code is cut to 7; the 16-bit cache's own rounding
        assert (near.abs() <= 1.51 * step + 2.0 ** -8 * plain[0][where].double().abs()).all()


@pytest.mark.gpu
def test_captured_step_and_registered_operator():
    req = Requests4([2, 1], [10, 5], 8, 2, 64, 16, BF16)
    args = _inputs(req, 8, 2, 64, BF16)
    call = lambda: fap.append_paged_kv_int4(*args, *req.cache, req.table, req.seq_lens, req.cu)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    req.seq_lens -= 1
    graph.replay()
    replayed = out.clone(), req.codes[0].clone()
    assert torch.equal(call(), replayed[0]) and torch.equal(req.codes[0], replayed[1])
    flat = (*args, *(t.nan_to_num(0.0) if t.dtype == BF16 else t for t in req.cache), req.table, req.seq_lens, req.cu)
    result = torch.library.opcheck(torch.ops.flash_prologue.append_paged_kv_int4.default, (*flat, 1e-5),
                                   test_utils=("test_schema", "test_faketensor"))
    assert set(result.values()) == {"SUCCESS"}, result
    eager = fap.append_paged_kv_int4(*flat)
    assert torch.equal(torch.compile(fap.append_paged_kv_int4, fullgraph=True)(*flat), eager)
    version = req.codes[1]._version, req.scales[0]._version
    call()
    assert (req.codes[1]._version, req.scales[0]._version) > version


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("lead", [(), (1,), (3, 7, 5), (2000, 3)])
def test_unpack(lead, dtype, D):
    g = torch.Generator(device="cuda").manual_seed(0)
    codes, scales = encode64(torch.randn(*lead, D, generator=g, device="cuda"), dtype is FP16)
    packed, scales = pack(codes), scales.to(BF16)
    out = fap.unpack_int4(packed, scales, dtype)
    assert out.dtype is dtype and torch.equal(out.double(), values64(packed, scales))
    if len(lead) > 1:  # views that are not contiguous
        out = fap.unpack_int4(packed[1:, ::2], scales[1:, ::2], dtype)
        assert torch.equal(out.double(), values64(packed, scales)[1:, ::2])


@pytest.mark.gpu
def test_an_empty_cache_stands_for_zeros():
    cache = fap.int4_cache(3, 16, 2, 128)
    assert [t.shape for t in cache] == [(3, 16, 2, 64)] * 2 + [(3, 16, 2, 4)] * 2
    assert not fap.unpack_int4(cache[0], cache[2]).any()
    assert torch.equal(torch.compile(fap.unpack_int4, fullgraph=True)(cache[0], cache[2]),
                       fap.unpack_int4(cache[0], cache[2]))
    with pytest.raises(ValueError, match="head dimension"):
        fap.int4_cache(3, 16, 2, 32)


def _cpu_step(T=3, Hq=8, Hk=2, D=64, page=16, dtype=BF16):
    sin, cos = tables(8, D, "cpu")
    caches = fap.int4_cache(4, page, Hk, D, "cpu")
    return dict(q=torch.zeros(T, Hq, D, dtype=dtype), k=torch.zeros(T, Hk, D, dtype=dtype),
                v=torch.zeros(T, Hk, D, dtype=dtype), rmsnorm_weight=torch.ones(2, 1, D), scales=torch.zeros(Hq, 1, 1),
                sin=sin, cos=cos, **dict(zip(("k_cache", "v_cache", "k_scale", "v_scale"), caches)),
                page_table=torch.zeros(3, 1, dtype=torch.int32), seq_lens=torch.ones(3, dtype=torch.int32))


@pytest.mark.parametrize("change,text", [
    (dict(q=torch.zeros(1, 3, 8, 64, dtype=BF16)), "must be packed"),
    (dict(q=torch.zeros(3, 8, 64)), "BF16 or FP16"),
    (dict(q=torch.zeros(3, 8, 32, dtype=BF16)), "head dimension"),
    (dict(v=torch.zeros(3, 4, 64, dtype=BF16)), "must be packed"),
    (dict(q=torch.zeros(3, 8, 64, dtype=BF16, requires_grad=True)), "not differentiable"),
    (dict(), "CUDA devices only"),
])
def test_refusals(change, text):
    with pytest.raises(ValueError, match=text):
        fap.append_paged_kv_int4(**{**_cpu_step(), **change})


@pytest.mark.gpu
@pytest.mark.parametrize("change,text", [
    (dict(k_cache=torch.zeros(4, 16, 2, 64, dtype=torch.uint8)), "matching"),
    (dict(k_cache=torch.zeros(4, 16, 2, 32, dtype=BF16), v_cache=torch.zeros(4, 16, 2, 32, dtype=BF16)), "uint8"),
    (dict(k_scale=torch.zeros(4, 16, 2, 4, dtype=BF16)), "scales must be matching"),
    (dict(v_scale=torch.zeros(4, 8, 2, 2, dtype=BF16)), "scales must be matching"),
    (dict(v_scale=torch.zeros(4, 16, 2, 2)), "scales must be bfloat16"),
    (dict(k_scale=torch.zeros(4, 16, 2, 1, dtype=BF16).expand(4, 16, 2, 2)), "contiguous along the groups"),
    (dict(k_scale=torch.zeros(4, 1, 2, 2, dtype=BF16).expand(4, 16, 2, 2)), "expanded"),
    (dict(positions=torch.zeros(2, 3, dtype=torch.int32)), "positions must be"),
    (dict(positions=torch.zeros(2, dtype=torch.int32)), "positions must be"),
])
def test_refused_caches(change, text):
    # .cuda() would lay out expanded tensors anew
    args = {n: t.cuda() if t.is_contiguous() else t[:, :1].cuda().expand_as(t) if text == "expanded" else
            t[..., :1].cuda().expand_as(t) for n, t in {**_cpu_step(), **change}.items()}
    with pytest.raises(ValueError, match=text):
        fap.append_paged_kv_int4(**args)


@pytest.mark.parametrize("cache,scale,dtype,text", [
    (torch.zeros(3, 32), torch.zeros(3, 2, dtype=BF16), BF16, "uint8"),
    (torch.zeros(3, 32, dtype=torch.uint8), torch.zeros(3, 2), BF16, "bfloat16"),
    (torch.zeros(3, 16, dtype=torch.uint8), torch.zeros(3, 1, dtype=BF16), BF16, "head dimension"),
    (torch.zeros(3, 32, dtype=torch.uint8), torch.zeros(3, 4, dtype=BF16), BF16, "scales must be"),
    (torch.zeros(3, 32, dtype=torch.uint8), torch.zeros(3, 2, dtype=BF16), torch.float32, "BF16 or FP16"),
    (torch.zeros(3, 32, dtype=torch.uint8), torch.zeros(3, 2, dtype=BF16), BF16, "CUDA devices only"),
])
def test_refused_unpacks(cache, scale, dtype, text):
    with pytest.raises(ValueError, match=text):
        fap.unpack_int4(cache, scale, dtype)
