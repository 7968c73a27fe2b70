"""append_paged_kv: rotated K, V and Q of a step's new tokens against the formula in 64 bits."""
import pytest
import torch

import flash_attn_prologue_b200 as fap
from flash_attn_prologue_b200 import _lib
from tests._paged import Requests, assert_within, rotate64, tables

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


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


def _check(req, args, decode=False):
    q, k, v, w, s, sin, cos = args
    k0, v0 = req.k.clone(), req.v.clone()
    got = fap.append_paged_kv(*args, req.k, req.v, req.table, req.seq_lens, None if decode else req.cu)
    assert got.shape == q.shape and got.is_contiguous()
    at = torch.cat([torch.arange(t - n, t, device="cuda") for n, t in zip(req.news, req.totals)])
    sn, cs = sin[at][:, None], cos[at][:, None]
    gain = 1.0 if s is None else s.double().exp().view(-1, 1)
    assert_within(got, *rotate64(q, None if w is None else w[0], sn, cs, gain), "q")
    k_rows, k_size = rotate64(k, None if w is None else w[1], sn, cs, 1.0)
    begin = 0
    for r, (n, t) in enumerate(zip(req.news, req.totals)):
        where = req.places(r, t - n, t)
        assert_within(req.k[where], k_rows[begin:begin + n], k_size[begin:begin + n], "k")
        assert torch.equal(req.v[where], v[begin:begin + n])
        k0[where], v0[where] = req.k[where], req.v[where]
        begin += n
    # nothing else of the cache has changed
    for now, was in ((req.k, k0), (req.v, v0)):
        assert torch.equal(now.nan_to_num(77.0), was.nan_to_num(77.0)) and torch.equal(now.isnan(), was.isnan())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("Hq,Hk,page,hnd,norm,odd", [
    (8, 2, 16, False, True, False), (15, 5, 8, True, True, False), (4, 4, 64, False, False, False),
    (6, 1, 128, True, True, True),
])
def test_chunks(Hq, Hk, page, hnd, norm, odd, D, dtype):
    req = Requests([3, 0, 40, 1, 17], [3, 9, 140, 1, 64], Hq, Hk, D, page, dtype, hnd)
    _check(req, _inputs(req, Hq, Hk, D, dtype, norm, odd))


@pytest.mark.gpu
@pytest.mark.parametrize("totals", [[1], [8, 9, 7, 1], list(range(1, 200, 2))])
def test_single_tokens(totals):
    req = Requests([1] * len(totals), totals, 32, 8, 128, 8, BF16)
    _check(req, _inputs(req, 32, 8, 128, BF16), decode=True)


@pytest.mark.gpu
def test_long_chunk_and_empty_step():
    req = Requests([2500, 0, 1111], [2500, 30, 6000], 32, 8, 128, 64, BF16)
    _check(req, _inputs(req, 32, 8, 128, BF16))
    req = Requests([0, 0], [5, 0], 8, 2, 64, 16, BF16)
    _check(req, _inputs(req, 8, 2, 64, BF16))


@pytest.mark.gpu
def test_the_same_rows_as_the_training_prologue():
    req = Requests([50], [50], 8, 2, 64, 16, BF16)
    q, k, v, w, s, sin, cos = _inputs(req, 8, 2, 64, BF16)
    got = fap.append_paged_kv(q, k, v, w, s, sin, cos, req.k, req.v, req.table, req.seq_lens, req.cu)
    q_out, k_out = fap.qknorm_rope_scale_gqa(q, k, w, s, sin, cos)
    assert torch.equal(got, q_out) and torch.equal(req.k[req.places(0, 0, 50)], k_out)


@pytest.mark.gpu
def test_indices_out_of_range_are_not_followed():
    def step(change, lost):
        req = Requests([4, 3, 1], [20, 3, 9], 8, 2, 64, 8, BF16)
        args = _inputs(req, 8, 2, 64, BF16)
        changed = change(req, args)
        rotation = changed if isinstance(changed, tuple) else args[5:]
        k0 = req.k.clone()
        _lib.device_error()
        got = fap.append_paged_kv(*args[:5], *rotation, req.k, req.v, req.table, req.seq_lens, req.cu)
        assert _lib.device_error() == 2
        zero = (got == 0).flatten(1).all(1).tolist()
        assert zero == [i in lost for i in range(8)]
        written = (req.k.nan_to_num(77.0) != k0.nan_to_num(77.0)).flatten(2).any(2).sum()
        assert int(written) == 8 - len(lost)

    step(lambda r, a: r.table[0].fill_(-1), {0, 1, 2, 3})
    step(lambda r, a: r.table[2].fill_(10 ** 6), {7})
    step(lambda r, a: r.seq_lens.copy_(torch.tensor([20, 1, 9])), {4, 5})       # starts before position 0
    step(lambda r, a: r.seq_lens.copy_(torch.tensor([20, 3, 10 ** 6])), {7})    # past the page table
    step(lambda r, a: tuple(t[:18] for t in a[5:]), {2, 3})                              # past the tables


@pytest.mark.gpu
@pytest.mark.parametrize("ragged", [True, False])
@pytest.mark.parametrize("pages", [5, 0])
def test_requests_without_pages_write_nothing(pages, ragged):
    """A page table without columns (its tensor has no address), with and without a cache behind it."""
    g = torch.Generator(device="cuda").manual_seed(0)
    news = [4, 0, 2] if ragged else [1, 1, 1]
    q, k, v = (torch.randn(sum(news), h, 64, generator=g, device="cuda").to(BF16) for h in (8, 2, 2))
    w, s = torch.ones(2, 1, 64, device="cuda"), torch.zeros(8, 1, 1, device="cuda")
    caches = [torch.randn(pages, 16, 2, 64, generator=g, device="cuda").to(BF16) for _ in range(2)]
    kept = [c.clone() for c in caches]
    table = torch.zeros(3, 0, dtype=torch.int32, device="cuda")
    lens = torch.tensor(news, dtype=torch.int32, device="cuda")
    cu = torch.tensor([0] + news).cumsum(0).to(torch.int32).cuda() if ragged else None
    _lib.device_error()
    got = fap.append_paged_kv(q, k, v, w, s, *tables(8, 64), *caches, table, lens, cu)
    assert _lib.device_error() == 2
    assert got.shape == q.shape and not got.any()
    assert all(torch.equal(a, b) for a, b in zip(caches, kept))
    out, lse = fap.paged_attention(q, *caches, table, lens, cu, return_lse=True)
    assert _lib.device_error() == 2
    assert out.isnan().all() and lse.isnan().all()


@pytest.mark.gpu
def test_padding_tokens_come_back_as_zeros():
    req = Requests([4, 3, 2], [20, 3, 9], 8, 2, 64, 8, BF16)
    args = _inputs(req, 8, 2, 64, BF16)
    k0 = req.k.clone()
    _lib.device_error()
    got = fap.append_paged_kv(*args, req.k, req.v, req.table[:2], req.seq_lens[:2], req.cu[:3])
    assert not got[7:].any() and got[:7].any(-1).all() and _lib.device_error() == 0
    where = req.places(2, 7, 9)
    assert torch.equal(req.k[where], k0[where])


@pytest.mark.gpu
def test_captured_step_follows_its_buffers():
    req = Requests([2, 1], [10, 5], 8, 2, 64, 16, BF16)
    args = _inputs(req, 8, 2, 64, BF16)
    call = lambda: fap.append_paged_kv(*args, req.k, req.v, req.table, req.seq_lens, req.cu)  # noqa: E731
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
    replayed = out.clone(), req.k.clone()
    assert torch.equal(call(), replayed[0])
    assert torch.equal(req.k.nan_to_num(77.0), replayed[1].nan_to_num(77.0))


@pytest.mark.gpu
def test_opcheck_and_compiled():
    req = Requests([2, 1], [10, 5], 8, 2, 64, 16, BF16)
    args = (*_inputs(req, 8, 2, 64, BF16), req.k.nan_to_num(0.0), req.v.nan_to_num(0.0), req.table, req.seq_lens, req.cu)
    result = torch.library.opcheck(torch.ops.flash_prologue.append_paged_kv.default, (*args, 1e-5),
                                   test_utils=("test_schema", "test_faketensor"))
    assert set(result.values()) == {"SUCCESS"}, result
    eager = fap.append_paged_kv(*args)
    assert torch.equal(torch.compile(fap.append_paged_kv, fullgraph=True)(*args), eager)


def _cpu_step(T=3, Hq=8, Hk=2, D=64, page=16, dtype=BF16):
    sin, cos = tables(8, D, "cpu")
    return dict(q=torch.zeros(T, Hq, D, dtype=dtype), k=torch.zeros(T, Hk, D, dtype=dtype),
                v=torch.zeros(T, Hk, D, dtype=dtype), rmsnorm_weight=torch.ones(2, 1, D), scales=torch.zeros(Hq, 1, 1),
                sin=sin, cos=cos, k_cache=torch.zeros(4, page, Hk, D, dtype=dtype),
                v_cache=torch.zeros(4, page, Hk, D, dtype=dtype), page_table=torch.zeros(3, 1, dtype=torch.int32),
                seq_lens=torch.ones(3, dtype=torch.int32))


@pytest.mark.parametrize("change,text", [
    (dict(q=torch.zeros(1, 3, 8, 64, dtype=BF16)), "must be packed"),
    (dict(v=torch.zeros(3, 4, 64, dtype=BF16)), "must be packed"),
    (dict(v=torch.zeros(3, 2, 64)), "must be packed"),
    (dict(scales=torch.zeros(2, 1, 1)), "log-scales"),
    (dict(q=torch.zeros(3, 8, 64, dtype=BF16, requires_grad=True)), "not differentiable"),
    (dict(), "CUDA devices only"),
])
def test_refusals(change, text):
    with pytest.raises(ValueError, match=text):
        fap.append_paged_kv(**{**_cpu_step(), **change})


@pytest.mark.gpu
@pytest.mark.parametrize("change,text", [
    (dict(k_cache=torch.zeros(4, 16, 2, 32, dtype=BF16)), "matching"),
    (dict(v_cache=torch.zeros(5, 16, 2, 64, dtype=BF16)), "matching"),
    (dict(k_cache=torch.zeros(4, 12, 2, 64, dtype=BF16), v_cache=torch.zeros(4, 12, 2, 64, dtype=BF16)), "power of two"),
    (dict(k_cache=torch.zeros(4, 4, 2, 64, dtype=BF16), v_cache=torch.zeros(4, 4, 2, 64, dtype=BF16)), "power of two"),
    (dict(k_cache=torch.zeros(4, 16, 4, 64, dtype=BF16), v_cache=torch.zeros(4, 16, 4, 64, dtype=BF16)), "same key heads"),
    (dict(k_cache=torch.zeros(4, 16, 2, 64), v_cache=torch.zeros(4, 16, 2, 64)), "share a dtype"),
    (dict(page_table=torch.zeros(3, 1, dtype=torch.int64)), "must be int32"),
    (dict(page_table=torch.zeros(2, 1, dtype=torch.int32)), "page_table must be"),
    (dict(cu_seqlens=torch.zeros(3, dtype=torch.int32)), "cu_seqlens must be"),
    (dict(page_table=torch.zeros(2, 1, dtype=torch.int32), seq_lens=torch.ones(2, dtype=torch.int32)), "one token"),
])
def test_refused_caches(change, text):
    args = {n: t.cuda() for n, t in {**_cpu_step(), **change}.items()}
    with pytest.raises(ValueError, match=text):
        fap.append_paged_kv(**args)
    with pytest.raises(ValueError, match="expanded"):
        good = {n: t.cuda() for n, t in _cpu_step().items()}
        good["v_cache"] = good["v_cache"][:, :, :1].expand(-1, -1, 2, -1)
        fap.append_paged_kv(**good)
    with pytest.raises(ValueError, match="contiguous along D"):
        good = {n: t.cuda() for n, t in _cpu_step().items()}
        good["k_cache"] = good["k_cache"].transpose(0, 3).contiguous().transpose(0, 3)
        fap.append_paged_kv(**good)
