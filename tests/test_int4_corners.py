"""Calls of the 4-bit cache's operators at the ends of what they take."""
import math

import pytest
import torch

import flash_attn_prologue_b200 as fap
from flash_attn_prologue_b200 import _lib
from tests._int4 import Requests4
from tests._paged import tables
from tests.test_int4_attention import _attend, _check

BF16, FP16 = torch.bfloat16, torch.float16


def _int(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("news", [[1, 1], [40, 30]])
@pytest.mark.parametrize("Hk", [2, 4])
def test_a_cache_without_pages(news, Hk):
    """Requests without tokens have rows of zeros; those that should have some have NaN, and the error word is set."""
    cache = fap.int4_cache(0, 16, Hk, 64)
    q = torch.randn(sum(news), 8, 64, device="cuda").to(BF16)
    cu = _int(0, news[0], sum(news))
    for width in (0, 3):
        table = torch.zeros(2, width, dtype=torch.int32, device="cuda")
        _lib.device_error()
        out, lse = fap.paged_attention_int4(q, *cache, table, _int(0, 0), cu, return_lse=True)
        assert not out.any() and (lse == -math.inf).all() and _lib.device_error() == 0
        out = fap.paged_attention_int4(q, *cache, table, _int(48, 48), cu)
        assert out[news[0] - 1].isnan().all() and out[-1].isnan().all() and _lib.device_error() == 2


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [0, 5])
def test_no_requests(rows):
    cache = fap.int4_cache(4, 16, 2, 64)
    q, k, v = (torch.ones(rows, h, 64, dtype=BF16, device="cuda") for h in (8, 2, 2))
    table, lens, cu = torch.zeros(0, 3, dtype=torch.int32, device="cuda"), _int(), _int(0)
    sin, cos = tables(16, 64)
    calls = (lambda: fap.paged_attention_int4(q, *cache, table, lens, cu),
             lambda: fap.append_paged_kv_int4(q, k, v, None, None, sin, cos, *cache, table, lens, cu))
    for call in calls:
        if rows:  # whose tokens are they? refused, as over a 16-bit cache
            with pytest.raises(ValueError, match="invalid argument"):
                call()
        else:
            assert call().shape == q.shape


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hk", [(512, 1), (512, 2), (300, 1), (512, 512)])
@pytest.mark.parametrize("news,totals", [([1, 1], [300, 40]), ([3, 0, 25], [200, 5, 90])])
def test_many_heads(Hq, Hk, news, totals):
    req = Requests4(news, totals, Hq, Hk, 64, 16, FP16)
    _check(req, req.q.half())


@pytest.mark.gpu
@pytest.mark.parametrize("page", [8, 1024])
@pytest.mark.parametrize("news", [[1, 1, 1, 1], [70, 1, 40, 200]])
def test_pages_of_every_size(page, news):
    req = Requests4(news, [2100, 1, 1025, 1024], 8, 2, 128, page, BF16)
    _check(req, req.q.to(BF16))


@pytest.mark.gpu
@pytest.mark.parametrize("news,totals", [([1] * 6, [9000, 3, 900, 77, 2000, 5000]), ([900, 40, 300], [900, 2500, 3000])])
def test_two_calls_at_once(news, totals):
    reqs = [Requests4(news, totals, 16, 4, 128, 16, BF16, seed=s) for s in (0, 1)]
    qs = [r.q.to(BF16) for r in reqs]
    alone = [_attend(r, q) for r, q in zip(reqs, qs)]
    streams = [torch.cuda.Stream() for _ in reqs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    outs = []
    for _ in range(10):
        for s, r, q in zip(streams, reqs, qs):
            with torch.cuda.stream(s):
                outs.append(_attend(r, q))
    torch.cuda.synchronize()
    assert all(torch.equal(out, alone[i % 2]) for i, out in enumerate(outs))


@pytest.mark.gpu
@pytest.mark.parametrize("news", [[1], [40]])
def test_strides_of_64_bits(news):
    """A single page's stride means nothing; two pages too far apart are refused before they are read."""
    req = Requests4(news, [50], 8, 2, 64, 64, BF16)
    q = req.q.to(BF16)
    clean = _attend(req, q)
    one = [t[req.table[0, 0]:][:1] for t in req.cache]
    far = [torch.as_strided(t, t.shape, (2 ** 33, *t.stride()[1:]), t.storage_offset()) for t in one]
    got = fap.paged_attention_int4(q, *far, torch.zeros_like(req.table), req.seq_lens, req.cu)
    assert torch.equal(got, clean)
    storage = torch.empty(2 ** 31 + 2 ** 20, dtype=torch.uint8, device="cuda")
    wide = torch.as_strided(storage, (2, 64, 2, 32), (2 ** 31, 64, 32, 1))
    scale = torch.zeros(2, 64, 2, 2, dtype=BF16, device="cuda")
    with pytest.raises(ValueError, match="unsupported"):
        fap.paged_attention_int4(q, wide, wide, scale, scale, torch.zeros_like(req.table), req.seq_lens, req.cu)


@pytest.mark.gpu
def test_the_same_slot_written_twice_in_a_row():
    """A step taken back by its length: the slot is written anew, and attention sees the later row only."""
    g = torch.Generator(device="cuda").manual_seed(0)
    sin, cos = tables(64, 64)
    caches = [fap.int4_cache(3, 16, 2, 64) for _ in range(2)]
    rows = [[torch.randn(1, h, 64, generator=g, device="cuda").to(BF16) for h in (8, 2, 2)] for _ in range(2)]
    table, lens = _int(2, 0, 1).view(1, 3), _int(20)
    for r in rows:
        fap.append_paged_kv_int4(*r, None, None, sin, cos, *caches[0], table, lens)
    fap.append_paged_kv_int4(*rows[1], None, None, sin, cos, *caches[1], table, lens)
    assert all(torch.equal(a, b) for a, b in zip(*caches))
