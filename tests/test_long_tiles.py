"""Tiles of rows that take longer than a wait for one block may."""
import pytest
import torch

import flash_attn_prologue_b200 as fap
from flash_attn_prologue_b200 import _lib


@pytest.mark.gpu
def test_a_tile_of_seconds_sets_no_error():
    """As many tiles as the GPU holds at once, of 335 million keys each (a table that names the same pages again)."""
    g = torch.Generator(device="cuda").manual_seed(0)
    tokens = 2 * torch.cuda.get_device_properties(0).multi_processor_count  # of 128 rows, whole tiles
    cache = fap.int4_cache(4, 1024, 1, 64)
    for codes, scale in zip(cache[:2], cache[2:]):
        codes.random_(0, 256, generator=g)
        scale.fill_(0.25)
    width = 327680
    table = torch.randint(0, 4, (1, width), generator=g, device="cuda", dtype=torch.int32)
    lens = torch.tensor([1024 * width], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, tokens], dtype=torch.int32, device="cuda")
    q = (0.1 * torch.randn(tokens, 128, 64, generator=g, device="cuda")).to(torch.bfloat16)
    _lib.device_error()
    out = fap.paged_attention_int4(q, *cache, table, lens, cu)
    assert _lib.device_error() == 0
    assert out.isfinite().all()


@pytest.mark.gpu
def test_warps_without_rows_beside_tiles_of_seconds():
    """At D = 128 tiles are of 256 rows; here each has 128, so half a CTA's row warps only wait, and then one has 256."""
    g = torch.Generator(device="cuda").manual_seed(0)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    cache = fap.int4_cache(4, 1024, 1, 128)
    for codes, scale in zip(cache[:2], cache[2:]):
        codes.random_(0, 256, generator=g)
        scale.fill_(0.25)
    # the last tiles come first: one a CTA over all keys, then a short one, then the first request's tile of two tokens
    news, long = [2] + [1] * (2 * sms - 1), 1024 * 360448
    totals = [64] * sms + [long] * sms
    width = long // 1024
    row = torch.randint(0, 4, (1, width), generator=g, device="cuda", dtype=torch.int32)
    table = torch.as_strided(row, (len(news), width), (0, 1))
    lens = torch.tensor(totals, dtype=torch.int32, device="cuda")
    cu = torch.tensor([0] + news).cumsum(0).to(torch.int32).cuda()
    q = (0.1 * torch.randn(sum(news), 128, 128, generator=g, device="cuda")).to(torch.bfloat16)
    short = fap.paged_attention_int4(q[:sms + 1], *cache, table[:sms, :1].contiguous(), lens[:sms], cu[:sms + 1])
    _lib.device_error()
    out = fap.paged_attention_int4(q, *cache, table, lens, cu)
    assert _lib.device_error() == 0
    assert out.isfinite().all()
    torch.testing.assert_close(out[:sms + 1], short, rtol=2 ** -7, atol=2 ** -7)


@pytest.mark.gpu
def test_a_tile_of_seconds_over_a_16_bit_cache():
    g = torch.Generator(device="cuda").manual_seed(0)
    tokens = 2 * torch.cuda.get_device_properties(0).multi_processor_count
    k, v = (torch.randn(4, 1024, 1, 64, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    width = 360448
    table = torch.randint(0, 4, (1, width), generator=g, device="cuda", dtype=torch.int32)
    lens = torch.tensor([1024 * width], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, tokens], dtype=torch.int32, device="cuda")
    q = (0.1 * torch.randn(tokens, 128, 64, generator=g, device="cuda")).to(torch.bfloat16)
    _lib.device_error()
    out = fap.paged_attention(q, k, v, table, lens, cu)
    assert _lib.device_error() == 0
    assert out.isfinite().all()
