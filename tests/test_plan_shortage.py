"""plan_paged_step after pages ran out: what ended requests return, and the steps that follow."""
import random

import pytest
import torch

import flash_attn_prologue_b200 as fap
from flash_attn_prologue_b200 import _lib
from tests._paged import tables


def _by_hand(table, lens, news, free, count, page, tokens, keep):
    """The step on lists; only entries that are pages go back. Returns what _run returns."""
    table, free, width = [list(r) for r in table], list(free), len(table[0])
    clean = True
    for r, (n, new) in enumerate(zip(lens, news)):
        if new < 0:
            for p in table[r][keep[r] if keep else 0:-(-n // page)]:
                if p >= 0 and count < len(free):
                    free[count] = p
                    count += 1
                elif p >= 0:
                    clean = False
    out, cu, rows = [], [0], []
    for r, (n, new) in enumerate(zip(lens, news)):
        total = 0 if new < 0 else n + new
        for c in range(-(-n // page), min(-(-total // page), width)):
            count -= 1
            clean = clean and count >= 0
            table[r][c] = free[count] if count >= 0 else -1
        for at in range(n, total):
            p = table[r][at // page] if at // page < width else -1
            clean = clean and p >= 0
            rows.append((at, p * page + at % page if p >= 0 else -1, r))
        out.append(total)
        cu.append(cu[-1] + max(new, 0))
    clean = clean and len(rows) <= tokens
    rows = rows[:tokens] + [(0, -1, -1)] * (tokens - len(rows))
    return table, free, max(count, 0), out, cu, *([x[i] for x in rows] for i in range(3)), clean


def _dev(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _run(table, lens, news, free, count, page, tokens, keep):
    t, f = _dev(table), _dev(free)
    _lib.device_error()
    for _ in range(2):  # a second call with the same lengths and count does the same again
        got = fap.plan_paged_step(t, _dev(lens), _dev(news), f, _dev([count]), page, tokens, keep=keep and _dev(keep))
    return (t.tolist(), f.tolist(), int(got.free_count), got.seq_lens.tolist(), got.cu_seqlens.tolist(),
            got.positions.tolist(), got.slots.tolist(), got.requests.tolist(), _lib.device_error() == 0)


def _step(table, lens, news, free, count, page, tokens=None, keep=None):
    tokens = sum(max(n, 0) for n in news) if tokens is None else tokens
    args = (table, lens, news, free, count, page, tokens, keep)
    got = _run(*args)
    for name, a, b in zip(("table", "stack", "count", "lengths", "starts", "positions", "slots", "requests", "clean"),
                          got, _by_hand(*args)):
        assert a == b, name
    return got


@pytest.mark.gpu
def test_a_short_request_returns_the_pages_that_it_has():
    table, free, lens, count = [[-1] * 4 for _ in range(3)], [0, 1, 2], [0, 0, 0], 3
    table, free, count, lens, *_, clean = _step(table, lens, [8, 24, 0], free, count, 8)
    assert not clean and count == 0 and table[1][2] == -1
    table, free, count, lens, *_, clean = _step(table, lens, [0, -1, 0], free, count, 8)
    assert clean and count == 2 and sorted(free[:2] + table[0][:1]) == [0, 1, 2]
    table, free, count, lens, *_, clean = _step(table, lens, [0, 0, 8], free, count, 8)
    assert clean and count == 1 and table[2][0] >= 0
    table, free, count, lens, *_, clean = _step(table, lens, [-1, 0, -1], free, count, 8)
    assert clean and count == 3 and sorted(free) == [0, 1, 2]


@pytest.mark.gpu
@pytest.mark.parametrize("B,width,pool,page,seed", [(3, 6, 10, 8, 0), (40, 12, 150, 8, 1), (70, 9, 200, 16, 2), (1100, 5, 2300, 8, 3)])
def test_no_page_is_lost_or_doubled_over_short_steps(B, width, pool, page, seed):
    rng = random.Random(seed)
    table, lens, count = [[-1] * width for _ in range(B)], [0] * B, pool
    free = rng.sample(range(pool), pool)
    shortages = 0
    for _ in range(14 if B < 1000 else 5):
        news = [-1 if n and rng.random() < 0.3 else rng.randint(0, min(3 * page, width * page - n)) for n in lens]
        table, free, count, lens, *_, clean = _step(table, lens, news, free, count, page, tokens=sum(map(abs, news)) + 3)
        held = [p for r, n in enumerate(lens) for p in table[r][:-(-n // page)]]
        shortages += -1 in held
        assert sorted(free[:count] + [p for p in held if p >= 0]) == list(range(pool))
    assert shortages > 1
    table, free, count, lens, *_, clean = _step(table, lens, [-1] * B, free, count, page)
    assert clean and sorted(free) == list(range(pool)) and count == pool


@pytest.mark.gpu
@pytest.mark.parametrize("width", [3, 40, 3000])
def test_entries_that_are_no_pages_anywhere_in_a_row(width):
    """Pages that a server took out of its rows itself, kept ones among them."""
    rng = random.Random(width)
    pages = rng.sample(range(10 ** 6), 5 * width + 30)
    table = [[pages.pop() if rng.random() < 0.7 or c == width // 2 else rng.choice([-1, -9]) for c in range(width)]
             for _ in range(5)]
    table[3] = [-1] * width
    lens = [8 * width, 8 * (width - 1) - 3, 8 * width, 8 * width, 8 * (width - 2)]
    free = [pages.pop() for _ in range(20)] + [-5] * (4 * width)
    for keep in (None, [2, 0, 1, 1, 0]):
        for size in (len(free), 20 + width):  # room on the stack for all of them, and not
            _step(table, lens, [-1, -1, 0, -1, 9], free[:size], 20, 8, keep=keep)
            _step(table, lens, [-1, 10, -1, -1, -1], free[:size], 20, 8, tokens=14, keep=keep)


@pytest.mark.gpu
@pytest.mark.parametrize("int4", [False, True])
def test_a_request_served_from_pages_that_a_short_one_gave_back(int4):
    g = torch.Generator(device="cuda").manual_seed(0)
    table, free = torch.full((3, 4), -1, dtype=torch.int32, device="cuda"), _dev([0, 1, 2])
    lens, count = _dev([0, 0, 0]), _dev([3])
    sin, cos = tables(32, 64)

    def caches():
        if int4:
            return fap.int4_cache(3, 8, 2, 64)
        return [torch.zeros(3, 8, 2, 64, dtype=torch.bfloat16, device="cuda") for _ in range(2)]

    append, attend = (fap.append_paged_kv_int4, fap.paged_attention_int4) if int4 else (fap.append_paged_kv, fap.paged_attention)
    cache = caches()
    for news, short in (([8, 24, 0], True), ([0, -1, 0], False), ([0, 0, 8], False)):
        tokens = sum(max(n, 0) for n in news)
        q, k, v = (torch.randn(tokens, h, 64, generator=g, device="cuda").to(torch.bfloat16) for h in (8, 2, 2))
        _lib.device_error()
        step = fap.plan_paged_step(table, lens, _dev(news), free, count, 8, tokens)
        lens, count = step.seq_lens, step.free_count
        rows = append(q, k, v, None, None, sin, cos, *cache, table, lens, step.cu_seqlens)
        out = attend(rows, *cache, table, lens, step.cu_seqlens, softmax_scale=0.125)
        assert (_lib.device_error() != 0) == short
        assert not tokens or bool(out[-1].isnan().all()) == short
    alone = caches()
    rows = append(q, k, v, None, None, sin, cos, *alone, _dev([[0], [0], [1]]), lens, step.cu_seqlens)
    assert torch.equal(out, attend(rows, *alone, _dev([[0], [0], [1]]), lens, step.cu_seqlens, softmax_scale=0.125))
