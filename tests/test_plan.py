"""plan_paged_step: page tables, lengths, positions and slots of a step against a walk through it in Python."""
import random

import pytest
import torch

import flash_attn_prologue_b200 as fap
from flash_attn_prologue_b200 import _lib


def _walk(table, lens, news, free, count, page, tokens, keep):
    """The step by hand, on lists. Returns (table, free, count, lens, cu, positions, slots, requests, clean)."""
    table, free, size = [list(r) for r in table], list(free), len(free)
    width = len(table[0]) if table else 0
    clean, out, cu, grown = True, [], [0], []
    for r, (n, new) in enumerate(zip(lens, news)):
        held = -(-n // page)
        if new < 0:
            for c in range(keep[r] if keep else 0, held):
                if count < size:
                    free[count] = table[r][c]
                    count += 1
                else:
                    clean = False
        cu.append(cu[-1] + max(new, 0))
    for r, (n, new) in enumerate(zip(lens, news)):
        total = 0 if new < 0 else n + new
        if new >= 0:
            for c in range(-(-n // page), min(-(-total // page), width)):
                count -= 1
                if count < 0:
                    clean = False
                table[r][c] = free[count] if count >= 0 else -1
            clean = clean and total <= width * page
        out.append(total)
        for i in range(max(new, 0)):
            at = n + i
            p = table[r][at // page] if at // page < width else -1
            grown.append((at, p * page + at % page if p >= 0 else -1, r))
            clean = clean and p >= 0
    clean = clean and len(grown) <= tokens
    grown = grown[:tokens] + [(0, -1, -1)] * (tokens - len(grown))
    return table, free, max(count, 0), out, cu, *(list(x) for x in zip(*grown)), clean


def _check(lens, news, page, width, pool, tokens=None, keep=None, size=None, seed=0, stride=0):
    rng = random.Random(seed)
    B = len(lens)
    order = list(range(pool))
    rng.shuffle(order)
    table = [[-1] * width for _ in range(B)]
    for r, n in enumerate(lens):
        for c in range(min(-(-n // page), width)):
            table[r][c] = order.pop()
    count = len(order)
    size = pool if size is None else size
    free = order + [-7] * (size - count)
    tokens = sum(max(n, 0) for n in news) if tokens is None else tokens
    want = _walk(table, lens, news, free, count, page, tokens, keep)
    dev = lambda x: torch.tensor(x, dtype=torch.int32).reshape(-1).cuda()  # noqa: E731
    t = torch.full((B, width + stride), 99, dtype=torch.int32, device="cuda")[:, :width]
    t.copy_(torch.tensor(table, dtype=torch.int32).reshape(B, width))
    f = dev(free)
    given = (dev(lens), dev(news), dev([count]), None if keep is None else dev(keep))
    _lib.device_error()
    for _ in range(2):  # a second call with the same lengths does the same again
        got = fap.plan_paged_step(t, given[0], given[1], f, given[2], page, tokens, keep=given[3])
        assert t.tolist() == want[0]
        assert f.tolist() == want[1]
        assert got.free_count.tolist() == [want[2]]
        assert got.seq_lens.tolist() == want[3] and got.cu_seqlens.tolist() == want[4]
        if tokens:
            assert got.positions.tolist() == want[5] and got.slots.tolist() == want[6]
            assert got.requests.tolist() == want[7]
        assert (_lib.device_error() == 0) == want[-1]
    assert given[0].tolist() == lens and given[2].tolist() == [count]
    return got, t, f


@pytest.mark.gpu
@pytest.mark.parametrize("lens,news", [
    ([0], [1]), ([0], [0]), ([5], [-1]), ([8, 7, 9, 0], [1, 1, 1, 1]), ([8, 7, 9, 0, 31], [0, 20, -1, 3, -1]),
    ([16, 16, 16], [-1, -1, -1]), ([0, 0, 0, 0], [40, 0, 0, 17]), ([3, 60, 0, 22], [0, 0, 0, 0]),
])
@pytest.mark.parametrize("page", [8, 16])
def test_small_steps(lens, news, page):
    _check(lens, news, page, 9, 40, stride=3)
    _check(lens, news, page, 9, 40, tokens=sum(max(n, 0) for n in news) + 5)  # padding behind the tokens


@pytest.mark.gpu
@pytest.mark.parametrize("B", [1, 31, 32, 33, 1023, 1024, 1025, 2500])
def test_batches(B):
    rng = random.Random(B)
    lens = [rng.choice([0, 1, rng.randint(0, 300)]) for _ in range(B)]
    news = [rng.choice([-1, 0, 1, 1, 1, rng.randint(0, 60)]) for _ in range(B)]
    _check(lens, news, 16, 24, sum(-(-n // 16) for n in lens) + sum(-(-max(n, 0) // 16) + 1 for n in news), seed=B)


@pytest.mark.gpu
def test_many_tokens_and_the_largest_batch():
    _check([100, 0, 7], [20000, 9000, -1], 64, 400, 500)
    _check([9] * 8192, [-1, 8] * 4096, 8, 3, 20000)


@pytest.mark.gpu
def test_kept_pages_stay_out():
    _check([50, 33, 8, 20], [-1, -1, -1, 30], 8, 9, 40, keep=[2, 9, 0, 1])


@pytest.mark.gpu
def test_shortages():
    _check([8, 8, 8], [9, 9, 1], 8, 4, 6)                 # three pages left for five
    _check([8, 8], [40, 1], 8, 3, 30)                     # no room in the table
    _check([24, 24], [-1, -1], 8, 3, 10, size=7)          # no room on the stack
    _check([0, 0], [8, 8], 8, 3, 10, tokens=11)           # more tokens than rows
    _check([0], [4], 8, 0, 3)                             # a table without columns


@pytest.mark.gpu
def test_lengths_out_of_range_are_not_followed():
    for lens, news, count in (([-5, 8], [1, 1], 10), ([10 ** 9, 8], [1, 1], 10), ([8, 8], [2 ** 31 - 1, 1], 10),
                              ([8, 8], [1, 1], -3), ([8, 8], [-1, 1], 10 ** 9)):
        guard = torch.full((6, 4), 3, dtype=torch.int32, device="cuda")
        stack = torch.full((40,), 5, dtype=torch.int32, device="cuda")
        _lib.device_error()
        dev = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
        fap.plan_paged_step(guard[2:4], dev(lens), dev(news), stack[10:20], dev([count]), 8, 2)
        assert _lib.device_error() == 2
        assert (guard[:2] == 3).all() and (guard[4:] == 3).all()
        assert (stack[:10] == 5).all() and (stack[20:] == 5).all()


@pytest.mark.gpu
def test_steps_in_a_row_hand_out_every_page_once():
    rng = random.Random(3)
    page, B, width, pool = 8, 40, 20, 500
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    free = torch.randperm(pool, device="cuda").to(torch.int32)
    lens, count = torch.zeros(B, dtype=torch.int32, device="cuda"), torch.tensor([pool], dtype=torch.int32, device="cuda")
    for _ in range(30):
        now = lens.tolist()
        news = [-1 if n and rng.random() < 0.2 else rng.randint(0, min(25, width * page - n)) for n in now]
        step = fap.plan_paged_step(table, lens, torch.tensor(news, dtype=torch.int32, device="cuda"), free, count, page,
                                   sum(max(n, 0) for n in news))
        lens, count = step.seq_lens, step.free_count
        held = [p for r, n in enumerate(lens.tolist()) for p in table[r, :-(-n // page)].tolist()]
        left = free[:int(count)].tolist()
        assert sorted(held + left) == list(range(pool))
        slots = step.slots.tolist()
        assert len(set(slots)) == len(slots)
    assert _lib.device_error() == 0


@pytest.mark.gpu
def test_captured_steps_follow_their_buffers():
    table = torch.full((3, 8), -1, dtype=torch.int32, device="cuda")
    free = torch.arange(20, dtype=torch.int32, device="cuda")
    lens, news = (torch.zeros(3, dtype=torch.int32, device="cuda") for _ in range(2))
    count = torch.tensor([20], dtype=torch.int32, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fap.plan_paged_step(table, lens, news, free, count, 8, 4)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step = fap.plan_paged_step(table, lens, news, free, count, 8, 4)
        lens.copy_(step.seq_lens)
        count.copy_(step.free_count)
    grown = [0, 0, 0]
    for new in ([4, 0, 0], [1, 1, 1], [0, 3, 1], [4, 0, 0], [0, 0, 4]):
        news.copy_(torch.tensor(new))
        graph.replay()
        grown = [a + b for a, b in zip(grown, new)]
        assert lens.tolist() == grown and int(count) == 20 - sum(-(-n // 8) for n in grown)
        request, position = step.requests[:sum(new)].long(), step.positions[:sum(new)].long()
        assert request.tolist() == [r for r, n in enumerate(new) for _ in range(n)]
        assert torch.equal(step.slots[:sum(new)], table[request, position // 8].long() * 8 + position % 8)


@pytest.mark.gpu
def test_opcheck_and_compiled():
    def args():
        return (torch.full((2, 3), -1, dtype=torch.int32, device="cuda"),
                *(torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 0], [9, 1], list(range(8)), [8])), 8, 10)

    result = torch.library.opcheck(torch.ops.flash_prologue.plan_paged_step.default, args(),
                                   test_utils=("test_schema", "test_faketensor"))
    assert set(result.values()) == {"SUCCESS"}, result
    a, b = args(), args()
    for x, y in zip(fap.plan_paged_step(*a), torch.compile(fap.plan_paged_step, fullgraph=True)(*b)):
        assert torch.equal(x, y)
    assert torch.equal(a[0], b[0])


def _cpu():
    i = lambda *x: torch.zeros(*x, dtype=torch.int32)  # noqa: E731
    return dict(page_table=i(2, 3), seq_lens=i(2), new_lens=i(2), free_pages=i(8), free_count=i(1), page_size=8, tokens=2)


@pytest.mark.parametrize("change,text", [
    (dict(page_table=torch.zeros(6, dtype=torch.int32)), "page_table must be"),
    (dict(seq_lens=torch.zeros(3, dtype=torch.int32)), "page_table must be"),
    (dict(new_lens=torch.zeros(1, dtype=torch.int32)), "page_table must be"),
    (dict(free_pages=torch.zeros(2, 4, dtype=torch.int32)), "stack"),
    (dict(free_count=torch.zeros((), dtype=torch.int32)), "stack"),
    (dict(keep=torch.zeros(3, dtype=torch.int32)), "keep must be"),
    (dict(seq_lens=torch.zeros(2, dtype=torch.int64)), "must be int32"),
    (dict(keep=torch.zeros(2, dtype=torch.int64)), "must be int32"),
    (dict(page_table=torch.zeros(3, 2, dtype=torch.int32).T), "contiguous"),
    (dict(free_pages=torch.zeros(16, dtype=torch.int32)[::2]), "contiguous"),
    (dict(page_table=torch.zeros(1, 3, dtype=torch.int32).expand(2, 3)), "share memory"),
    (dict(page_size=12), "power of two"),
    (dict(page_size=4), "power of two"),
    (dict(tokens=-1), "negative"),
    (dict(), "CUDA devices only"),
])
def test_refusals(change, text):
    with pytest.raises(ValueError, match=text):
        fap.plan_paged_step(**{**_cpu(), **change})


def test_too_many_requests_are_refused():
    n = 8193
    i = lambda *x: torch.zeros(*x, dtype=torch.int32)  # noqa: E731
    with pytest.raises(ValueError, match="8192"):
        fap.plan_paged_step(i(n, 1), i(n), i(n), i(8), i(1), 8, 0)


@pytest.mark.gpu
def test_nothing_to_plan():
    empty = torch.zeros(0, dtype=torch.int32, device="cuda")
    count = torch.zeros(1, dtype=torch.int32, device="cuda")
    _lib.device_error()
    for tokens in (0, 3):
        step = fap.plan_paged_step(empty.view(0, 4), empty, empty, empty, count, 16, tokens)
        assert step.cu_seqlens.tolist() == [0] and step.free_count.tolist() == [0] and step.seq_lens.numel() == 0
        assert step.requests.tolist() == step.slots.tolist() == [-1] * tokens and step.positions.tolist() == [0] * tokens
    assert _lib.device_error() == 0
