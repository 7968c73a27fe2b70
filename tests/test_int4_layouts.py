"""Which layouts of a 4-bit cache single-token attention copies by tensor maps, seen by the kernels that run; each is right."""
import pytest
import torch

from tests._int4 import Requests4
from tests.test_int4_attention import _attend, _check

BF16 = torch.bfloat16


def _by_copies(call):
    """Whether the kernel that `call` runs is the one with tensor copies."""
    call()
    names = set()
    for _ in range(3):  # a profile may come back without its events
        with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CUDA]) as p:
            call()
            torch.cuda.synchronize()
        names |= {e.name for e in p.events() if "paged_int4_decode_kernel<" in e.name}
        if names:
            break
    assert len(names) == 1, names
    name = names.pop()
    last = name[name.index("<") + 1:name.index(">")].split(",")[-1]
    return "true" in last or last.strip().endswith("1")


@pytest.mark.gpu
@pytest.mark.parametrize("Hk,D,page,hnd,copies", [
    # scales of a slot's heads next to each other: multiples of four heads with 16 slots a page, of two at D = 128 with 32
    (4, 64, 16, False, True), (8, 128, 16, False, True), (12, 64, 32, False, True), (4, 128, 8, False, False),
    (2, 128, 32, False, True), (6, 128, 32, False, True), (2, 128, 16, False, False), (2, 64, 64, False, False),
    (6, 64, 64, False, False), (1, 128, 64, False, True), (1, 64, 128, False, True), (1, 64, 32, False, False), (3, 128, 64, False, False), (5, 128, 64, False, False),
    # scales of a head's slots next to each other: also two heads at D = 64, and one or five with 64 slots
    (8, 64, 16, True, True), (2, 64, 32, True, True), (6, 128, 32, True, True), (1, 64, 64, True, True), (1, 128, 64, True, True),
    (5, 64, 64, True, True), (1, 128, 32, True, False), (3, 128, 64, True, False), (7, 64, 64, True, False),
])
def test_copies_by_layout(Hk, D, page, hnd, copies):
    req = Requests4([1, 1], [700, 200], 2 * Hk, Hk, D, page, BF16, hnd)
    q = req.q.to(BF16)
    assert _by_copies(lambda: _attend(req, q, decode=True)) == copies
    _check(req, q, decode=True)


@pytest.mark.gpu
def test_scales_off_sixteen_bytes_are_loaded_row_by_row():
    req = Requests4([1, 1], [700, 200], 16, 8, 128, 16, BF16)
    q = req.q.to(BF16)
    whole = _attend(req, q, decode=True)
    for i in range(2):
        kept = req.scales[i]
        room = torch.zeros(kept.numel() + 4, dtype=BF16, device="cuda")
        req.scales[i] = room[4:].view(kept.shape)
        req.scales[i].copy_(kept)
        assert not _by_copies(lambda: _attend(req, q, decode=True))
        out = _attend(req, q, decode=True)
        assert torch.equal(out, whole)
        req.scales[i] = kept
