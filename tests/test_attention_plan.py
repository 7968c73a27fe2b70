"""The shares that chunks' tiles are cut into fit the workspace of a call, whatever its sizes. Without a GPU."""
import ctypes
import random

import pytest

from flash_attn_prologue_b200 import _lib


def _bytes(tokens, batch, ragged, kv_heads, group, dim, pages, page, window, sms, int4):
    cache = (0,) * 8 + (1, page, 0, 0, pages, 0, int(ragged), batch)
    args = _lib.ATTENTION_ARGS.pack(*(0,) * 9, *cache, 0, 0, tokens, kv_heads * group, kv_heads, dim, 0, window, 1.0)
    needed, available = ctypes.c_size_t(0), ctypes.c_size_t(0)
    assert _lib.load().flash_prologue_selftest_attention_plan(args, int(int4), sms, ctypes.byref(needed),
                                                              ctypes.byref(available)) == 0
    return needed.value, available.value


@pytest.mark.parametrize("int4", [False, True])
@pytest.mark.parametrize("dim", [64, 128])
def test_shares_fit_the_workspace(dim, int4):
    rng = random.Random(dim + int4)
    shared = fullest = 0
    for _ in range(40000):
        group = rng.choice([1, 2, 3, 4, 5, 7, 8, 16, 31, 64, 128])
        kv_heads = rng.randint(1, max(1, min(64, 512 // group)))
        batch = int(2 ** rng.uniform(0, 9))
        tokens = int(2 ** rng.uniform(0, 15))
        page = 2 ** rng.randint(3, 10)
        pages = int(2 ** rng.uniform(0, 20)) // page + 1
        window = rng.choice([0, 0, int(2 ** rng.uniform(0, 16))])
        sms = rng.choice([148, 148, 132, 20, 1])
        needed, available = _bytes(tokens, batch, rng.random() < 0.7, kv_heads, group, dim, pages, page, window, sms, int4)
        assert needed <= available, (tokens, batch, kv_heads, group, pages, page, window, sms)
        shared += needed > 0
        fullest = max(fullest, needed / available)
    assert shared > 1000 and fullest > 0.9  # shares there are, and they come near the end


def test_refusals():
    size = ctypes.c_size_t(0)
    call = _lib.load().flash_prologue_selftest_attention_plan
    assert call(None, 0, 148, ctypes.byref(size), ctypes.byref(size)) == 1
    assert call(bytes(_lib.ATTENTION_ARGS.size), 0, 148, ctypes.byref(size), ctypes.byref(size)) == 1
