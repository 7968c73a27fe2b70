"""plan_paged_step where the requests' new tokens are more than 32 bits can count."""
import pytest
import torch

import flash_attn_prologue_b200 as fap
from flash_attn_prologue_b200 import _lib


@pytest.mark.gpu
@pytest.mark.parametrize("B", [2, 33, 1100, 2100])
def test_counts_beyond_32_bits_stay_in_order(B):
    """Starts never fall and stay below 2^31, every row belongs to the first request, and the error word is set."""
    def dev(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    for news in ([2 ** 30] * B, [2 ** 31 - 1] * B, [2 ** 30 - 1] * (B - 1) + [2 ** 31 - 1], [5] + [2 ** 30] * (B - 1)):
        table, free = torch.full((B, 2), -1, dtype=torch.int32, device="cuda"), torch.arange(7, dtype=torch.int32, device="cuda")
        _lib.device_error()
        step = fap.plan_paged_step(table, dev([0] * B), dev(news), free, dev([7]), 8, 40)
        assert _lib.device_error() == 2
        starts = step.cu_seqlens.long()
        assert starts[0] == 0 and (starts[1:] >= starts[:-1]).all() and starts[1] == min(news[0], 2 ** 30)
        request = step.requests.tolist()
        assert request == ([0] * 40 if news[0] > 40 else [0] * 5 + [1] * 35)
        assert step.positions.tolist() == (list(range(40)) if news[0] > 40 else list(range(5)) + list(range(35)))
        # pages go to the requests in order, two each, while there are any
        assert table[:3].flatten().tolist()[:6] == [6, 5, 4, 3, 2, 1][:2 * B] if news[0] > 40 else table[0].tolist() == [6, -1]
