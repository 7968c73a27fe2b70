"""paged_attention_int4 where q has another type than the rows that were appended: right while the scales are in q's range."""
import pytest
import torch

from tests._int4 import Requests4
from tests.test_int4_attention import _check

BF16, FP16 = torch.bfloat16, torch.float16


@pytest.mark.gpu
@pytest.mark.parametrize("news", [[1, 1], [3, 2], [60, 40]])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("appended,q", [(BF16, FP16), (FP16, BF16)])
def test_rows_of_the_other_type(appended, q, D, news):
    req = Requests4(news, [300, 90], 8, 2, D, 16, appended)
    sizes = torch.cat([s.double().abs().nan_to_num(0.0).flatten() for s in req.scales])
    sizes = sizes[sizes > 0]
    assert float(sizes.min()) >= 2.0 ** -20 and float(sizes.max()) <= 7936  # what FP16 takes without a rounding
    _check(req, req.q.to(q))
