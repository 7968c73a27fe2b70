"""The serving example with its cache in 4 bits runs to its end."""
import math

import pytest


@pytest.mark.gpu
def test_serves_from_a_cache_in_4_bits():
    from examples.serve_paged import main
    _, _, worst = main(["--steps", "5", "--requests", "4", "--new", "6", "--int4"])
    assert math.isfinite(worst)
