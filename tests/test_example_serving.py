"""The serving example end to end: training lowers the loss, and chunked, paged serving gives the
logits of the model run over each whole text."""
import pytest


@pytest.mark.gpu
def test_trains_and_serves():
    from examples.serve_paged import main
    first, final, worst = main(["--steps", "20", "--requests", "5", "--new", "10"])
    assert final < 0.9 * first
    # BF16 rows on both sides: each of the two layers' attention is within about 2^-8 of the other
    # path's, in logits of order 1
    assert worst < 0.1
