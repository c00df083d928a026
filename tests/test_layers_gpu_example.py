"""GPU: the feed-forward example (explicit Q of a batched QR, rms_norm, linear, quantize_rows, and training).

Bounds on the relative error against float64.  16 bits: the inputs, the norm's output, the hidden layer and
the result are each rounded to bf16 (2^-8 of a value at most, 2^-9 in the mean), four roundings that add up as
independent errors at most by 2: 2^-7.  8 bits: the two products' operands are rounded to e4m3 (2^-4 of a value at
most, about 2.7e-2 in the mean square), four of them, in a sum beside the stream itself: below 2 * 2.7e-2.
"""
import sys
from pathlib import Path

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _give_memory_back():
    """Leaves no cached blocks behind: with none, what the next module allocates comes from the device again."""
    yield
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


@pytest.mark.parametrize("width,hidden,tokens", [(512, 2048, 300), (64, 200, 17)])
def test_feed_forward_example(width, hidden, tokens):
    sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))
    import rotated_feed_forward as ex
    eight, single, sixteen, losses = ex.main(width, hidden, tokens, report=lambda s: None)
    assert sixteen < 2.0 ** -7
    assert eight < 5.4e-2 and single < 5.4e-2
    assert losses[-1] < losses[0]
