"""The attention layer example: prefill in chunks and decode against one pass.

Both read the same projections and the same cache codes (quantized per token);
they differ by the rounding of the weights to bfloat16 (2^-8 at most, either
way) and by one int8 step of the output projection's activations where that
moves one (half of 1 / 127 of a row's maximum, about four of its standard
deviations).  Both are random over a row's 768 inputs, so their root mean squares
add: sqrt(2 (2^-8 / sqrt 3)^2 + (4 / 127 / sqrt 12)^2 2) = 0.013.
"""
import os
import sys

import pytest

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def test_attention_layer(hip):
    import attention_layer
    assert attention_layer.main() <= 0.013
