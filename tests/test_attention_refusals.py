"""Arguments that the attention entry points refuse on the host, before any device."""
import ctypes as C

import pytest

from tokenvector.inference_amd import _lib
from tokenvector.inference_amd import attention as A


def _rows():
    return C.byref(A._Rows(16, 64, 64))


@pytest.mark.parametrize("tokens_k", [(1 << 31) - 255, (1 << 31) - 1, 1 << 31, 1 << 62])
def test_prompt_keys_beyond_the_kernels_numbers(tokens_k):
    """Ends of keys are rounded up to tiles in 32 bits."""
    r = _rows()
    assert _lib.lib().tkv_hip_dev_attention_prompt(0, A.BF16, 1, tokens_k, 1, 1, 64, 1, r, r, r, r, A.BF16, 16,
                                                   16, 1.0, 1, 0) == _lib.BAD_ARG


@pytest.mark.parametrize("tokens,heads", [((1 << 62) + 1, 4), (1 << 62, 4), (1 << 31, 1), ((1 << 63) - 1, 2)])
def test_rope_tokens_whose_rows_pass_64_bits(tokens, heads):
    """tokens * heads wraps to 4 or 0 for the first two."""
    r = _rows()
    assert _lib.lib().tkv_hip_dev_rope_append(0, A.F32, tokens, heads, 0, 64, r, None, None, None, None, 0, 0, 0, r,
                                              None, A.F32, 0, None) == _lib.BAD_ARG
