"""Arguments that the attention entry points refuse on the host, before any device."""
import ctypes as C

import pytest

from tokenvector.inference_amd import _lib
from tokenvector.inference_amd import attention as A
from tokenvector.inference_amd import device as D


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


class _Memory(D.DeviceBuffer):
    """A buffer's Python side alone."""

    def __init__(self):
        self.ptr, self.nbytes, self.ctx = 16, 64, None

    def close(self):
        self.ptr = 0


class _Cache(A.KVCache):
    """A cache's Python side alone."""

    def __init__(self, *kept):
        self.handle, self.head_dim, self._kept = 16, 64, kept

    def close(self):
        self.handle = 0


class _Ctx:
    handle = 0


def _calls(cache, buffer):
    rows = A.Rows(buffer, 64, 64)
    yield A.RopeAppend(_Ctx, A.BF16, 1, 1, 1, 64, rows, rows, rows, cache=cache, slots=buffer)
    yield A.AttentionPaged(_Ctx, A.BF16, 1, 1, cache, 1, rows, rows, buffer, 1, buffer)


@pytest.mark.parametrize("which", [0, 1], ids=["append", "attention"])
@pytest.mark.parametrize("closed", ["cache", "pool", "buffer"])
def test_call_of_a_closed_cache_or_buffer(which, closed):
    """The address or handle that the call holds is no longer anybody's."""
    pool, buffer = _Memory(), _Memory()
    cache = _Cache(pool, None)
    call, launched = list(_calls(cache, buffer))[which], []
    call._fn = lambda *args: launched.append(args) and 0
    call()
    assert len(launched) == 1
    {"cache": cache, "pool": pool, "buffer": buffer}[closed].close()
    with pytest.raises(ValueError, match="closed"):
        call()
    assert len(launched) == 1


def test_call_made_of_a_closed_cache():
    """Its handle is 0, which to the append means no cache."""
    cache, buffer = _Cache(), _Memory()
    cache.close()
    for call in _calls(cache, buffer):
        call._fn = lambda *args: pytest.fail("launched")
        with pytest.raises(ValueError, match="closed"):
            call()


def test_prompt_keys_of_their_own_come_with_their_number():
    """Taken for the number of query tokens, it cut longer keys off unsaid."""
    rows, cu = A.Rows(16, 64, 64), _Memory()
    with pytest.raises(ValueError, match="tokens_k"):
        A.AttentionPrompt(_Ctx, A.BF16, 1, 1, 1, 64, 1, rows, rows, rows, rows, cu, cu)
    A.AttentionPrompt(_Ctx, A.BF16, 1, 1, 1, 64, 1, rows, rows, rows, rows, cu, cu, 5)
