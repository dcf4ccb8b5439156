"""CPU tests of the sizes that the serving entries of the C ABI take: what the kernels' 32-bit counts and a launch's threads do
not hold is refused before anything runs (no pointer here is read)."""

import ctypes

import pytest

from fa2 import _lib
from test_step import P, c_cache, c_seq, c_turn, needs_lib, strides

MOST_WGS = ((1 << 32) - 1) // 256  # workgroups of 256 threads: a launch holds fewer than 2^32 threads


def rotary_qk(n, B=1, h_q=1, D=16):
    r = strides(0 if B == 1 else n * h_q * D, D, h_q * D)
    turn = c_turn(rotation=_lib.Rotation(P, D // 2, 0, 1.0))
    return _lib.lib().fa2_rotary_qk(P, None, P, None, r, strides(0, 0, 0), r, strides(0, 0, 0), P, 8, strides(0, 0, 0),
                                    ctypes.byref(turn), B, h_q, 0, n, D, 1, None)


@needs_lib
@pytest.mark.parametrize("n,B,h_q,D", [(2 ** 31 - 1, 1, 1, 16), (2 ** 31 - 14, 1, 1, 16), (2 ** 31 - 15, 2, 1, 16),
                                       (16 * MOST_WGS + 1, 1, 1, 16), (8 * MOST_WGS, 3, 1, 32), (16, 2 ** 31 - 1, 4, 64)])
def test_rotary_qk_of_more_tokens_than_a_launch_holds(n, B, h_q, D):
    assert rotary_qk(n, B, h_q, D) == -1 and "too large" in _lib.last_error()


@needs_lib
def test_other_launches():
    r, s = strides(0, 64, 2048), strides(2048, 64)
    rot = ctypes.byref(_lib.Rotation(P, 32, 0, 1.0))
    assert _lib.lib().fa2_rotary(P, P, r, r, P, 4, strides(0, 1), rot, 1, 32, MOST_WGS + 1, 64, 1, None) == -1
    assert "too large" in _lib.last_error()
    many = 16 * MOST_WGS + 1
    cache, seq, turn = ctypes.byref(c_cache()), ctypes.byref(c_seq(n_tokens=many)), ctypes.byref(c_turn())
    calls = [lambda: _lib.lib().fa2_cache_write(cache, seq, P, P, s, s, None, None, s, s, 0, rot, 1, None),
             lambda: _lib.lib().fa2_cache_read(cache, seq, P, P, s, s, 1, None),
             lambda: _lib.lib().fa2_cache_write_turned(cache, seq, P, P, s, s, None, None, s, s, 0, None, 0, strides(0, 0), turn, 1, None),
             lambda: _lib.lib().fa2_attn_paged_shared(P, P, s, s, cache, seq, P, 4, 1, 1, 0.1, None, P, 1 << 62, None),
             lambda: _lib.lib().fa2_attn_packed(P, P, P, P, s, s, s, s, P, P, 2 ** 31 - 2049, 2 ** 30, 3, 2, 2, 64, 1, 1, 0.1, None, None),
             lambda: _lib.lib().fa2_attn_packed_window(P, P, P, P, s, s, s, s, P, P, 2 ** 31 - 2049, 2 ** 30, 3, 2, 2, 64, 1, 9, 0, 0.1,
                                                       None, None)]
    for call in calls:
        assert call() == -1 and "too large" in _lib.last_error()


@needs_lib
@pytest.mark.parametrize("n", [2 ** 31 - 1, 2 ** 31 - 64])
def test_more_sequences_than_are_counted_in_32_bits(n):
    """The kernels go through the sequences 64 at a time, up to 64 past the last."""
    s = strides(256, 64)
    seq = ctypes.byref(c_seq(n_seq=n))
    calls = [lambda: _lib.lib().fa2_attn_packed(P, P, P, P, s, s, s, s, P, P, n, 3, 3, 4, 4, 64, 1, 1, 0.1, None, None),
             lambda: _lib.lib().fa2_attn_packed_window(P, P, P, P, s, s, s, s, P, P, n, 3, 3, 4, 4, 64, 1, 9, 0, 0.1, None, None),
             lambda: _lib.lib().fa2_attn_paged(P, P, s, s, ctypes.byref(c_cache()), seq, 4, 1, 1, 0.1, None, P, 1 << 62, None),
             lambda: _lib.lib().fa2_attn_paged_window(P, P, s, s, ctypes.byref(c_cache()), seq, 4, 1, 9, 0, 0.1, None, P, 1 << 62, None),
             lambda: _lib.lib().fa2_attn_paged_shared(P, P, s, s, ctypes.byref(c_cache()), seq, P, 4, 1, 1, 0.1, None, P, 1 << 62, None)]
    for call in calls:
        assert call() == -1 and "n_seq" in _lib.last_error()


@needs_lib
@pytest.mark.parametrize("n", [2 ** 31 - 1, 2 ** 31 - 256, 2 ** 20 + 1])
def test_more_sequences_than_a_step_has(n):
    """Every workgroup of the pages' kernels goes through all sequences, in 32 bits."""
    assert _lib.lib().fa2_pages_extend(P, 8, P, P, None, 0, n, 0, 16, P, P, P, P, P, P, 4, None) == -1
    assert "2^20" in _lib.last_error()
    assert _lib.lib().fa2_pages_release(P, 8, P, P, None, 0, n, 0, P, P, P, None) == -1
    assert "2^20" in _lib.last_error()
