"""Argument checks of pk_fp8_quantize_rows_of, every call refused before a launch."""
import ctypes

from piper_amd import _lib

ARG, SHAPE, ALIGN = -1, -2, -3


def test_quantize_rows_of():
    buf = ctypes.create_string_buffer(1 << 12)
    p = (ctypes.addressof(buf) + 15) // 16 * 16
    rows = _lib.load().pk_fp8_quantize_rows_of
    assert rows(p, 1, -1, None, 1, p, p, 1, 128, None) == ARG
    assert rows(p, 1, 3, None, 1, p, p, 4, 128, None) == ARG      # more rows than x has
    assert rows(p, 7, 4, p, 1, p, p, 1, 128, None) == ARG
    assert rows(p, 1, 4, p, 0, p, p, 1, 128, None) == ARG
    assert rows(None, 1, 4, p, 1, p, p, 1, 128, None) == ARG
    assert rows(p, 1, 4, p, 1, p + 4, p, 1, 128, None) == ALIGN
    assert rows(p, 1, 4, p, 2 ** 31, p, p, 1, 128, None) == SHAPE
    assert rows(None, 1, 0, None, 1, None, None, 0, 128, None) == 0
