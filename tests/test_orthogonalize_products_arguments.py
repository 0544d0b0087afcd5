"""What the orthogonalization with single products refuses, on the CPU."""
import ctypes as C

from oracle import orthogonalize as O
from piper_amd import _lib


def refused(rc, word):
    assert rc < 0 and word in _lib.status_string(rc)


def test_half_products_refuse_what_the_others_do():
    buf = C.create_string_buffer(1 << 16)
    p = (C.addressof(buf) + 255) // 256 * 256

    def run(x=p, dtype=_lib.PK_BF16, out=p, count=1, rows=4, cols=4, steps=5, eps=1e-7, ws=p, bytes_=1 << 15):
        return _lib.load().pk_orthogonalize_half(x, dtype, out, count, rows, cols, steps, *O.COEFFICIENTS, eps, ws, bytes_, None)

    for bad in (dict(x=None), dict(out=None), dict(dtype=7), dict(count=-1), dict(steps=-1), dict(steps=101), dict(eps=0.0), dict(eps=float("nan"))):
        refused(run(**bad), "argument")
    refused(run(cols=32769), "shape")
    for bad in (dict(ws=None), dict(ws=p + 8), dict(bytes_=1000)):
        refused(run(**bad), "workspace")
    assert run(count=0, x=None, ws=None, bytes_=0) == 0


def test_workspace_of_either_kind():
    ws = _lib.load().pk_orthogonalize_workspace_bytes
    one = [(C.c_int64 * 1)(v) for v in (1, 270, 140)]
    # A and B in two planes, or in one
    assert ws(*one, 1, 1) - ws(*one, 1, 0) == 2 * 256 * 256 * 2
