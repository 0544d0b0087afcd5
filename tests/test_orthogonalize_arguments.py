"""What the orthogonalization and the Muon step refuse, on the CPU: nothing of it reaches a launch."""
import ctypes as C

import pytest
import torch

from oracle import orthogonalize as O
from piper_amd import _lib, ops


def i64(*v):
    return (C.c_int64 * len(v))(*v)


def refused(rc, word):
    assert rc < 0 and word in _lib.status_string(rc)


@pytest.fixture()
def buffer():
    buf = C.create_string_buffer(1 << 16)
    return buf, (C.addressof(buf) + 255) // 256 * 256


def test_workspace_query():
    ws = _lib.load().pk_orthogonalize_workspace_bytes
    one = ws(i64(1), i64(100), i64(300), 1, 1)
    # X twice in two planes of fp16, A and B in two, padded to 128, and the partial sums of squares
    assert one == 4 * 2 * 128 * 384 + 4 * 2 * 128 * 128 + (4 * 8 + 255) // 256 * 256
    assert ws(i64(3), i64(300), i64(100), 1, 1) == 3 * one
    assert ws(i64(1), i64(100), i64(300), 1, 0) == one                      # a short side: the products of float32 in any case
    assert ws(i64(1), i64(200), i64(300), 1, 0) < ws(i64(1), i64(200), i64(300), 1, 1)
    largest = ws(i64(1), i64(16384), i64(16384), 1, 1)
    assert ws(i64(1, 5), i64(16384, 10), i64(16384, 10), 2, 1) == largest   # what the largest matrix takes
    assert ws(i64(100000), i64(128), i64(128), 1, 1) <= 2560 << 20          # groups
    assert ws(i64(0, 4), i64(8, 0), i64(8, 8), 2, 1) == 0 == ws(None, None, None, 0, 1)
    refused(ws(i64(1), i64(32769), i64(1), 1, 1), "shape")
    refused(ws(i64(-1), i64(1), i64(1), 1, 1), "argument")
    refused(ws(None, None, None, 1, 1), "argument")


def test_orthogonalize_refuses(buffer):
    _, p = buffer
    call = _lib.load().pk_orthogonalize

    def run(x=p, dtype=_lib.PK_F32, out=p, count=1, rows=4, cols=4, steps=5, eps=1e-7, ws=p, bytes_=1 << 15):
        return call(x, dtype, out, count, rows, cols, steps, *O.COEFFICIENTS, eps, ws, bytes_, None)

    refused(run(x=None), "argument")
    refused(run(out=None), "argument")
    refused(run(dtype=7), "argument")
    refused(run(count=-1), "argument")
    for steps in (-1, 101):
        refused(run(steps=steps), "argument")
    for eps in (0.0, -1.0, float("nan")):
        refused(run(eps=eps), "argument")
    refused(run(rows=32769), "shape")
    refused(run(ws=None), "workspace")
    refused(run(ws=p + 8), "workspace")
    refused(run(bytes_=1000), "workspace")
    for empty in (dict(count=0), dict(rows=0), dict(cols=0)):
        assert run(**empty, x=None, ws=None, bytes_=0) == 0


def test_step_refuses(buffer):
    _, p = buffer
    call = _lib.load().pk_muon_fused
    one, none = (C.c_void_p * 1)(p), (C.c_void_p * 1)(None)

    def run(w=one, m=one, count=1, rows=4, cols=4, n=1, dtype=_lib.PK_BF16, adjust=0, steps=5, eps=1e-7, ws=p, bytes_=1 << 15):
        return call(w, m, None, None, None, i64(count), i64(rows), i64(cols), n, dtype, 0.1, 0.9, 0.0, 1, adjust, 0, 1, steps, *O.COEFFICIENTS, eps, ws,
                    bytes_, None)

    refused(run(w=none), "argument")
    refused(run(m=none), "argument")
    refused(run(w=None), "argument")
    refused(run(dtype=3), "argument")
    refused(run(adjust=2), "argument")
    refused(run(n=-1), "argument")
    refused(run(rows=40000), "shape")
    refused(run(steps=101), "argument")
    refused(run(eps=0.0), "argument")
    refused(run(ws=None), "workspace")
    refused(run(bytes_=100), "workspace")
    assert run(n=0) == 0 and run(count=0, w=none, ws=None) == 0


def test_tensors_on_the_cpu_and_bad_arguments():
    x = torch.zeros(4, 4)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.orthogonalize(x)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.muon_fused([x], [x], [x], lr=0.1)
    with pytest.raises(ValueError, match="three coefficients"):
        ops.orthogonalize(x, coefficients=(1.0, 2.0))
    with pytest.raises(ValueError, match="one momentum"):
        ops.muon_fused([x], [], [x], lr=0.1)
    with pytest.raises(ValueError, match="adjust_lr"):
        ops.muon_fused([x], [x], [x], lr=0.1, adjust_lr="no")
    with pytest.raises(ValueError, match="hyper-parameters"):
        ops.muon_fused([x], [x], [x], lr=-0.1)
    ops.muon_fused([], [], [], lr=0.1)


def test_oracle_is_an_odd_polynomial_of_the_singular_values():
    x = torch.randn(5, 9, dtype=torch.float64, generator=torch.Generator().manual_seed(0))
    u, s, vh = torch.linalg.svd(x, full_matrices=False)
    s = s / s.norm()
    for _ in range(5):
        a, b, c = O.COEFFICIENTS
        s = a * s + b * s ** 3 + c * s ** 5
    assert torch.allclose(O.orthogonalize(x), u @ torch.diag(s) @ vh, atol=1e-12)
    assert torch.allclose(O.orthogonalize(x.mT), O.orthogonalize(x).mT, atol=1e-14)
    w, m = O.muon_step(x, x * 0, x, lr=0.1, momentum=0.9, weight_decay=0.5)
    assert torch.allclose(m, 0.1 * x) and torch.allclose(w, 0.95 * x - 0.1 * O.orthogonalize(x), atol=1e-12)
