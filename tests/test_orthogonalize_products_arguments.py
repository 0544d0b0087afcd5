"""What the orthogonalization refuses of products and coefficients, on the CPU."""
import ctypes as C

import pytest
import torch

from oracle import orthogonalize as O
from piper_amd import _lib, ops
from piper_amd.optim import FusedMuon


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


# ------------------------------------------------------------------------------------------------ the range of singular values
def reached(steps, coefficients, n=20001):
    """The largest singular value that the polynomial makes of n in [0, 1], at any step."""
    a, b, c = (float(torch.tensor(v, dtype=torch.float32)) for v in coefficients)
    x = torch.linspace(0, 1, n, dtype=torch.float64)
    most = 1.0
    for _ in range(steps):
        x = a * x + b * x ** 3 + c * x ** 5
        most = max(most, x.abs().max().item())
    return most


GOOD = [(5, O.COEFFICIENTS), (100, O.COEFFICIENTS), (3, (2.0, -1.5, 0.5)), (8, (1.875, -1.25, 0.375)), (100, (1.5, -0.5, 0.0)), (0, (20.0, 0.0, 0.0)),
        (1, (14.0, 0.0, 0.0)), (2, (3.5, 0.0, 0.0)), (10, (1.0, 0.0, 0.0)), (5, (0.0, 0.0, 0.0)), (3, (-1.5, 0.5, 0.0)), (1, (60.0, -180.0, 128.0))]
BAD = [(1, (20.0, 0.0, 0.0)), (5, (3.0, 0.0, 0.0)), (2, (4.0, 0.0, 0.0)), (1, (0.0, 0.0, -16.0)), (1, (0.0, 16.0, 0.0)), (4, (3.4445, -4.775, 5.0)), (100, (1.1, 0.0, 0.0)),
       (1, (80.0, -160.0, 81.0)), (1, (float("nan"), 0.0, 0.0)), (1, (1.0, float("inf"), 0.0)), (1, (1.0, 0.0, float("-inf"))), (2, (1e30, 1e30, 1e30))]


def test_range_covers_what_the_polynomial_reaches():
    bound = _lib.load().pk_newton_schulz_range
    for steps, k in GOOD:
        assert reached(steps, k) <= bound(steps, *k) <= 15.0, (steps, k)
    for steps, k in BAD:
        assert bound(steps, *k) > 15.0, (steps, k)
    assert bound(5, *O.COEFFICIENTS) < 1.3
    gen = torch.Generator().manual_seed(0)
    taken = 0
    for _ in range(2000):
        k = (torch.randn(3, generator=gen) * torch.tensor([3.0, 6.0, 6.0])).tolist()
        steps = int(torch.randint(1, 8, (1,), generator=gen))
        if bound(steps, *k) <= 15.0:
            taken += 1
            assert reached(steps, k, 501) <= bound(steps, *k), (steps, k)
    assert 100 < taken < 1900


def test_coefficients_past_the_range_are_refused():
    buf = C.create_string_buffer(1 << 16)
    p = (C.addressof(buf) + 255) // 256 * 256
    lib, one = _lib.load(), [(C.c_int64 * 1)(4)] * 3
    ptrs = (C.c_void_p * 1)(p)
    x = torch.zeros(4, 4)
    for steps, k in BAD:
        for entry in (lib.pk_orthogonalize, lib.pk_orthogonalize_half):
            refused(entry(p, _lib.PK_F32, p, 1, 4, 4, steps, *k, 1e-7, p, 1 << 15, None), "argument")
        refused(lib.pk_muon_fused(ptrs, ptrs, None, None, None, *one, 1, _lib.PK_F32, 0.1, 0.9, 0.0, 1, 0, 0, 1, steps, *k, 1e-7, p, 1 << 15, None), "argument")
        with pytest.raises(ValueError, match="singular values"):
            ops.muon_fused([x], [x], [x], lr=0.1, steps=steps, coefficients=k)
        with pytest.raises(ValueError, match="singular values"):
            FusedMuon([torch.nn.Parameter(x)], ns_steps=steps, ns_coefficients=k)
    for steps, k in GOOD:
        FusedMuon([torch.nn.Parameter(x)], ns_steps=steps, ns_coefficients=k)
