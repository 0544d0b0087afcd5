"""Which products the orthogonalization takes: bf16 results are roundings of exact ones, single products are the caller's choice.

Tolerances, relative to the result's 2-norm.  A bf16 result fl(y) of an fp32 one y that is off the exact x: |fl(y) - x| <= |fl(y) - y| +
|y - x| <= |fl(x) - y| + |y - x| <= |fl(x) - x| + 2 |y - x|, since fl rounds to nearest: what rounding the exact result costs, and twice
what fp32 results may be off (twice the error of the same products in float32, and 5 steps of 2^-22).  Single products:
5e-3 where errors average out (the head of test_gpu_orthogonalize.py).  Where they do not, every direction is off as one alone is.  With
eps = 2^-12, half a step of 11 bits, x' = B x and B = a + b A + c A^2 a step's roundings are, of x' itself,
  (3 |b + 2 c A| A  +  |b A + c A^2|  +  |B|) eps / |B|:   x twice in A = x^2 and A's own;  x beside b A + c A^2 (a x is exact);  B's,
and what was there before grows by |x p'(x) / p(x)|.  Added up along five steps from any 0.02 <= x <= 1, and the result's own eps: 0.0356 at most."""
import ctypes as C
import math

import pytest
import torch

from oracle import orthogonalize as O
from piper_amd import _lib, ops
from test_gpu_orthogonalize import BF16_TOL, DEV, matrices, off_each

pytestmark = pytest.mark.gpu
ONE_DIRECTION = 0.0356


def worst_direction():
    a, b, c = O.COEFFICIENTS
    eps = 2.0 ** -12
    x = torch.exp(torch.linspace(math.log(0.02), 0.0, 200001, dtype=torch.float64))
    off = torch.zeros_like(x)
    for _ in range(5):
        A = x * x
        B = a + b * A + c * A * A
        off = off * ((a + 3 * b * A + 5 * c * A * A) / B).abs() + (3 * (b + 2 * c * A).abs() * A + (b * A + c * A * A).abs() + B.abs()) * eps / B.abs()
        x = B * x
    return (off + eps).max().item()


def test_the_bound_of_one_direction():
    assert 0.0355 < worst_direction() < ONE_DIRECTION


def few_rows(rows, cols, n, seed, dtype):
    gen = torch.Generator().manual_seed(seed)
    x = torch.zeros(rows, cols)
    x[torch.randperm(rows, generator=gen)[:n]] = torch.randn(n, cols, generator=gen)
    return x.to(dtype)


def inputs(dtype):
    for shape in [(1, 1, 7), (2, 128, 128), (1, 129, 127), (4, 300, 363), (1, 363, 1000), (24, 1000, 363), (176, 300, 600), (16, 700, 1500), (1, 640, 384)]:
        for kind in ("spiked", "rows", "lowrank"):
            yield f"{shape} {kind}", matrices(shape, 3, kind, dtype)
    for n in (1, 2, 4, 8):
        for rows, cols in ((256, 1100), (768, 2048), (1100, 256)):
            x = torch.stack([few_rows(min(rows, cols), max(rows, cols), n, 10 * n + s, dtype) for s in range(3)])
            yield f"{n} rows of {rows} x {cols}", x if rows < cols else x.mT.contiguous()
    for n in (129, 200, 512):
        yield f"identity {n}", 3 * torch.eye(n, dtype=dtype)[None]


def test_bfloat16_results_are_roundings_of_exact_ones():
    for name, x in inputs(torch.bfloat16):
        x = x.to(DEV)
        exact = O.orthogonalize(x.double())
        got = ops.orthogonalize(x)
        f32 = 2 * off_each(O.orthogonalize(x.float()), exact) + 5 * 2.0 ** -22
        assert got.dtype == torch.bfloat16 and (off_each(got, exact) <= off_each(exact.bfloat16(), exact) + 2 * f32).all(), name
        assert torch.equal(got, ops.orthogonalize(x.float()).bfloat16()), name       # one rounding of the same sums


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_half_products(dtype):
    for name, x in inputs(dtype):
        x = x.to(DEV)
        exact = O.orthogonalize(x.double())
        got = ops.orthogonalize(x, half_products=True)
        assert got.dtype == dtype and got.shape == x.shape
        assert (off_each(got, exact) <= (BF16_TOL if "(" in name else ONE_DIRECTION)).all(), name
        if min(x.shape[-2:]) <= 128:
            assert torch.equal(got, ops.orthogonalize(x)), name


@pytest.mark.parametrize("shape", [(1, 200, 1500), (1, 2100, 260), (1, 513, 2048), (40, 1100, 520), (260, 257, 385), (102, 800, 900), (128, 700, 800)])
def test_half_products_in_shares_and_wide_tiles(shape):
    x = matrices(shape, 12, "spiked", torch.bfloat16).to(DEV)
    got = ops.orthogonalize(x, half_products=True)
    assert (off_each(got, O.orthogonalize(x.double())) <= BF16_TOL).all()
    assert torch.equal(ops.orthogonalize(x, half_products=True), got)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("half", [False, True])
def test_groups_of_any_size_give_the_same_bits(dtype, half):
    """The workspace decides how many matrices a launch takes, nothing else."""
    x = matrices((5, 270, 140), 6, dtype=dtype).to(DEV)
    want = ops.orthogonalize(x, half_products=half)
    least = int(_lib.load().pk_orthogonalize_workspace_bytes(*[(C.c_int64 * 1)(v) for v in (1, 270, 140)], 1, int(not half)))
    for bytes_ in (least, 2 * least + 100, 5 * least):
        ws, out = torch.empty(bytes_, dtype=torch.uint8, device=DEV), torch.empty_like(x)
        _lib.call("pk_orthogonalize_half" if half else "pk_orthogonalize", x.data_ptr(), _lib.dtype_code(dtype), out.data_ptr(), 5, 270, 140, 5,
                  *O.COEFFICIENTS, 1e-7, ws.data_ptr(), bytes_, _lib.current_stream())
        assert torch.equal(out, want)


def test_half_products_captured():
    xs = [matrices((20, 300, 600), 30 + i, dtype=torch.bfloat16).to(DEV) for i in range(3)]
    want = [ops.orthogonalize(x, half_products=True) for x in xs]
    fixed = torch.zeros_like(xs[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.orthogonalize(fixed, half_products=True)
    for x, w in zip(xs, want):
        fixed.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, w)
        ops.orthogonalize(x.float())


def test_singular_values_up_to_the_range_are_right_and_past_it_refused():
    one = torch.ones(1, 1, device=DEV)
    assert ops.orthogonalize(one, steps=1, coefficients=(14.0, 0.0, 0.0)).item() == 14.0
    for coefficients in ((14.0, 0.0, 0.0), (-9.0, -3.0, -2.0)):
        x = torch.cat([few_rows(200, 330, 1, s, torch.float32)[None] for s in range(2)] + [matrices((2, 200, 330), 7)]).to(DEV)
        exact = O.orthogonalize(x.double(), 1, coefficients)
        for half, tol in ((False, 2 * off_each(O.orthogonalize(x, 1, coefficients), exact) + 2.0 ** -22), (True, BF16_TOL)):
            assert (off_each(ops.orthogonalize(x, steps=1, coefficients=coefficients, half_products=half), exact) <= tol).all()
    with pytest.raises(ValueError, match="singular values to 20"):
        ops.orthogonalize(one, steps=1, coefficients=(20.0, 0.0, 0.0))
