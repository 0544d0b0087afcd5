"""Newton-Schulz orthogonalization and the Muon step on the GPU against the definition in 64 bits.

Tolerances, relative to the result's 2-norm.  float32: what the same products in float32 are off, twice, and 5 steps of 2^-22 (X is
held in 22 bits).  bfloat16: a step rounds four operands to 11 bits (root mean square 2^-12 / sqrt 3), an error that |b| + |c| = 6.8
multiplies; later steps carry it on with a slope of about 1: sqrt(5 steps * 4) * 6.8 * 1.4e-4 = 4.3e-3, and the result's own rounding
2^-9 / sqrt 3 = 1.1e-3: 5e-3 in all.  That is an average over many directions: matrices with a side of at most 128 take the products
of float32."""
import pytest
import torch

from oracle import orthogonalize as O
from piper_amd import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16_TOL = 5e-3


def matrices(shape, seed, kind="spiked", dtype=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=gen)
    if kind == "spiked":          # a few strong directions over noise
        x = x + 0.3 * torch.randn((*shape[:-1], 4), generator=gen) @ torch.randn((*shape[:-2], 4, shape[-1]), generator=gen)
    elif kind == "rows":          # rows of very different size
        x = x * torch.exp(2 * torch.randn((*shape[:-1], 1), generator=gen))
    elif kind == "lowrank":
        x = torch.randn((*shape[:-1], 3), generator=gen) @ torch.randn((*shape[:-2], 3, shape[-1]), generator=gen)
    return (x * 1e-3).to(dtype)


def off(a, b):
    a, b = a.detach().double().cpu(), b.double()
    return ((a - b).norm() / b.norm().clamp_min(1e-300)).item()


def f32_tolerance(x):
    exact = O.orthogonalize(x.double())
    return 2 * off(O.orthogonalize(x.float()), exact) + 5 * 2.0 ** -22, exact


SHAPES = [(1, 1, 1), (1, 1, 7), (3, 5, 1), (2, 128, 128), (1, 129, 127), (4, 100, 363), (1, 363, 100), (2, 256, 512), (1, 257, 255), (1, 640, 384),
          (1, 384, 1000), (2, 3, 1100)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("kind", ["spiked", "rows", "lowrank"])
def test_float32_is_as_exact_as_float32_products(shape, kind):
    x = matrices(shape, 1, kind)
    tol, exact = f32_tolerance(x)
    got = ops.orthogonalize(x.to(DEV))
    assert got.dtype == torch.float32 and got.shape == x.shape and got.is_contiguous()
    for e in range(shape[0]):
        assert off(got[e], exact[e]) <= max(tol, 2 * f32_tolerance(x[e])[0])


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("kind", ["spiked", "rows", "lowrank"])
def test_bfloat16(shape, kind):
    x = matrices(shape, 2, kind, torch.bfloat16)
    exact = O.orthogonalize(x.double())
    got = ops.orthogonalize(x.to(DEV))
    assert got.dtype == torch.bfloat16
    for e in range(shape[0]):
        assert off(got[e], exact[e]) <= BF16_TOL


@pytest.mark.parametrize("steps,coefficients", [(0, O.COEFFICIENTS), (1, O.COEFFICIENTS), (3, (2.0, -1.5, 0.5)), (8, (1.875, -1.25, 0.375))])
def test_steps_and_coefficients(steps, coefficients):
    x = matrices((2, 150, 260), 3)
    exact = O.orthogonalize(x.double(), steps, coefficients)
    tol = 2 * off(O.orthogonalize(x, steps, coefficients), exact) + max(1, steps) * 2.0 ** -22
    assert off(ops.orthogonalize(x.to(DEV), steps=steps, coefficients=coefficients), exact) <= tol


def test_strided_unaligned_and_stacked_inputs():
    x = matrices((3, 40, 72), 4)
    want = ops.orthogonalize(x.to(DEV))
    turned = x.transpose(1, 2).contiguous().to(DEV).transpose(1, 2)             # strided
    assert torch.equal(ops.orthogonalize(turned), want)
    room = torch.empty(x.numel() + 1, device=DEV)
    room[1:] = x.to(DEV).reshape(-1)
    assert torch.equal(ops.orthogonalize(room[1:].view(x.shape)), want)         # starts 4 bytes behind a boundary
    assert torch.equal(ops.orthogonalize(x.to(DEV).view(1, 3, 40, 72))[0], want)
    assert torch.equal(ops.orthogonalize(x[0].to(DEV)), want[0])
    for empty in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
        assert ops.orthogonalize(torch.empty(empty, device=DEV)).shape == empty


def test_zeros_tiny_and_huge_matrices_and_values_that_are_not_finite():
    x = matrices((6, 70, 50), 5)
    want = ops.orthogonalize(x.to(DEV))
    y = x.clone()
    y[0] = 0                        # stays zero
    y[1, 3, 7] = float("nan")       # NaN throughout, nobody else's
    y[2] *= 1e30                    # its squares leave fp32
    y[3] *= 1e-25                   # below eps: shorter than a unit matrix, but the definition's
    y[4, 0, 0] = float("inf")
    got = ops.orthogonalize(y.to(DEV))
    assert not got[0].any() and got[1].isnan().all() and got[4].isnan().all()
    assert torch.equal(got[5], want[5])
    tol, exact = f32_tolerance(x[2])
    assert off(got[2], exact) <= 2 * tol
    # X is held times 2^12 with a smallest step of 2^-24, rounded to half of that: 2^-37 an element, which grows at most as the elements do
    exact = O.orthogonalize(y[3].double())
    assert (got[3].cpu().double() - exact).norm() <= 3.4445 ** 5 * 2.0 ** -37 * (70 * 50) ** 0.5


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_groups_of_any_size_give_the_same_bits(dtype):
    """The workspace decides how many matrices a launch takes, nothing else."""
    x = matrices((5, 130, 70), 6, dtype=dtype).to(DEV)
    want = ops.orthogonalize(x)
    import ctypes as C
    one = [(C.c_int64 * 1)(v) for v in (1, 130, 70)]
    least = int(_lib.load().pk_orthogonalize_workspace_bytes(*one, 1, int(dtype == torch.float32)))      # (of one matrix)
    for bytes_ in (least, 2 * least + 100, 5 * least):
        ws, out = torch.empty(bytes_, dtype=torch.uint8, device=DEV), torch.empty_like(x)
        _lib.call("pk_orthogonalize", x.data_ptr(), _lib.dtype_code(dtype), out.data_ptr(), 5, 130, 70, 5, *O.COEFFICIENTS, 1e-7, ws.data_ptr(), bytes_,
                  _lib.current_stream())
        assert torch.equal(out, want)
    out = torch.zeros_like(x)
    with pytest.raises(RuntimeError, match="workspace"):
        _lib.call("pk_orthogonalize", x.data_ptr(), _lib.dtype_code(dtype), out.data_ptr(), 5, 130, 70, 5, *O.COEFFICIENTS, 1e-7, ws.data_ptr(), least - 1,
                  _lib.current_stream())
    assert not out.any()


# ------------------------------------------------------------------------------------------------ the step
def step_inputs(shapes, seed, grad_dtype, flat, own):
    ws = [matrices(s, seed + i) * 20 for i, s in enumerate(shapes)]
    ms = [matrices(s, seed + 20 + i) for i, s in enumerate(shapes)]
    gs = [matrices(s, seed + 40 + i, dtype=grad_dtype) if own(i) else None for i, s in enumerate(shapes)]
    fs = [matrices(s, seed + 60 + i) if flat(i) else None for i, s in enumerate(shapes)]
    return ws, ms, gs, fs


STEP_SHAPES = [(64, 200), (3, 96, 40), (129, 129), (2, 2, 30, 50), (1, 17), (300, 1)]


@pytest.mark.parametrize("grad_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("nesterov,adjust", [(True, "original"), (False, "match_rms_adamw")])
@pytest.mark.parametrize("sources", ["own", "flat", "both", "mixed"])
def test_step(grad_dtype, nesterov, adjust, sources):
    flat = {"own": lambda i: False, "flat": lambda i: True, "both": lambda i: True, "mixed": lambda i: i % 2 == 0}[sources]
    own = {"own": lambda i: True, "flat": lambda i: False, "both": lambda i: True, "mixed": lambda i: i % 3 == 0}[sources]
    ws, ms, gs, fs = step_inputs(STEP_SHAPES, 7, grad_dtype, flat, own)
    to = lambda ts: [None if t is None else t.to(DEV) for t in ts]  # noqa: E731
    w, m, g, f = to(ws), to(ms), to(gs), to(fs)
    shadows = [torch.empty(s, dtype=torch.bfloat16, device=DEV) if i != 1 else None for i, s in enumerate(STEP_SHAPES)]
    hyper = dict(lr=0.01, momentum=0.9, weight_decay=0.1, nesterov=nesterov, adjust_lr=adjust)
    ops.muon_fused(w, m, g, flat_grads=f, shadows=shadows, zero_grad=sources == "both", **hyper)
    for i, s in enumerate(STEP_SHAPES):
        grad = (0 if fs[i] is None else fs[i].double()) + (0 if gs[i] is None else gs[i].double()) + torch.zeros(s, dtype=torch.float64)
        want_w, want_m = O.muon_step(ws[i].double(), ms[i].double(), grad, **hyper)
        assert (m[i].cpu().double() - want_m).abs().max() <= 2.0 ** -22 * max(ms[i].abs().max(), grad.abs().max())
        # the weights: a rounding of themselves, and what the fp32 result of the update may be off
        plain_w, _ = O.muon_step(ws[i], ms[i], grad.float(), **hyper)
        step = hyper["lr"] * O.rate(*s[-2:], adjust)
        assert off(w[i], want_w) <= 2 * off(plain_w, want_w) + 2.0 ** -23 + step * 5 * 2.0 ** -22 * (min(s[-2:]) ** 0.5 / want_w.norm().item())
        if shadows[i] is not None:
            assert torch.equal(shadows[i], w[i].to(torch.bfloat16))
        if fs[i] is not None:
            assert (not f[i].any()) if sources == "both" else torch.equal(f[i].cpu(), fs[i])


def test_step_with_half_products():
    ws, ms, gs, fs = step_inputs(STEP_SHAPES, 8, torch.bfloat16, lambda i: False, lambda i: True)
    w, m = [t.to(DEV) for t in ws], [t.to(DEV) for t in ms]
    ops.muon_fused(w, m, [t.to(DEV) for t in gs], lr=0.01, half_products=True)
    for i, s in enumerate(STEP_SHAPES):
        want_w, _ = O.muon_step(ws[i].double(), ms[i].double(), gs[i].double(), lr=0.01, momentum=0.95, weight_decay=0.0)
        assert off(w[i].cpu().double() - ws[i].double(), want_w - ws[i].double()) <= BF16_TOL


# ------------------------------------------------------------------------------------------------ many units, long sums, mixed sizes
# (definitions in 64 bits on the GPU: the library's products of doubles)
def off_each(a, b):
    d = (a.double() - b).flatten(1).norm(dim=1) / b.flatten(1).norm(dim=1).clamp_min(1e-300)
    return d


@pytest.mark.parametrize("shape", [(176, 300, 600), (176, 700, 290), (40, 1100, 520), (260, 257, 385), (102, 800, 900), (16, 700, 1500), (128, 700, 800)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_enough_matrices_for_wide_tiles(shape, dtype):
    """Sides whose last wide tile is half a tile or a few rows."""
    x = torch.cat([matrices((shape[0] // 4, *shape[1:]), 11 + i, kind, dtype).to(DEV) for i, kind in enumerate(["spiked", "rows", "lowrank", "spiked"])])
    exact = O.orthogonalize(x.double())
    got = ops.orthogonalize(x)
    if dtype == torch.float32:
        assert (off_each(got, exact) <= 2 * off_each(O.orthogonalize(x), exact) + 5 * 2.0 ** -22).all()
    else:
        assert (off_each(got, exact) <= BF16_TOL).all()
    assert torch.equal(ops.orthogonalize(x), got)


@pytest.mark.parametrize("shape", [(1, 100, 1900), (1, 200, 1500), (1, 2100, 260), (2, 128, 4000), (1, 1, 5000), (1, 513, 2048)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_few_matrices_of_long_rows(shape, dtype):
    """X X^T in shares of k, whose numbers do not divide k."""
    x = matrices(shape, 12, "spiked", dtype).to(DEV)
    exact = O.orthogonalize(x.double())
    got = ops.orthogonalize(x)
    if dtype == torch.float32:
        assert (off_each(got, exact) <= 2 * off_each(O.orthogonalize(x), exact) + 5 * 2.0 ** -22).all()
    else:
        assert (off_each(got, exact) <= BF16_TOL).all()


@pytest.mark.parametrize("half", [False, True])
def test_step_of_many_sizes(half):
    """Small and large matrices, tall and wide ones, single and stacked, in one call: their tiles share launches."""
    shapes = [(24, 500, 640)] + [(300 + 8 * i, 900 - 8 * i) for i in range(24)] + [(1100, 512)] * 6 + [(5, 100, 70), (64, 1000), (1, 1), (700, 2), (1024, 1024)]
    w, m, g = ([matrices(s, k + i).to(DEV) * f for i, s in enumerate(shapes)] for k, f in ((20, 20), (60, 1), (100, 1)))
    start = [(a.double(), b.double(), c.double()) for a, b, c in zip(w, m, g)]
    hyper = dict(lr=0.05, momentum=0.9, weight_decay=0.0)
    plain = [O.muon_step(a.clone(), b.clone(), c, **hyper)[0] for a, b, c in zip(w, m, g)]
    ops.muon_fused(w, m, g, half_products=half, **hyper)
    for (a, b, c), p, x in zip(start, plain, w):
        want = O.muon_step(a, b, c, **hyper)[0]
        size = lambda t: t.double().norm().item()  # noqa: E731
        update = size(want - a)
        if half and min(x.shape[-2:]) > 128:      # and a rounding of the weights
            assert size(x.double() - want) <= BF16_TOL * update + 2.0 ** -23 * size(want)
        else:
            assert size(x.double() - want) <= 2 * size(p.double() - want) + 5 * 2.0 ** -22 * update + 2.0 ** -23 * size(want)


@pytest.mark.parametrize("shape,dtype", [((3, 200, 1500), torch.bfloat16), ((1, 100, 1900), torch.float32), ((20, 300, 600), torch.bfloat16)])
def test_two_at_once_and_a_captured_one(shape, dtype):
    xs = [matrices(shape, 30 + i, dtype=dtype).to(DEV) for i in range(3)]
    want = [ops.orthogonalize(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    for x, s in zip(xs, streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(ops.orthogonalize(x))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    fixed = torch.zeros_like(xs[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.orthogonalize(fixed)
    for x, w in zip(xs, want):
        fixed.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, w)
        ops.orthogonalize(x.float())


def test_more_elements_than_32_bits_count():
    """2.2e9 of them, in several groups: matrices at either end as by themselves."""
    x = torch.zeros(2800, 1024, 768, dtype=torch.bfloat16, device=DEV)
    ends = matrices((4, 1024, 768), 40, dtype=torch.bfloat16).to(DEV)
    x[:2], x[-2:] = ends[:2], ends[2:]
    got = ops.orthogonalize(x)
    exact = O.orthogonalize(ends.double())
    assert (off_each(torch.cat([got[:2], got[-2:]]), exact) <= BF16_TOL).all()
    assert not got[2:-2].any()
