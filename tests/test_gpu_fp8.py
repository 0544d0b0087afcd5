"""The experts in 8-bit blocks: quantisation bit for bit, products and gradients within the bounds that oracle/blocks.py derives for
sums and functions in fp32, and the operator where callers meet it (strides, streams, graphs, split backward, tracing)."""
import math

import pytest
import torch

from oracle import blocks as B
from piper_amd import _lib, ops
from piper_amd import functional as F_
from piper_amd.moe import AnnotatedMoE, BmmExperts, MoEArgs

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


def _same(got, want):
    """Equal values, NaN in the same places."""
    got, want = got.double().cpu(), want.double().cpu()
    return torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


def _exponents(s):
    return s.view(torch.uint8).cpu().to(torch.int64) - 127


def _awkward(shape, dtype, seed):
    """Normal values with rows of every magnitude, zeros, subnormals, values on the border of two scales."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g)
    flat = x.view(-1, shape[-1])
    for i, f in enumerate((1.0, 0.0, 1e-38, 1e-30, 1e30, 448.0, 1e-45, 3.0)):
        if i < flat.shape[0]:
            flat[i] *= f
    flat[-1, : shape[-1] // 2] = 1.75
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,width", [(1, 1), (9, 128), (3, 129), (17, 1000), (5, 2048), (40, 127), (300, 384)])
def test_rows_are_quantized_bit_for_bit(dev, rows, width, dtype):
    print(f"[case] quantize rows {rows} x {width} {dtype}", flush=True)
    x = _awkward((rows, width), dtype, rows)
    q, s = ops.quantize_rows_fp8(x.to(dev))
    want, k = B.rows(x)
    assert q.dtype == E4M3 and q.shape == want.shape and _same(q, want) and torch.equal(_exponents(s), k)


def test_rows_gathered_strided_unaligned_and_not_finite(dev):
    print("[case] quantize rows: map, strides, offsets, NaN", flush=True)
    x = _awkward((12, 264), torch.bfloat16, 3)
    x[4, 130], x[7, 0], x[8, 263] = math.inf, math.nan, -math.inf
    perm = torch.tensor([23, 0, 5, 5, 11, 22, 9], dtype=torch.int32)
    want, k = B.rows(x[(perm // 2).long()])
    q, s = ops.quantize_rows_fp8(x.to(dev), perm.to(dev), 2)
    assert _same(q, want) and torch.equal(_exponents(s), k)
    wide = torch.zeros(12, 300, dtype=torch.bfloat16)
    wide[:, 3:267] = x
    for view in (wide.to(dev)[:, 3:267], x.to(dev).t().contiguous().t(), torch.cat([torch.zeros(1, dtype=x.dtype), x.reshape(-1)]).to(dev)[1:].view(12, 264)):
        q, s = ops.quantize_rows_fp8(view)
        want, k = B.rows(x)
        assert _same(q, want) and torch.equal(_exponents(s), k)
    q, s = ops.quantize_rows_fp8(x[:0].to(dev))
    assert q.shape == (0, 384) and s.shape == (0, 3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("E,I,H", [(1, 128, 128), (2, 1, 1), (3, 130, 257), (2, 360, 1000), (1, 384, 256), (4, 127, 200)])
def test_weights_are_quantized_bit_for_bit_both_ways(dev, E, I, H, dtype):
    print(f"[case] quantize weights {E} x {I} x {H} {dtype}", flush=True)
    w1, w3, w2 = _awkward((E, I, H), dtype, 0), _awkward((E, I, H), dtype, 1), _awkward((E, H, I), dtype, 2)
    w1[-1, -1, -1] = math.nan
    got = F_.quantize_experts(w1.to(dev), w2.to(dev), w3.to(dev))
    for w, q, s, t in ((w1, got.q1, got.s1, got.t1), (w2, got.q2, got.s2, got.t2), (w3, got.q3, got.s3, got.t3)):
        want, k = B.weights(w)
        N, K = w.shape[1:]
        assert torch.equal(_exponents(s), k)
        assert q.shape == (E, N, want.shape[2]) and _same(q, want[:, :N])
        assert t.shape == (E, K, want.shape[1]) and _same(t, want[:, :, :K].transpose(1, 2))
    less = F_.quantize_experts(w1.to(dev), w2.to(dev), w3.to(dev), for_backward=False)
    assert less.t1 is None and _same(less.q2, got.q2)


# ------------------------------------------------------------------------------ products
def _inputs(E, H, I, counts, spare, seed, integers):
    g = torch.Generator().manual_seed(seed)
    A = sum(counts) + spare
    if integers:      # sums of these are exact in fp32 in any order, and every value is a code
        mk = lambda *shape, unit: (torch.randint(-4, 5, shape, generator=g) * unit).bfloat16()  # noqa: E731
        return (mk(E, I, H, unit=2.0 ** -7), mk(E, H, I, unit=2.0 ** -6), mk(E, I, H, unit=2.0 ** -7), mk(A, H, unit=0.5), mk(A, H, unit=1.0))
    mk = lambda *shape, unit: (torch.randn(shape, generator=g) * unit).bfloat16()  # noqa: E731
    return mk(E, I, H, unit=0.05), mk(E, H, I, unit=0.05), mk(E, I, H, unit=0.05), mk(A, H, unit=1.0), mk(A, H, unit=1.0)


def _within(name, got, value, err, deviation):
    got = got.detach().double().cpu()
    far = (got - value).abs()
    outside = int((far > err).sum())
    assert outside == 0, f"{name}: {outside} of {far.numel()} values are outside, the worst by {(far - err).max().item():.3g}"
    assert far.norm() <= deviation.norm(), f"{name}: off by {(far.norm() / value.norm()).item():.3g}, at most {(deviation.norm() / value.norm()).item():.3g}"


def _decoded(E, rows):
    """Whether a pass over so many rows multiplies decoded values."""
    return rows <= max(40 * E, 128)


SHAPES = [
    (2, 256, 128, [5, 0], 0, "one row tile, an empty expert"),
    (3, 128, 256, [1, 257, 0], 3, "a row, a row more than a tile, none; rows of nobody"),
    (4, 130, 70, [17, 33, 1, 16], 0, "odd widths below a block"),
    (2, 1000, 360, [40, 61], 37, "widths that are no multiple of a block"),
    (1, 8, 8, [3], 0, "tiny"),
    (3, 384, 512, [255, 256, 129], 1, "around a tile's rows"),
    (2, 257, 300, [30, 12], 0, "odd widths of two and three blocks"),
    (70, 128, 128, [i % 4 for i in range(70)], 0, "more experts than lanes"),
    (2, 257, 300, [140, 90], 3, "odd widths and many rows"),
    (200, 200, 136, [i % 31 for i in range(200)], 5, "enough experts for wide units, decoded values"),
    (200, 199, 139, [i % 31 for i in range(200)], 0, "the same with odd widths"),
    (200, 200, 136, [i % 87 for i in range(200)], 9, "the same with more rows"),
    (200, 199, 139, [i % 87 for i in range(200)], 0, "the same with odd widths and more rows"),
    (4, 256, 512, [200, 33, 0, 64], 7, "weight gradients from transposed copies if that pays"),
]


@pytest.mark.parametrize("integers", [True, False])
@pytest.mark.parametrize("E,H,I,counts,spare,what", SHAPES)
def test_forward_and_backward_are_within_their_bounds(dev, E, H, I, counts, spare, what, integers):
    print(f"[case] fp8 experts {what} integers={integers}", flush=True)
    w1, w2, w3, x, d_y = _inputs(E, H, I, counts, spare, E + H, integers)
    want = B.experts_between(w1, w2, w3, x, counts, d_y, decoded=_decoded(E, sum(counts) + spare))
    leaves = [t.to(dev).requires_grad_(True) for t in (w1, w2, w3, x)]
    n = torch.tensor(counts, dtype=torch.int32, device=dev)
    y = F_.bmm_experts_fp8(F_.quantize_experts(*leaves[:3]), leaves[3], n)
    with torch.no_grad():
        plain = F_.bmm_experts_fp8(F_.quantize_experts(*leaves[:3], for_backward=False), leaves[3], n.long())
    assert torch.equal(plain, y)
    y.backward(d_y.to(dev))
    _within("y", y, *want["y"])
    for name, leaf in zip(("d_w1", "d_w2", "d_w3", "d_x"), leaves):
        _within(name, leaf.grad, *want[name])


@pytest.mark.parametrize("A,E,H,I", [(8, 8, 2048, 768), (1, 1, 2048, 768), (24, 16, 1024, 512), (3, 2, 200, 130)])
def test_few_rows(dev, A, E, H, I):
    print(f"[case] fp8 experts, few rows {A} {E} {H} {I}", flush=True)
    g = torch.Generator().manual_seed(A)
    counts = torch.bincount(torch.randint(0, E, (A,), generator=g), minlength=E).tolist()
    w1, w2, w3, x, _ = _inputs(E, H, I, counts, 0, A, False)
    want = B.experts_between(w1, w2, w3, x, counts, decoded=_decoded(E, x.shape[0]))
    with torch.no_grad():
        y = F_.bmm_experts_fp8(F_.quantize_experts(*(w.to(dev) for w in (w1, w2, w3)), for_backward=False), x.to(dev),
                               torch.tensor(counts, device=dev))
    _within("y", y, *want["y"])


@pytest.mark.parametrize("E,H,I,counts,spare", [(3, 256, 384, [40, 0, 17], 5), (2, 130, 70, [1, 33], 0), (130, 72, 200, [i % 3 for i in range(130)], 2)])
def test_both_ways_of_the_forward_take_any_rows(dev, E, H, I, counts, spare):
    """pk_fp8_experts_few_rows where pk_fp8_few_rows_pays would not choose it, and the tiles where it would."""
    print(f"[case] fp8 experts both ways E={E} H={H} I={I}", flush=True)
    lib, A = _lib.load(), sum(counts) + spare
    w1, w2, w3, x, _ = _inputs(E, H, I, counts, spare, 9, False)
    want = B.experts_between(w1, w2, w3, x, counts, decoded=_decoded(E, x.shape[0]))
    e = F_.quantize_experts(*(w.to(dev) for w in (w1, w2, w3)))
    xd, n, st = x.to(dev), torch.tensor(counts, dtype=torch.int64, device=dev), _lib.current_stream(dev)
    p = lambda t: t.data_ptr()  # noqa: E731
    y, h = torch.full((A, H), 7.0, device=dev).bfloat16(), torch.empty(A, I, device=dev)
    g, u = (torch.empty(A, I, device=dev).bfloat16() for _ in range(2))
    assert lib.pk_fp8_experts_few_rows(p(xd), p(n), 1, p(e.q1), p(e.s1), p(e.q2), p(e.s2), p(e.q3), p(e.s3), p(g), p(u), p(h), p(y), A, H, I, E, st) == 0
    _within("y, few rows", y, *want["y"])
    bare = torch.full((A, H), 7.0, device=dev).bfloat16()
    assert lib.pk_fp8_experts_few_rows(p(xd), p(n), 1, p(e.q1), p(e.s1), p(e.q2), p(e.s2), p(e.q3), p(e.s3), None, None, p(h), p(bare), A, H, I, E, st) == 0
    assert torch.equal(y, bare)
    q, s = ops.quantize_rows_fp8(xd)
    plan = torch.empty(lib.pk_fp8_plan_bytes(A, E) // 4, dtype=torch.int32, device=dev)
    h8, hs = torch.empty(A, -(-I // 128) * 128, dtype=torch.uint8, device=dev), torch.empty(A, -(-I // 512) * 4, dtype=torch.uint8, device=dev)
    tiles = torch.full((A, H), 7.0, device=dev).bfloat16()
    g2, u2 = (torch.empty(A, I, device=dev).bfloat16() for _ in range(2))
    assert lib.pk_fp8_plan(p(n), 1, E, A, p(plan), st) == 0
    assert plan[:E + 1].tolist() == [0] + torch.tensor(counts).cumsum(0).tolist()
    assert lib.pk_fp8_gate_up(p(q), p(s), p(e.q1), p(e.s1), p(e.q3), p(e.s3), p(plan), p(g2), p(u2), p(h8), p(hs), A, H, I, E, st) == 0
    assert lib.pk_fp8_down(p(h8), p(hs), p(e.q2), p(e.s2), p(plan), p(tiles), A, H, I, E, st) == 0
    owned = sum(counts)
    assert (tiles[owned:] == 0).all() and (y[owned:] == 0).all()
    _within("y, tiles", tiles, *want["y"])
    # both are the bf16 rounding of sums that differ in the last places
    for a, b in ((g, g2), (u, u2)):
        assert ((a[:owned].float() - b[:owned].float()).abs() <= 2.0 ** -7 * a[:owned].float().abs() + 1e-3).all()


@pytest.mark.parametrize("rows", [1, 40])
def test_few_rows_lose_no_small_products(dev, rows):
    """Two large products that cancel, 126 others that are 2^-15 of them: exact in fp32 (and in bf16 at the end) if nothing is cut off."""
    print(f"[case] fp8 experts, products of very different size, {rows} rows", flush=True)
    lib, E, H, I, st = _lib.load(), 2, 128, 136, _lib.current_stream(dev)
    x = torch.full((rows, H), 2.0 ** -6)
    x[:, 0], x[:, 8] = 256.0, -256.0
    w = torch.full((E, I, H), 0.5)
    w[:, :, 0] = w[:, :, 8] = 1.0
    x, w, w2 = x.bfloat16().to(dev), w.bfloat16().to(dev), torch.zeros(E, H, I).bfloat16().to(dev)
    with torch.no_grad():
        e = F_.quantize_experts(w, w2, w)
    p = lambda t: t.data_ptr()  # noqa: E731
    n = torch.tensor([rows // 2, rows - rows // 2], device=dev)
    plan = torch.empty(lib.pk_fp8_plan_bytes(rows, E) // 4, dtype=torch.int32, device=dev)
    q, s = torch.empty(rows, 128, dtype=torch.uint8, device=dev), torch.empty(rows, 4, dtype=torch.uint8, device=dev)
    h8, hs = torch.empty(rows, 256, dtype=torch.uint8, device=dev), torch.empty(rows, 4, dtype=torch.uint8, device=dev)
    h, y = torch.empty(rows, I, device=dev), torch.empty(rows, H, device=dev).bfloat16()
    for few in (True, False):
        g, u = (torch.zeros(rows, I, device=dev).bfloat16() for _ in range(2))
        if few:
            assert lib.pk_fp8_experts_few_rows(p(x), p(n), 1, p(e.q1), p(e.s1), p(e.q2), p(e.s2), p(e.q3), p(e.s3), p(g), p(u), p(h), p(y), rows, H, I, E, st) == 0
        else:
            assert lib.pk_fp8_begin(p(x), p(n), 1, p(q), p(s), p(plan), rows, H, E, st) == 0
            assert lib.pk_fp8_gate_up(p(q), p(s), p(e.q1), p(e.s1), p(e.q3), p(e.s3), p(plan), p(g), p(u), p(h8), p(hs), rows, H, I, E, st) == 0
        assert (g == 126 * 2.0 ** -7).all() and torch.equal(g, u)


def test_counts_that_do_not_fit_lead_nowhere(dev):
    """More rows than there are, and negative counts: cut off, so that nothing is read or written out of bounds."""
    print("[case] fp8 experts, counts that do not fit", flush=True)
    w, x, d_y, _ = _setup(dev, counts=(20, 0, 44))
    with torch.no_grad():
        e = F_.quantize_experts(*w)
        for bad, good in (((20, -3, 1000), (20, 0, 44)), ((10 ** 6, 5, 5), (64, 0, 0)), ((-1, -1, 7), (0, 0, 7)), ((2 ** 40, 2 ** 40, 2 ** 40), (64, 0, 0))):
            for A in (64, 20):
                b, g = torch.tensor(bad, device=dev), [0, 0, 0]
                left = A
                for i, c in enumerate(good):
                    g[i] = min(c, left)
                    left -= g[i]
                assert torch.equal(F_.bmm_experts_fp8(e, x[:A], b), F_.bmm_experts_fp8(e, x[:A], torch.tensor(g, device=dev)))


@pytest.mark.parametrize("counts", [[4, 5], [170, 161]])
def test_a_row_that_is_not_finite_stays_a_row(dev, counts):
    print(f"[case] fp8 experts, NaN and infinity, {counts}", flush=True)
    w1, w2, w3, x, _ = _inputs(2, 256, 128, counts, 0, 5, False)
    bad = x.clone()
    bad[1, 7], bad[6, 200] = math.inf, math.nan
    experts = F_.quantize_experts(*(w.to(dev) for w in (w1, w2, w3)))
    n = torch.tensor(counts, device=dev)
    y, z = F_.bmm_experts_fp8(experts, x.to(dev), n), F_.bmm_experts_fp8(experts, bad.to(dev), n)
    whole = torch.ones(sum(counts), dtype=torch.bool)
    whole[[1, 6]] = False
    assert torch.equal(y[whole], z[whole]) and torch.isnan(z[~whole]).all()


# ------------------------------------------------------------------------------ the operator
def _setup(dev, seed=0, counts=(20, 0, 44), H=256, I=128):
    w1, w2, w3, x, d_y = _inputs(len(counts), H, I, counts, 0, seed, False)
    w = [t.to(dev).requires_grad_(True) for t in (w1, w2, w3)]
    return w, x.to(dev).requires_grad_(True), d_y.to(dev), torch.tensor(counts, dtype=torch.int32, device=dev)


def _pass(w, x, d_y, n):
    y = F_.bmm_experts_fp8(F_.quantize_experts(*w), x, n)
    return (y.detach(), *torch.autograd.grad(y, (*w, x), d_y))


def _equal(a, b):
    return all(torch.equal(p, q) for p, q in zip(a, b))


def test_strides_streams_and_which_gradients(dev):
    print("[case] fp8 experts: strides, a stream, partial gradients", flush=True)
    w, x, d_y, n = _setup(dev)
    want = _pass(w, x, d_y, n)
    xt = x.detach().t().contiguous().t().requires_grad_(True)
    assert _equal(want, _pass(w, xt, d_y.t().contiguous().t(), n))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _pass(w, x, d_y, n)
    torch.cuda.current_stream().wait_stream(side)
    assert _equal(want, got)
    experts = F_.quantize_experts(*w)
    only_x = torch.autograd.grad(F_.bmm_experts_fp8(experts._replace(w1=None, w2=None, w3=None), x, n), x, d_y)[0]
    assert torch.equal(only_x, want[4])
    only_w = torch.autograd.grad(F_.bmm_experts_fp8(experts, x.detach(), n), w[1], d_y)[0]
    assert torch.equal(only_w, want[2])
    expanded = torch.autograd.grad(F_.bmm_experts_fp8(experts, x, n).sum(), x)[0]      # a gradient of stride zero
    assert torch.equal(expanded, torch.autograd.grad(F_.bmm_experts_fp8(experts, x, n), x, torch.ones_like(d_y))[0])


def test_empty_input(dev):
    print("[case] fp8 experts: no rows", flush=True)
    w, x, d_y, _ = _setup(dev)
    n = torch.zeros(3, dtype=torch.int32, device=dev)
    got = _pass(w, x.detach()[:0].requires_grad_(True), d_y[:0], n)
    assert got[0].shape == (0, 256) and all((t == 0).all() for t in got[1:4]) and got[4].shape == (0, 256)
    got = _pass(w, x, d_y, n)                              # rows, but nobody's
    assert all((t == 0).all() for t in got)


@pytest.mark.parametrize("counts,spare", [([45, 0, 64, 131], 70), ([1, 500, 31, 32], 0), ([0, 0, 0, 200], 3)])
def test_transposed_copies_give_the_same_weight_gradients(dev, counts, spare):
    """pk_fp8_dgrad_dh_t with pk_fp8_begin_backward's row map and pk_grouped_swiglu_wgrad_scaled_t against the row-major pair.  What stands in rows of no
    expert does not matter."""
    print(f"[case] fp8 d_h, transposed copies, {counts}", flush=True)
    lib, E, H, I = _lib.load(), 4, 512, 256
    A, st = sum(counts) + spare, _lib.current_stream(dev)
    w1, w2, w3, x, d_y = (t.to(dev) for t in _inputs(E, H, I, counts, spare, 3, False))
    x[sum(counts):] = math.nan
    d_y[sum(counts):] = math.inf
    e = F_.quantize_experts(w1, w2, w3)
    gu = (torch.randn(2, A, I, generator=torch.Generator().manual_seed(1))).bfloat16().to(dev)
    p = lambda t: t.data_ptr()  # noqa: E731
    n = torch.tensor(counts, dtype=torch.int32, device=dev)
    plan = torch.empty(lib.pk_fp8_plan_bytes(A, E) // 4, dtype=torch.int32, device=dev)
    assert lib.pk_fp8_plan(p(n), 0, E, A, p(plan), st) == 0
    q, s = ops.quantize_rows_fp8(d_y)
    ldt = lib.pk_grouped_swiglu_transposed_ld(A, H, I, E, _lib.PK_BF16)
    sides = []
    for transposed in (False, True):
        codes = [torch.zeros(A, I, dtype=torch.uint8, device=dev) for _ in range(2)] + [torch.zeros(A, -(-I // 512) * 4, dtype=torch.uint8, device=dev) for _ in range(2)]
        g8, u8, gs, us = codes
        copies = torch.full((3, ldt if transposed else A, I), math.nan, device=dev).bfloat16()
        args = (p(q), p(s), p(e.t2), p(e.s2), p(gu[0]), p(gu[1]), p(plan), p(copies[0]), p(copies[1]), p(copies[2]))
        tail = (p(g8), p(gs), p(u8), p(us), A, H, I, E, st)
        d1, d2, d3 = (torch.empty(s_, device=dev).bfloat16() for s_ in ((E, I, H), (E, H, I), (E, I, H)))
        if transposed:
            row_map = torch.empty(A, dtype=torch.int32, device=dev)
            again = [torch.zeros_like(q), torch.zeros(A, 4, dtype=torch.float8_e8m0fnu, device=dev)]
            assert lib.pk_fp8_begin_backward(p(d_y), p(plan), p(again[0]), p(again[1]), p(row_map), A, H, E, st) == 0
            assert torch.equal(again[0].view(torch.uint8), q.view(torch.uint8)) and torch.equal(again[1].view(torch.uint8), s.view(torch.uint8))
            assert row_map.tolist() == [min(r, sum(counts) - 1) for r in range(A)]
            assert lib.pk_fp8_dgrad_dh_t(*args, ldt, *tail) == 0
            assert lib.pk_grouped_swiglu_wgrad_scaled_t(p(d_y), p(copies[2]), p(copies[0]), p(copies[1]), ldt, p(x), p(row_map), 1, p(plan), None, p(d1),
                                                        p(d2), p(d3), 0, A, H, I, E, _lib.PK_BF16, st) == 0
        else:
            assert lib.pk_fp8_dgrad_dh(*args, *tail) == 0
            assert lib.pk_grouped_swiglu_wgrad(p(d_y), p(copies[2]), p(copies[0]), p(copies[1]), p(x), None, 1, p(plan), None, p(d1), p(d2), p(d3), 0, A, H,
                                               I, E, _lib.PK_BF16, st) == 0
        sides.append((codes, (d1, d2, d3)))
    for a, b in zip(*(side[0] for side in sides)):
        assert torch.equal(a, b)
    for a, b in zip(*(side[1] for side in sides)):
        # the same bf16 operands, summed in another order: both are within the rounding of the result and of n sums
        assert torch.isfinite(a).all()
        size = a.double().abs() + 2.0 ** -20 * max(counts) * a.double().abs().max()
        assert ((a.double() - b.double()).abs() <= 2.0 ** -7 * size).all()


def test_accumulated_and_postponed_weight_gradients(dev):
    print("[case] fp8 experts: accumulate, defer", flush=True)
    w, x, d_y, n = _setup(dev)
    want = _pass(w, x, d_y, n)
    experts = F_.quantize_experts(*w)
    with F_.defer_weight_grads() as q:
        F_.bmm_experts_fp8(experts, x, n).backward(d_y)
    assert torch.equal(x.grad, want[4]) and all(p.grad is None for p in w) and len(q) == 1
    q.run()
    assert _equal([p.grad for p in w], want[1:4])
    kept = [p.grad for p in w]
    with F_.accumulate_weight_grads():
        F_.bmm_experts_fp8(experts, x, n).backward(d_y)
    for p, k, g in zip(w, kept, want[1:4]):
        assert p.grad is k
        # the old gradient is bf16 and twice it is exact; the new one is added before it is rounded: half a step of bf16 of the sum
        assert ((p.grad.double() - 2 * g.double()).abs() <= 2.0 ** -8 * 2 * g.double().abs() + 2.0 ** -8 * g.double().abs()).all()


def test_captured_and_replayed(dev):
    print("[case] fp8 experts in a graph", flush=True)
    w, x, d_y, n = _setup(dev, counts=(30, 3, 31))
    w = [p.detach() for p in w]
    x = x.detach()
    n = n.clone()

    def forward():
        with torch.no_grad():
            return F_.bmm_experts_fp8(F_.quantize_experts(*w, for_backward=False), x, n)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        forward()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = forward()
    for rep in range(4):
        g = torch.Generator().manual_seed(rep)
        x.copy_(torch.randn(x.shape, generator=g))
        n.copy_(torch.tensor([(64, 0, 0), (1, 62, 1), (0, 0, 17), (20, 22, 22)][rep], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, forward()), f"replay {rep}"


MANY = dict(counts=(300, 0, 129, 171), H=512, I=256)      # tiles, products of codes, transposed copies where they pay


def test_many_rows_strides_streams_and_accumulation(dev):
    """What the tests above ask of a few rows, of passes that go through the tiles."""
    print("[case] fp8 experts, many rows: strides, streams, partial gradients, accumulate, defer", flush=True)
    w, x, d_y, n = _setup(dev, **MANY)
    want = _pass(w, x, d_y, n)
    xt = x.detach().t().contiguous().t().requires_grad_(True)
    assert _equal(want, _pass(w, xt, d_y.t().contiguous().t(), n))
    odd = torch.cat([x.new_zeros(1), x.detach().reshape(-1)])[1:].view(x.shape).requires_grad_(True)      # 2-byte aligned rows
    got = _pass(w, odd, d_y, n)
    assert torch.equal(got[0], want[0]) and torch.equal(got[4], want[4])
    # the weights' gradients are summed in another order where 16-byte loads do not fit
    bounds = B.experts_between(*(t.detach().cpu() for t in (*w, x)), MANY["counts"], d_y.cpu())
    for name, t in zip(("d_w1", "d_w2", "d_w3"), got[1:4]):
        _within(name, t, *bounds[name])
    sides = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for side in sides:                                     # two passes at once
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got.append(_pass(w, x, d_y, n))
    for side, g in zip(sides, got):
        torch.cuda.current_stream().wait_stream(side)
        assert _equal(want, g)
    experts = F_.quantize_experts(*w)
    only_x = torch.autograd.grad(F_.bmm_experts_fp8(experts._replace(w1=None, w2=None, w3=None), x, n), x, d_y)[0]
    only_w = torch.autograd.grad(F_.bmm_experts_fp8(experts, x.detach(), n), w[1], d_y)[0]
    assert torch.equal(only_x, want[4]) and torch.equal(only_w, want[2])
    with F_.defer_weight_grads() as q:
        F_.bmm_experts_fp8(experts, x, n).backward(d_y)
    assert torch.equal(x.grad, want[4]) and all(p.grad is None for p in w)
    q.run()
    assert _equal([p.grad for p in w], want[1:4])
    kept = [p.grad for p in w]
    with F_.accumulate_weight_grads():
        F_.bmm_experts_fp8(experts, x, n).backward(d_y)
    for p, k, g in zip(w, kept, want[1:4]):
        assert p.grad is k
        # as above: half a step of bf16 of the sum, and of the new gradient
        assert ((p.grad.double() - 2 * g.double()).abs() <= 2.0 ** -8 * 2 * g.double().abs() + 2.0 ** -8 * g.double().abs()).all()


def test_many_rows_and_counts_that_do_not_fit(dev):
    print("[case] fp8 experts, many rows, counts that do not fit, rows of nobody", flush=True)
    w, x, d_y, n = _setup(dev, **MANY)
    for bad, good in (((300, -3, 1000, 5), (300, 0, 300, 0)), ((10 ** 6, 5, 5, 5), (600, 0, 0, 0)), ((-1, -1, 7, -2 ** 31), (0, 0, 7, 0)),
                      ((2 ** 40,) * 4, (600, 0, 0, 0)), ((0, 0, 0, 0), (0, 0, 0, 0))):
        got, want = (_pass(w, x, d_y, torch.tensor(c, device=dev)) for c in (bad, good))
        assert _equal(got, want)
        assert all((t[sum(good):] == 0).all() for t in (got[0], got[4]))
        assert all((g[e] == 0).all() for g in got[1:4] for e in range(4) if good[e] == 0)


def test_many_rows_captured_and_replayed_with_their_backward(dev):
    print("[case] fp8 experts, many rows, forward and backward in a graph", flush=True)
    w, x, d_y, n = _setup(dev, **MANY)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _pass(w, x, d_y, n)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _pass(w, x, d_y, n)
    for rep in range(4):
        g = torch.Generator().manual_seed(rep)
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, generator=g))
            w[1].mul_(0.5)
        d_y.copy_(torch.randn(d_y.shape, generator=g))
        n.copy_(torch.tensor([(600, 0, 0, 0), (1, 1, 597, 1), (0, 0, 17, 200), (150, 150, 150, 150)][rep], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert _equal(out, _pass(w, x, d_y, n)), f"replay {rep}"


@pytest.mark.parametrize("rows", [20, 300])
def test_largest_widths(dev, rows):
    """H 8192 and I 4096, through the C ABI, on integers whose sums are exact in any order (products are at most 16 units, so the matrix
    instructions cut nothing off either)."""
    print(f"[case] fp8 experts, largest widths, {rows} rows", flush=True)
    lib, E, H, I, st = _lib.load(), 1, 8192, 4096, _lib.current_stream(dev)
    w1, w2, w3, x, d_y = (t.to(dev) for t in _inputs(E, H, I, [rows], 0, 5, True))
    e = F_.quantize_experts(w1, w2, w3)
    p = lambda t: t.data_ptr()  # noqa: E731
    n = torch.tensor([rows], dtype=torch.int32, device=dev)
    new = lambda *shape, dtype=torch.bfloat16: torch.zeros(shape, dtype=dtype, device=dev)  # noqa: E731
    plan, byte = torch.empty(lib.pk_fp8_plan_bytes(rows, E) // 4, dtype=torch.int32, device=dev), dict(dtype=torch.uint8)
    q, s, h8, hs = new(rows, H, **byte), new(rows, H // 128, **byte), new(rows, I, **byte), new(rows, I // 128, **byte)
    g, u, y, d_x = new(rows, I), new(rows, I), new(rows, H), new(rows, H)
    dot = lambda a, b: (a.double() @ b.double().t().contiguous())  # noqa: E731
    assert lib.pk_fp8_begin(p(x), p(n), 0, p(q), p(s), p(plan), rows, H, E, st) == 0
    assert lib.pk_fp8_gate_up(p(q), p(s), p(e.q1), p(e.s1), p(e.q3), p(e.s3), p(plan), p(g), p(u), p(h8), p(hs), rows, H, I, E, st) == 0
    assert torch.equal(g, dot(x, w1[0]).bfloat16()) and torch.equal(u, dot(x, w3[0]).bfloat16())
    if rows <= 128:
        g2, u2, h = new(rows, I), new(rows, I), new(rows, I, dtype=torch.float32)
        assert lib.pk_fp8_experts_few_rows(p(x), p(n), 0, p(e.q1), p(e.s1), p(e.q2), p(e.s2), p(e.q3), p(e.s3), p(g2), p(u2), p(h), p(y), rows, H, I, E, st) == 0
        assert torch.equal(g, g2) and torch.equal(u, u2) and torch.isfinite(y).all()
    ints = x[:, :I].contiguous()                           # in the place of h, d_g and d_u
    hq, hqs = ops.quantize_rows_fp8(ints)
    assert lib.pk_fp8_down(p(hq), p(hqs), p(e.q2), p(e.s2), p(plan), p(y), rows, H, I, E, st) == 0
    assert torch.equal(y, dot(ints, w2[0]).bfloat16())
    assert lib.pk_fp8_dgrad_dx(p(hq), p(hqs), p(hq), p(hqs), p(e.t1), p(e.s1), p(e.t3), p(e.s3), p(plan), p(d_x), rows, H, I, E, st) == 0
    assert torch.equal(d_x, (ints.double() @ (w1[0].double() + w3[0].double())).bfloat16())
    # silu(64) = 64 in fp32, so d_u = 64 d_h
    g.fill_(64.0)
    u.fill_(1.0)
    out = [new(rows, I) for _ in range(3)]
    codes = [new(rows, I, **byte), new(rows, I // 128, **byte), new(rows, I, **byte), new(rows, I // 128, **byte)]
    assert lib.pk_fp8_begin_backward(p(d_y), p(plan), p(q), p(s), None, rows, H, E, st) == 0
    assert lib.pk_fp8_dgrad_dh(p(q), p(s), p(e.t2), p(e.s2), p(g), p(u), p(plan), *(p(t) for t in out), *(p(t) for t in codes), rows, H, I, E, st) == 0
    want = 64 * (d_y.double() @ w2[0].double())
    assert torch.equal(out[1], want.bfloat16()) and (out[2] == 64).all()
    wq, ws = B.rows(out[1].cpu())
    assert _same(codes[2].view(E4M3), wq) and torch.equal(_exponents(codes[3]), ws)


def test_modules_call_it(dev):
    print("[case] fp8 experts in the modules", flush=True)
    torch.manual_seed(0)
    args = MoEArgs(num_experts=4, top_k=2, route_norm=True)
    moe = AnnotatedMoE(args, 256, 128, dtype=torch.bfloat16, fused=False).to(dev)
    moe.init_weights()
    x = torch.randn(2, 33, 256, device=dev).bfloat16()
    e8 = moe.experts.quantize()
    out = moe(x, experts_fp8=e8)
    out.float().square().sum().backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in moe.parameters())
    ref = moe(x)
    # the two differ by the rounding of three operands to e4m3 (half a step 2^-4 each), averaged over sums of 128 terms and more
    assert (out - ref).float().norm() <= 3 * 2.0 ** -4 * ref.float().norm()
    experts = BmmExperts(256, 128, 2, dtype=torch.bfloat16).to(dev)
    for p in experts.parameters():
        torch.nn.init.normal_(p, std=0.05)
    rows, n = torch.randn(9, 256, device=dev).bfloat16(), torch.tensor([4, 5], device=dev)
    assert torch.equal(experts(rows, n, experts.quantize()), F_.bmm_experts_fp8(F_.quantize_experts(experts.w1, experts.w2, experts.w3), rows, n))


def test_captured_by_dynamo_as_one_node(dev):
    print("[case] fp8 experts under dynamo", flush=True)
    w, x, d_y, n = _setup(dev)
    experts = F_.quantize_experts(*w)
    seen = []

    def backend(gm, inputs):
        seen.extend(str(node.target) for node in gm.graph.nodes if node.op == "call_function")
        return gm.forward

    def fn(x):
        return F_.bmm_experts_fp8(experts, x * 1, n)

    got = torch.compile(fn, backend=backend, fullgraph=True)(x)
    assert any("bmm_experts_fp8" in s for s in seen)
    assert torch.equal(got, fn(x))


def test_refusals(dev):
    w, x, d_y, n = _setup(dev)
    e = F_.quantize_experts(*w)
    with pytest.raises(TypeError, match="rows are bfloat16"):
        F_.bmm_experts_fp8(e, x.float(), n)
    with pytest.raises(ValueError, match="row count for every expert"):
        F_.bmm_experts_fp8(e, x[:, :-1], n)
    with pytest.raises(ValueError, match="row count for every expert"):
        F_.bmm_experts_fp8(e, x, n[:2])
    with pytest.raises(ValueError, match="transposed codes"):
        F_.bmm_experts_fp8(F_.quantize_experts(*w, for_backward=False), x, n)
    with pytest.raises(ValueError, match="expected a contiguous"):
        F_.bmm_experts_fp8(e._replace(q2=e.q1), x, n)
    with pytest.raises(ValueError, match="expected a contiguous"):
        F_.bmm_experts_fp8(e._replace(s1=e.s1.view(torch.uint8)), x, n)
    with pytest.raises(ValueError, match="counts must be int32 or int64"):
        F_.bmm_experts_fp8(e, x, n.float())
    with pytest.raises(TypeError, match="float32 and bfloat16"):
        F_.quantize_experts(*(p.detach().half() for p in w))
    with pytest.raises(ValueError, match="shapes disagree"):
        F_.quantize_experts(w[0], w[0], w[2])
    with pytest.raises(ValueError):
        ops.quantize_rows_fp8(x, row_map_div=2)
    wide = torch.zeros(1, 8, 8200, dtype=torch.bfloat16, device=dev)
    with pytest.raises(RuntimeError, match="shape not supported"):
        with torch.no_grad():
            F_.bmm_experts_fp8(F_.quantize_experts(wide, wide.view(1, 8200, 8), wide), torch.zeros(2, 8200, dtype=torch.bfloat16, device=dev),
                               torch.tensor([2], device=dev))
