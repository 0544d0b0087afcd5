"""The experts in 8-bit blocks with many rows an expert: what every sum keeps, and the kernels that passes of real size run."""
import pytest
import torch

from oracle import blocks as B
from piper_amd import _lib, ops
from piper_amd import functional as F_
from test_gpu_fp8 import _inputs, _within

pytestmark = pytest.mark.gpu


def _p(t):
    return None if t is None else t.data_ptr()


def _plan(lib, counts, A, dev):
    n = torch.tensor(counts, dtype=torch.int32, device=dev)
    plan = torch.empty(lib.pk_fp8_plan_bytes(A, len(counts)) // 4, dtype=torch.int32, device=dev)
    assert lib.pk_fp8_plan(_p(n), 0, len(counts), A, _p(plan), _lib.current_stream(dev)) == 0
    return plan


# ------------------------------------------------------------------------------ sums
def _cancelling(rows, K):
    """Rows whose products with ones are 256, 2^-6, ..., -256 within eight values: 2^-6 (K - 2) in all, exact in fp32 and lost if
    less than 15 bits are kept below the largest product."""
    x = torch.full((rows, K), 2.0 ** -6)
    x[:, 0], x[:, 5] = 256.0, -256.0
    return x.bfloat16()


# (2 experts: units of 128 columns; 130: of 256, and more of them than CUs)
@pytest.mark.parametrize("E,each,N", [(2, 150, 264), (130, 45, 512), (130, 45, 391)])
def test_many_rows_lose_no_small_products(dev, E, each, N):
    print(f"[case] fp8 experts, products of very different size, {E} x {each} rows, {N} columns", flush=True)
    lib, K, A, st = _lib.load(), 256, E * each, _lib.current_stream(dev)
    assert A > 40 * E and A > 128
    plan = _plan(lib, [each] * E, A, dev)
    q, s = ops.quantize_rows_fp8(_cancelling(A, K).to(dev))
    ones = lambda *shape: torch.ones(shape, device=dev).bfloat16()  # noqa: E731
    e = F_.quantize_experts(ones(E, N, K), ones(E, K, N), ones(E, N, K))
    down = F_.quantize_experts(ones(E, K, N), ones(E, N, K), ones(E, K, N))      # [N, K] as the second weight, and its transposes
    new = lambda w, dtype=torch.bfloat16: torch.zeros(A, w, dtype=dtype, device=dev)  # noqa: E731
    whole, words = -(-N // 128) * 128, -(-N // 512) * 4
    codes = lambda: [new(whole, torch.uint8), new(words, torch.uint8), new(whole, torch.uint8), new(words, torch.uint8)]  # noqa: E731
    want = 2.0 ** -6 * (K - 2)                             # 127 * 2^-5: seven bits, a bf16 value
    g, u, c = new(N), new(N), codes()
    assert lib.pk_fp8_gate_up(_p(q), _p(s), _p(e.q1), _p(e.s1), _p(e.q3), _p(e.s3), _p(plan), _p(g), _p(u), _p(c[0]), _p(c[1]), A, K, N, E, st) == 0
    assert (g == want).all() and (u == want).all()
    y = new(N)
    assert lib.pk_fp8_down(_p(q), _p(s), _p(down.q2), _p(down.s2), _p(plan), _p(y), A, N, K, E, st) == 0
    assert (y == want).all()
    d_x = new(N)
    assert lib.pk_fp8_dgrad_dx(_p(q), _p(s), _p(q), _p(s), _p(down.t1), _p(down.s1), _p(down.t3), _p(down.s3), _p(plan), _p(d_x), A, N, K, E, st) == 0
    assert (d_x == 2 * want).all()
    # silu(64) = 64 in fp32: d_u = 64 d_h
    g.fill_(64.0)
    u.fill_(1.0)
    out = [new(N) for _ in range(3)]
    assert lib.pk_fp8_dgrad_dh(_p(q), _p(s), _p(e.t2), _p(e.s2), _p(g), _p(u), _p(plan), *map(_p, out), *map(_p, codes()), A, K, N, E, st) == 0
    assert (out[1] == 64 * want).all()
    if N % 256 == 0:
        ldt = lib.pk_grouped_swiglu_transposed_ld(A, K, N, E, _lib.PK_BF16)
        t = torch.zeros(3, ldt // 32, N, 32, dtype=torch.bfloat16, device=dev)
        assert lib.pk_fp8_dgrad_dh_t(_p(q), _p(s), _p(e.t2), _p(e.s2), _p(g), _p(u), _p(plan), _p(t[0]), _p(t[1]), _p(t[2]), ldt, *map(_p, codes()), A, K, N,
                                     E, st) == 0
        assert set(t[1].unique().tolist()) <= {0.0, 64 * want} and int((t[1] != 0).sum()) == A * N


@pytest.mark.parametrize("E,H,I,counts,spare", [(4, 256, 512, [200, 33, 0, 64], 7), (3, 257, 300, [150, 140, 90], 3)])
def test_many_rows_are_within_the_bounds_of_fp32_sums(dev, E, H, I, counts, spare):
    print(f"[case] fp8 experts, sums in fp32, {counts}", flush=True)
    w1, w2, w3, x, d_y = _inputs(E, H, I, counts, spare, E, False)
    want = B.experts_between(w1, w2, w3, x, counts, d_y, decoded=True)
    leaves = [t.to(dev).requires_grad_(True) for t in (w1, w2, w3, x)]
    y = F_.bmm_experts_fp8(F_.quantize_experts(*leaves[:3]), leaves[3], torch.tensor(counts, device=dev))
    y.backward(d_y.to(dev))
    for name, t in zip(("y", "d_w1", "d_w2", "d_w3", "d_x"), (y, *(leaf.grad for leaf in leaves))):
        _within(name, t, *want[name])


@pytest.mark.parametrize("E,H,I,counts,spare", [(4, 256, 512, [200, 33, 0, 64], 7), (3, 257, 300, [150, 140, 90], 3), (2, 256, 128, [30, 40], 0)])
def test_short_sums_are_the_callers_choice(dev, E, H, I, counts, spare):
    """Within the bounds that contain what the matrix instructions cut off; passes that are no faster for it are the default's."""
    print(f"[case] fp8 experts, short sums, {counts}", flush=True)
    w1, w2, w3, x, d_y = _inputs(E, H, I, counts, spare, E, False)
    few = x.shape[0] <= max(40 * E, 128)
    want = B.experts_between(w1, w2, w3, x, counts, d_y, decoded=few)
    n, passes = torch.tensor(counts, device=dev), []
    for short in (True, False):
        leaves = [t.to(dev).requires_grad_(True) for t in (w1, w2, w3, x)]
        experts = F_.quantize_experts(*leaves[:3], short_sums=short)
        assert experts.short_sums is short
        y = F_.bmm_experts_fp8(experts, leaves[3], n)
        y.backward(d_y.to(dev))
        with torch.no_grad():
            assert torch.equal(y, F_.bmm_experts_fp8(experts, leaves[3], n))
        passes.append((y.detach(), *(leaf.grad for leaf in leaves)))
    for name, t in zip(("y", "d_w1", "d_w2", "d_w3", "d_x"), passes[0]):
        _within(name, t, *want[name])
    assert not few or all(torch.equal(a, b) for a, b in zip(*passes))


# ------------------------------------------------------------------------------ weight gradients from transposed copies
PAYS = dict(E=4, H=2048, I=1024, counts=(50, 0, 97, 60))      # 128 units of 256 x 256 for fewer experts than XCDs


def _case(dev, E, H, I, counts, spare=0, seed=0):
    assert _lib.load().pk_region_transposed_pays(sum(counts) + spare, H, I, E, _lib.PK_BF16) == 1 and sum(counts) + spare > max(40 * E, 128)
    w1, w2, w3, x, d_y = (t.to(dev) for t in _inputs(E, H, I, counts, spare, seed, False))
    return [w.requires_grad_(True) for w in (w1, w2, w3)], x.requires_grad_(True), d_y, torch.tensor(counts, dtype=torch.int32, device=dev)


def _pass(w, x, d_y, n):
    y = F_.bmm_experts_fp8(F_.quantize_experts(*w), x, n)
    return (y.detach(), *torch.autograd.grad(y, (*w, x), d_y))


def _equal(a, b):
    return len(a) == len(b) and all(torch.equal(p, q) for p, q in zip(a, b))


def _odd(t):
    """The same values two bytes behind a 16-byte boundary."""
    t = t.detach()
    v = torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape)
    assert v.data_ptr() % 16 == 2
    return v


def test_views_that_start_anywhere(dev):
    print("[case] fp8 experts, transposed copies: unaligned rows, gradients and places of gradients", flush=True)
    w, x, d_y, n = _case(dev, **PAYS)
    want = _pass(w, x, d_y, n)
    assert _equal(want, _pass(w, _odd(x).requires_grad_(True), d_y, n))
    assert _equal(want, _pass(w, x, _odd(d_y), n))
    experts = F_.quantize_experts(*w)

    def added(places):
        for p, at in zip(w, places):
            p.grad = at
        F_.bmm_experts_fp8(experts, x, n).backward(d_y)
        assert all(p.grad is at for p, at in zip(w, places))
        return places

    with F_.accumulate_weight_grads():
        sums = added([g.clone() for g in want[1:4]])
        assert _equal(sums, added([_odd(g) for g in want[1:4]]))
        assert _equal(sums, added([want[1].clone(), _odd(want[2]), want[3].clone()]))
    places = [_odd(g) for g in want[1:4]]
    with F_.defer_weight_grads() as q:
        added(places)
        assert _equal(places, want[1:4])
    q.run()
    assert _equal(sums, places)


def test_rows_behind_4_gib(dev):
    """One expert has 1.05 million rows, those of the others begin behind 4 GiB of x and d_y, where the transposed pair's offsets end."""
    E, H, I, tail = 4, 2048, 1024, [0, 0, 50, 60]
    many = 1_049_900
    print(f"[case] fp8 experts, {many} rows and {tail}", flush=True)
    w1, w2, w3, x, d_y = _inputs(E, H, I, tail, 0, 4, False)
    want = B.experts_between(w1, w2, w3, x, tail, d_y, decoded=True)
    x_all, d_all = (torch.cat([torch.zeros(many, H, dtype=t.dtype, device=dev), t.to(dev)]).requires_grad_(t is x) for t in (x, d_y))
    assert many * H * 2 > 2 ** 32
    got = _pass([w.to(dev).requires_grad_(True) for w in (w1, w2, w3)], x_all, d_all, torch.tensor([many, *tail[1:]], device=dev))
    for name, t in zip(("y", "d_w1", "d_w2", "d_w3", "d_x"), got):
        rows = name in ("y", "d_x")
        assert (t[:many] == 0).all() if rows else (t[:2] == 0).all()
        _within(name, t[many:] if rows else t, *want[name])


@pytest.mark.parametrize("shape", [PAYS, dict(E=4, H=256, I=512, counts=(50, 0, 97, 60))])      # transposed copies, row-major operands
def test_weight_gradients_of_rows_that_are_not_finite(dev, shape):
    """The first and the last row of an expert, in x and in d_y: nobody else's gradients change."""
    counts, E = shape["counts"], shape["E"]
    print(f"[case] fp8 experts, backward with NaN and infinity, {shape}", flush=True)
    assert _lib.load().pk_region_transposed_pays(sum(counts), shape["H"], shape["I"], E, _lib.PK_BF16) == (shape is PAYS)
    w1, w2, w3, x, d_y = (t.to(dev) for t in _inputs(E, shape["H"], shape["I"], counts, 0, 8, False))
    w = [t.requires_grad_(True) for t in (w1, w2, w3)]
    n = torch.tensor(counts, device=dev)
    want = _pass(w, x.requires_grad_(True), d_y, n)
    for row, value in ((50, float("inf")), (146, float("nan"))):
        for which in (0, 1):
            rows = [x.detach().clone(), d_y.clone()]
            rows[which][row, ::9] = value
            got = _pass(w, rows[0].requires_grad_(True), rows[1], n)
            for g, t in zip(got[1:4], want[1:4]):
                assert not torch.isfinite(g[2]).all() and all(torch.equal(g[e], t[e]) for e in (0, 1, 3))
            others = torch.arange(sum(counts), device=dev) != row
            assert torch.equal(got[4][others], want[4][others]) and torch.isnan(got[4][row]).any()
