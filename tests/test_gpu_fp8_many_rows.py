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


# ------------------------------------------------------------------------------ the kernels that real sizes run
def _uneven(E, each, more):
    """`each` rows an expert or a few less and more, every ninth without any and some over a tile's 128."""
    return [0 if i % 9 == 4 else each + more * (i % 5 == 2) + i % 3 for i in range(E)]


# E, H, I, counts, rows of nobody.  Units of 256 columns, and more of them than CUs, so that workgroups go on to a second one: in down
# and d_h (of the last two in one each), with two to six k-tiles; odd widths; transposed copies where both are multiples of 256.
KERNELS = {
    "264 x 392": (150, 264, 392, _uneven(150, 45, 90), 5),
    "257 x 391": (150, 257, 391, _uneven(150, 45, 90), 0),
    "512 x 512": (130, 512, 512, _uneven(130, 47, 100), 3),
    "4096 x 384": (8, 4096, 384, [300, 291, 0, 513, 256, 128, 385, 527], 7),
    "384 x 4096": (8, 384, 4096, [300, 291, 0, 513, 256, 128, 385, 527], 0),
}


@pytest.mark.parametrize("short", [False, True])
@pytest.mark.parametrize("which", KERNELS)
def test_products_of_integers_are_exact(dev, which, short):
    """Through the C ABI, on integers whose sums are exact in any order and of which the short sums cut off nothing either.  Rows of nobody stay
    as they are but for y and d_x, which have zeros there."""
    E, H, I, counts, spare = KERNELS[which]
    print(f"[case] fp8 products of integers, {which}, short={short}", flush=True)
    lib, st, A, owned = _lib.load(), _lib.current_stream(dev), sum(counts) + spare, sum(counts)
    assert A > 40 * E and A > 128
    f = lambda name: getattr(lib, name + "_short" * short)  # noqa: E731
    w1, w2, w3, x, d_y = (t.to(dev) for t in _inputs(E, H, I, counts, spare, 6, True))
    e = F_.quantize_experts(w1, w2, w3)
    plan, starts = _plan(lib, counts, A, dev), [0]
    for c in counts:
        starts.append(starts[-1] + c)

    def per_expert(rows, w):                               # rows . w[e], w [E, K, N]
        out = torch.zeros(A, w.shape[2], dtype=torch.float64, device=dev)
        for i in range(E):
            r = slice(starts[i], starts[i + 1])
            out[r] = rows[r].double() @ w[i].double()
        return out.bfloat16()

    def same(t, want, rest):
        return torch.equal(t[:owned], want[:owned]) and bool((t[owned:] == rest).all())

    new = lambda w, dtype=torch.bfloat16: torch.full((A, w), 7, device=dev).to(dtype)  # noqa: E731
    codes = lambda w: (new(-(-w // 128) * 128, torch.uint8), new(-(-w // 512) * 4, torch.uint8))  # noqa: E731

    def blocks(of, t):
        q, s = ops.quantize_rows_fp8(of)
        blocks = -(-of.shape[1] // 128)
        return same(t[0], q.view(torch.uint8), 7) and same(t[1][:, :blocks], s.view(torch.uint8), 7)

    xq, xs = ops.quantize_rows_fp8(x)
    g, u, h = new(I), new(I), codes(I)
    assert f("pk_fp8_gate_up")(_p(xq), _p(xs), _p(e.q1), _p(e.s1), _p(e.q3), _p(e.s3), _p(plan), _p(g), _p(u), _p(h[0]), _p(h[1]), A, H, I, E, st) == 0
    assert same(g, per_expert(x, w1.transpose(1, 2).contiguous()), 7) and same(u, per_expert(x, w3.transpose(1, 2).contiguous()), 7)
    bare = codes(I)
    assert f("pk_fp8_gate_up")(_p(xq), _p(xs), _p(e.q1), _p(e.s1), _p(e.q3), _p(e.s3), _p(plan), None, None, _p(bare[0]), _p(bare[1]), A, H, I, E, st) == 0
    assert torch.equal(bare[0], h[0]) and torch.equal(bare[1], h[1])
    ints = x.repeat(1, -(-I // H))[:, :I].contiguous()     # in the place of h, d_g and d_u
    hq, hs = ops.quantize_rows_fp8(ints)
    y, d_x = new(H), new(H)
    assert f("pk_fp8_down")(_p(hq), _p(hs), _p(e.q2), _p(e.s2), _p(plan), _p(y), A, H, I, E, st) == 0
    assert same(y, per_expert(ints, w2.transpose(1, 2).contiguous()), 0)
    assert f("pk_fp8_dgrad_dx")(_p(hq), _p(hs), _p(hq), _p(hs), _p(e.t1), _p(e.s1), _p(e.t3), _p(e.s3), _p(plan), _p(d_x), A, H, I, E, st) == 0
    assert same(d_x, per_expert(ints, w1.double() + w3.double()), 0)
    # silu(64) = 64 and its derivative 1 in fp32: d_g = d_h, d_u = 64 d_h
    g.fill_(64.0)
    u.fill_(1.0)
    dq, ds = ops.quantize_rows_fp8(d_y)
    d_h = per_expert(d_y, w2)
    d_g, d_u, hb, g8, u8 = new(I), new(I), new(I), codes(I), codes(I)
    tail = (_p(g8[0]), _p(g8[1]), _p(u8[0]), _p(u8[1]), A, H, I, E, st)
    assert f("pk_fp8_dgrad_dh")(_p(dq), _p(ds), _p(e.t2), _p(e.s2), _p(g), _p(u), _p(plan), _p(d_g), _p(d_u), _p(hb), *tail) == 0
    assert same(d_g, d_h, 7) and same(d_u, 64 * d_h, 7) and same(hb, g, 7) and blocks(d_h, g8) and blocks(64 * d_h, u8)
    if H % 256 or I % 256:
        return
    ldt = lib.pk_grouped_swiglu_transposed_ld(A, H, I, E, _lib.PK_BF16)
    copies = torch.full((3, ldt // 32, I, 32), 7.0, device=dev).bfloat16()
    for t in (*g8, *u8):
        t.fill_(7)
    assert f("pk_fp8_dgrad_dh_t")(_p(dq), _p(ds), _p(e.t2), _p(e.s2), _p(g), _p(u), _p(plan), _p(copies[0]), _p(copies[1]), _p(copies[2]), ldt, *tail) == 0
    assert blocks(d_h, g8) and blocks(64 * d_h, u8)
    for copy, want in zip(copies, (d_h, 64 * d_h, g)):
        flat = copy.permute(0, 2, 1).reshape(ldt, I)       # by padded rows
        left = torch.ones(ldt, dtype=torch.bool, device=dev)
        for i, c in enumerate(counts):
            at = (starts[i] & ~63) + 64 * i
            end = -(-c // 32) * 32
            assert torch.equal(flat[at:at + c], want[starts[i]:starts[i + 1]]) and (flat[at + c:at + end] == 0).all()
            left[at:at + end] = False
        assert (flat[left] == 7).all()


@pytest.mark.parametrize("which", ["264 x 392", "257 x 391"])
def test_many_experts_are_within_their_bounds(dev, which):
    E, H, I, counts, spare = KERNELS[which]
    print(f"[case] fp8 experts, {E} of {which}", flush=True)
    w1, w2, w3, x, d_y = _inputs(E, H, I, counts, spare, 7, False)
    want = B.experts_between(w1, w2, w3, x, counts, d_y, decoded=True)
    got = _pass([w.to(dev).requires_grad_(True) for w in (w1, w2, w3)], x.to(dev).requires_grad_(True), d_y.to(dev), torch.tensor(counts, device=dev))
    for name, t in zip(("y", "d_w1", "d_w2", "d_w3", "d_x"), got):
        _within(name, t, *want[name])


# weight gradients from transposed copies: units handed out one after the other, and from 512 rows an expert on as they become free
@pytest.mark.parametrize("E,H,I,counts,spare", [(4, 2048, 1024, (50, 0, 97, 60), 9), (132, 256, 512, _uneven(132, 45, 90), 0), (4, 2048, 1024, (512, 3, 1025, 700), 11)])
def test_transposed_copies_are_within_their_bounds(dev, E, H, I, counts, spare):
    print(f"[case] fp8 experts, transposed copies, {E} of {H} x {I}, {sum(counts)} rows", flush=True)
    w, x, d_y, n = _case(dev, E, H, I, counts, spare, 3)
    want = B.experts_between(*(t.detach().cpu() for t in (*w, x)), counts, d_y.cpu(), decoded=True)
    for name, t in zip(("y", "d_w1", "d_w2", "d_w3", "d_x"), _pass(w, x, d_y, n)):
        _within(name, t, *want[name])


def test_transposed_copies_streams_postponed_and_added(dev):
    print("[case] fp8 experts, transposed copies: streams, partial gradients, accumulate, defer", flush=True)
    w, x, d_y, n = _case(dev, **PAYS)
    want = _pass(w, x, d_y, n)
    assert _equal(want, _pass(w, x.detach().t().contiguous().t().requires_grad_(True), d_y.t().contiguous().t(), n.long()))
    sides, got = [torch.cuda.Stream() for _ in range(2)], []
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
    assert torch.equal(x.grad, want[4]) and all(p.grad is None for p in w) and len(q) == 1
    junk = [torch.full_like(x, 9.0) for _ in range(8)]     # memory that the pass has given back
    q.run()
    assert _equal([p.grad for p in w], want[1:4]) and len(junk) == 8
    kept = [p.grad for p in w]
    with F_.accumulate_weight_grads():
        F_.bmm_experts_fp8(experts, x, n).backward(d_y)
    for p, k, g in zip(w, kept, want[1:4]):
        assert p.grad is k
        # the old gradient is bf16 and twice it is exact; the new one is added before it is rounded: half a step of bf16 of the sum
        assert ((p.grad.double() - 2 * g.double()).abs() <= 2.0 ** -8 * 2 * g.double().abs() + 2.0 ** -8 * g.double().abs()).all()


def test_transposed_copies_and_counts_that_do_not_fit(dev):
    print("[case] fp8 experts, transposed copies, counts that do not fit", flush=True)
    w, x, d_y, n = _case(dev, **PAYS)
    rows = sum(PAYS["counts"])
    for bad, good in (((50, -3, 1000, 5), (50, 0, rows - 50, 0)), ((10 ** 6, 5, 5, 5), (rows, 0, 0, 0)), ((-1, -1, 7, -2 ** 31), (0, 0, 7, 0)),
                      ((2 ** 40,) * 4, (rows, 0, 0, 0)), ((0, 0, 0, 0), (0, 0, 0, 0)), ((0, 0, 0, 64), (0, 0, 0, 64))):
        got, want = (_pass(w, x, d_y, torch.tensor(c, device=dev)) for c in (bad, good))
        assert _equal(got, want)
        assert all((t[sum(good):] == 0).all() for t in (got[0], got[4]))
        assert all((g[e] == 0).all() == (good[e] == 0) for g in got[1:4] for e in range(4))


def test_transposed_copies_captured_and_replayed_with_their_backward(dev):
    print("[case] fp8 experts, transposed copies, forward and backward in a graph", flush=True)
    w, x, d_y, n = _case(dev, **PAYS)
    rows = sum(PAYS["counts"])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _pass(w, x, d_y, n)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _pass(w, x, d_y, n)
    for rep, counts in enumerate([(rows, 0, 0, 0), (1, 1, rows - 3, 1), (0, 0, 17, 100), (50, 50, 50, 57)]):
        g = torch.Generator().manual_seed(rep)
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, generator=g))
            w[1].mul_(0.5)
        d_y.copy_(torch.randn(d_y.shape, generator=g))
        n.copy_(torch.tensor(counts, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert _equal(out, _pass(w, x, d_y, n)), f"replay {rep}"


# Few rows with more workgroups than it takes to fill the chip: whole reductions of five and more blocks to a wave in gate and up, four
# column tiles to a wave of down, with more blocks than it has on their way.
STREAMED = [(128, 960, 130, 256), (128, 1001, 139, 250), (150, 801, 257, 300)]


@pytest.mark.parametrize("E,H,I,A", STREAMED)
def test_few_rows_of_many_experts(dev, E, H, I, A):
    print(f"[case] fp8 experts, {A} rows of {E} experts {H} x {I}", flush=True)
    assert _lib.load().pk_fp8_few_rows_pays(A, H, I, E) == 1
    g = torch.Generator().manual_seed(A)
    counts = torch.bincount(torch.randint(0, E, (A - 3,), generator=g), minlength=E).tolist()
    w1, w2, w3, x, d_y = _inputs(E, H, I, counts, 3, A, False)
    want = B.experts_between(w1, w2, w3, x, counts, d_y, decoded=True)
    w, n = [t.to(dev).requires_grad_(True) for t in (w1, w2, w3)], torch.tensor(counts, device=dev)
    got = _pass(w, x.to(dev).requires_grad_(True), d_y.to(dev), n)
    with torch.no_grad():
        assert torch.equal(got[0], F_.bmm_experts_fp8(F_.quantize_experts(*w, for_backward=False), x.to(dev), n))
    for name, t in zip(("y", "d_w1", "d_w2", "d_w3", "d_x"), got):
        _within(name, t, *want[name])


def test_the_operator_takes_the_choice_last(dev):
    """Called by its name, as a captured graph does: without the choice it is the default."""
    print("[case] fp8 experts through the dispatcher, short sums", flush=True)
    w1, w2, w3, x, d_y = (t.to(dev) for t in _inputs(2, 256, 128, [150, 140], 0, 9, False))
    n = torch.tensor([150, 140], device=dev)
    F_.register_region_ops()
    for short in (False, True):
        e = F_.quantize_experts(w1, w2, w3, short_sums=short)
        want = F_.bmm_experts_fp8(e, x, n)
        tensors = (*e[:12], x, n)
        assert torch.equal(want, torch.ops.piper_amd.bmm_experts_fp8(*tensors, short))
        if not short:
            assert torch.equal(want, torch.ops.piper_amd.bmm_experts_fp8(*tensors))
        rows = x.clone().requires_grad_(True)
        got = torch.ops.piper_amd.bmm_experts_fp8(*e[:12], rows, n, short_sums=short)
        assert torch.equal(want, got)
        again = x.clone().requires_grad_(True)
        assert torch.equal(torch.autograd.grad(got, rows, d_y)[0], torch.autograd.grad(F_.bmm_experts_fp8(e, again, n), again, d_y)[0])

    @torch.compile(backend="eager", fullgraph=True)
    def compiled(x):
        return F_.bmm_experts_fp8(e, x, n)

    assert torch.equal(compiled(x), want)
