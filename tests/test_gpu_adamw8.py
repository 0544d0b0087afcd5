"""AdamW with 8-bit moments: every step against oracle/blocks.py in 64 bits with the bounds that fp32 arithmetic allows, the packed
form bit for bit against pack + step, and the optimizer around them."""
import math

import pytest
import torch

from oracle import blocks as B
from piper_amd import ops
from piper_amd.bucket import BucketState, ParamStorage, StageStore, flatten_params
from piper_amd.optim import FusedAdamW

pytestmark = pytest.mark.gpu

HOW = dict(lr=1e-2, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1)
U, TINY = 2.0 ** -24, 2.0 ** -150


def _bytes(moments):
    return [t.view(torch.uint8).cpu() for t in moments]


def _decoded(code, scale):
    # a byte of 0 stands for 0 (moments that have not been stepped yet)
    e = scale.view(torch.uint8).cpu().to(torch.int64)
    s = torch.where(e == 0, torch.zeros(e.shape, dtype=torch.float64), B.two_to(e - 127)).repeat_interleave(64)[:code.numel()]
    return code.cpu().double() * s


def _moment_between(name, code, scale, value, err, random16, mantissa):
    """The stored moment is what the format makes of some number within err of value."""
    stored = _decoded(code, scale)
    lo, hi = value - err, value + err
    if mantissa == 2:
        lo = lo.clamp(min=0)
    options = []
    for t in (value, lo, hi):      # the scale follows the block's largest value, which may be any of these
        v, k = B.encode(t, random16, mantissa)
        options.append(v * B.two_to(k).repeat_interleave(64)[:v.numel()])
    o = torch.stack(options)
    least, most = o.amin(0), o.amax(0)
    assert ((stored >= least) & (stored <= most)).all(), f"{name}: {((stored < least) | (stored > most)).sum().item()} of {stored.numel()} differ"
    return (least == most).double().mean().item()


def _step_and_check(p, m8, g, step, seed, shadow=None, n=None, **more):
    """One step of adamw8_fused against the oracle, from the state as it is."""
    n = p.numel()
    p0, m0, v0 = p.cpu().double(), _decoded(m8[0], m8[1]), _decoded(m8[2], m8[3])
    gs = g.cpu().double() * more.get("grad_scale", 1.0)
    ops.adamw8_fused(p, *m8, g, step=step, seed=seed, shadow=shadow, **HOW, **more)
    want, m, v = B.adamw8_step(p0, gs, m0, v0, step, **HOW)
    # m: a difference, a product, a sum (and the gradient's scaling); v: two products of g, one of v, a sum
    # and each of them by half of the smallest subnormal number where it falls below the normal ones
    # (zeros are exact)
    me = 4 * U * (m0.abs() + gs.abs()) + 4 * TINY * ((m0 != 0) | (gs != 0))
    ve = 5 * U * v + 4 * TINY * (v > 0)
    denom = torch.sqrt(v / (1 - HOW["beta2"] ** step)) + HOW["eps"]
    update = HOW["lr"] / (1 - HOW["beta1"] ** step) / denom
    tol = 3 * U * want.abs().clamp(min=1e-30) + U * p0.abs() + update * (me + 8 * U * m.abs() + 3 * U * gs.abs())
    assert ((p.cpu().double() - want).abs() <= tol).all()
    if shadow is not None:
        assert torch.equal(shadow.cpu(), p.cpu().to(shadow.dtype))
    bits = B.random_bits(n, seed)
    sure = [_moment_between("exp_avg", m8[0], m8[1], m, me, bits >> 16, 3), _moment_between("exp_avg_sq", m8[2], m8[3], v, ve, bits & 0xFFFF, 2)]
    assert n < 1000 or min(sure) > 0.99      # almost everywhere the bounds leave one code


@pytest.mark.parametrize("n", [1, 3, 63, 64, 65, 1000, 1024, 1025, 5000])
def test_steps_follow_the_definition(dev, n):
    print(f"[case] adamw8 flat n={n}", flush=True)
    g = torch.Generator().manual_seed(n)
    p = torch.randn(n, generator=g).to(dev)
    shadow = torch.empty(n, dtype=torch.bfloat16, device=dev)
    m8 = ops.adamw8_state(n, dev)
    for step in range(1, 7):
        grad = torch.randn(n, generator=g) * (1e-3 if step != 3 else 1e-12) * (torch.rand(n, generator=g) < 0.9)
        if step == 4:
            grad[: n // 2] *= 1e4
        grad = grad.to(dev)
        _step_and_check(p, m8, grad, step, 977 * step, shadow if step % 2 else None, grad_scale=0.5 if step == 5 else 1.0)
        kept = grad.clone()
        if step == 6:
            ops.adamw8_fused(p, *m8, grad, step=7, seed=1, zero_grad=True, **HOW)
            assert (grad == 0).all() and (kept != 0).any() | (n == 1)


def test_wide_and_tiny_magnitudes(dev):
    print("[case] adamw8 magnitudes", flush=True)
    n = 640
    scale = torch.tensor([1e-25, 1e-15, 1e-8, 1e-4, 1.0, 1e4, 1e10, 1e15, 0.0, 1e-3]).repeat_interleave(64)
    spread = torch.logspace(-9, 0, 64).repeat(10)           # nine decades inside a block
    g = torch.Generator().manual_seed(0)
    p, m8 = torch.randn(n, generator=g).to(dev), ops.adamw8_state(n, dev)
    for step in (1, 2, 3):
        grad = (torch.randn(n, generator=g) * scale * spread).to(dev)
        before = p.clone()
        _step_and_check(p, m8, grad, step, step)
        moved = (p - before * (1 - HOW["lr"] * HOW["weight_decay"])).abs()
        assert torch.isfinite(p).all() and moved.max() < 100 * HOW["lr"]      # no division by a second moment that was lost


def test_moments_that_are_not_finite_stay_alone(dev):
    print("[case] adamw8 NaN and infinity", flush=True)
    n = 256
    g = torch.Generator().manual_seed(1)
    grad = torch.randn(n, generator=g)
    bad = grad.clone()
    bad[5], bad[70], bad[200] = math.nan, math.inf, -math.inf
    p0 = torch.randn(n, generator=g)
    out = []
    for gr in (grad, bad):
        p, m8 = p0.to(dev), ops.adamw8_state(n, dev)
        # the three do not count for their blocks' scales; without them there neither
        gr = gr.clone()
        if gr is not bad and not torch.isnan(gr).any():
            gr[[5, 70, 200]] = 0.0
        ops.adamw8_fused(p, *m8, gr.to(dev), step=1, seed=3, **HOW)
        out.append((p.cpu(), *_bytes(m8)))
    keep = torch.ones(n, dtype=torch.bool)
    keep[[5, 70, 200]] = False
    for i in (0, 1, 3):
        assert torch.equal(out[0][i][keep], out[1][i][keep])
    assert torch.equal(out[0][2], out[1][2]) and torch.equal(out[0][4], out[1][4])
    assert torch.isnan(out[1][0][5]) and (out[1][1][~keep] & 0x7F == 0x7F).all() and (out[1][3][~keep] == 0x7F).all()


def test_stored_averages_keep_their_means(dev):
    """A constant second moment decays, and a constant gradient is approached, as in exact arithmetic: over n elements the mean stays
    within five deviations of a walk whose steps are at most half a step of the format to either side, weighted as the average does."""
    print("[case] adamw8 means", flush=True)
    n, steps, beta2 = 64 * 1024, 40, 0.99
    for first, then in ((1e-2, 0.0), (0.0, 1e-3)):
        p, m8 = torch.zeros(n, device=dev), ops.adamw8_state(n, dev)
        want = 0.0
        for step in range(1, steps + 1):
            value = first if step == 1 else then
            # not all of a block alike, or every value would be the block's largest: half of them a third of the others
            g = torch.full((n,), value, device=dev)
            g[::2] /= 3
            ops.adamw8_fused(p, *m8, g, step=step, seed=step * 7919, **dict(HOW, lr=0.0, beta2=beta2))
            want = beta2 * want + (1 - beta2) * value ** 2
        v = _decoded(m8[2], m8[3])[1::2]
        deviation = want * 0.25 / 2 * math.sqrt(steps / v.numel())
        assert abs(v.mean().item() - want) < 5 * deviation
        assert v.std() > 0                                  # and they are not all the same code


def _bucket(shapes, esize, seed, dev, dtype):
    g = torch.Generator().manual_seed(seed)
    offs, total = ops.bucket_plan([math.prod(s) for s in shapes], esize, 256)
    p = torch.zeros(total)
    grads = []
    for s, o in zip(shapes, offs):
        k = math.prod(s)
        p[o:o + k] = torch.randn(k, generator=g)
        grads.append((torch.randn(s, generator=g) * 1e-3).to(dtype).to(dev))
    return p.to(dev), offs, [math.prod(s) for s in shapes], grads


SHAPES = [(3, 5), (1024,), (1,), (777, 13), (64,), (2, 4100), (63,), (0,), (129,)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("flat", ["none", "kept", "cleared"])
def test_packed_is_pack_and_step_bit_for_bit(dev, dtype, flat):
    print(f"[case] adamw8 packed {dtype} flat={flat}", flush=True)
    p, offs, nums, grads = _bucket(SHAPES, 2 if dtype == torch.bfloat16 else 4, 2, dev, dtype)
    # a gradient that no 16-byte piece starts at, a strided one, one that is missing
    grads[1] = torch.cat([grads[1][:1], grads[1]])[1:]
    grads[3] = grads[3].t().contiguous().t()
    grads[5] = None
    n = p.numel()
    sides = []
    for packed in (True, False):
        q, m8 = p.clone(), ops.adamw8_state(n, dev)
        shadow = q.to(torch.bfloat16)
        for step in (1, 2, 3):
            fg = torch.zeros(n, device=dev)
            if flat != "none":
                ops.bucket_pack([None if g is None else g * 2 for g in grads], offs, fg, accumulate=True)
            before = fg.clone()
            how = dict(HOW, step=step, seed=step, shadow=shadow if step < 3 else None)
            if packed:
                ops.adamw8_fused_packed(q, *m8, None if flat == "none" else fg, grads, offs, nums, zero_grad=flat == "cleared", **how)
                assert torch.equal(fg, torch.zeros_like(fg) if flat == "cleared" else before)
            else:
                ops.bucket_pack(grads, offs, fg, accumulate=True, numels=nums)
                ops.adamw8_fused(q, *m8, fg, **how)
        sides.append((q, shadow, *m8))
    for i, (a, b) in enumerate(zip(*sides)):
        a, b = (t.view(torch.uint8) if t.element_size() == 1 else t for t in (a, b))
        if i in (3, 5):      # the scale of a block of padding alone: stored by the flat step only
            live = torch.zeros(a.numel(), dtype=torch.bool, device=dev)
            for o, k in zip(offs, nums):
                live[o // 64:(o + k + 63) // 64] = True
            a, b = a[live], b[live]
        assert torch.equal(a, b), i


def test_many_tensors_and_empty_calls(dev):
    print("[case] adamw8 packed 300 tensors", flush=True)
    shapes = [(17 + 3 * i,) for i in range(300)]
    p, offs, nums, grads = _bucket(shapes, 2, 5, dev, torch.bfloat16)
    q, m8 = p.clone(), ops.adamw8_state(p.numel(), dev)
    ops.adamw8_fused_packed(q, *m8, None, grads, offs, nums, step=1, seed=1, **HOW)
    r, w8 = p.clone(), ops.adamw8_state(p.numel(), dev)
    flat = torch.zeros_like(p)
    ops.bucket_pack(grads, offs, flat, accumulate=True)
    ops.adamw8_fused(r, *w8, flat, step=1, seed=1, **HOW)
    assert torch.equal(q, r)
    ops.adamw8_fused_packed(q, *m8, None, [], [], [], step=2, seed=1, **HOW)
    ops.adamw8_fused(q[:0], *ops.adamw8_state(0, dev), flat[:0], step=1, seed=1, **HOW)
    assert torch.equal(q, r)


def test_elements_behind_the_32_bit_border(dev):
    """A bucket whose last tensor starts behind 2^32 bytes of codes' worth of elements would not fit a test; 2^31 elements (2^33 bytes
    of masters) already pass every 32-bit offset in bytes and the sign of one in elements."""
    n = 2 ** 31 + 192
    print(f"[case] adamw8 with {n} elements", flush=True)
    if torch.cuda.mem_get_info()[0] < 40e9:
        pytest.skip("needs 40 GB")
    p = torch.zeros(n, device=dev)
    m8 = ops.adamw8_state(n, dev)
    tail = torch.randn(150, generator=torch.Generator().manual_seed(0))
    p[n - 192:n - 42] = tail.to(dev)
    grad = (tail * 1e-3).flip(0).to(dev)
    ops.adamw8_fused_packed(p, *m8, None, [grad], [n - 192], [150], step=1, seed=11, **HOW)
    q, w8 = tail.double(), None
    want, m, v = B.adamw8_step(q, grad.cpu(), torch.zeros(150), torch.zeros(150), 1, **HOW)
    assert torch.allclose(p[n - 192:n - 42].cpu().double(), want, rtol=1e-5, atol=1e-7) and (p[:100] == 0).all() and (p[n - 42:] == 0).all()
    stored = [t[n - 192:n - 42] if t.numel() == n else t[(n - 192) // 64:] for t in m8]
    bits = B.random_bits(150, 11, n - 192)
    _moment_between("exp_avg", stored[0], stored[1], m, 4 * U * grad.cpu().double().abs(), bits >> 16, 3)
    _moment_between("exp_avg_sq", stored[2], stored[3], v, 5 * U * v, bits & 0xFFFF, 2)


def test_optimizer_with_8_bit_states(dev):
    print("[case] FusedAdamW(state_bits=8) over a ZeRO bucket", flush=True)
    g = torch.Generator().manual_seed(3)
    shapes = [(40, 30), (130,), (7, 9)]
    init = [torch.randn(s, generator=g).bfloat16() for s in shapes]
    grads = [[(torch.randn(s, generator=g) * 1e-2).bfloat16() for s in shapes] for _ in range(6)]
    results = []
    for hold in (False, True):
        params = [torch.nn.Parameter(t.clone().to(dev)) for t in init]
        bucket = flatten_params(BucketState(), params, optim_class=lambda ps: FusedAdamW(ps, lr=1e-2, state_bits=8, seed=5))
        store = StageStore()
        store.buckets[0] = bucket
        store.zero_managed_ubids.add(0)
        storage = ParamStorage(store)
        for it in range(3):
            storage.zero_grad_buffers()
            for mb in range(2):
                for p, t in zip(params, grads[2 * it + mb]):
                    p.grad = t.to(dev)
                if hold and mb == 1:
                    storage.hold_param_grads(0)
                else:
                    storage.accumulate_zero_param_grads_to_flat(0)
            storage.step_zero_shard_optimizers()
        st = bucket.shard_optimizer.state[bucket.shard_param]
        assert st["exp_avg"].dtype == torch.float8_e4m3fn and st["step"] == 3
        results.append(([p.detach().clone() for p in params], _bytes(st[k] for k in ("exp_avg", "exp_avg_sq"))))
    for a, b in zip(results[0][0] + results[0][1], results[1][0] + results[1][1]):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_saved_and_loaded_state_continues_bit_for_bit(dev, dtype):
    print(f"[case] FusedAdamW(state_bits=8) state_dict {dtype}", flush=True)
    g = torch.Generator().manual_seed(4)
    start = torch.randn(300, generator=g).to(dtype)
    steps = [torch.randn(300, generator=g).to(dtype).to(dev) for _ in range(4)]
    p = torch.nn.Parameter(start.to(dev))
    opt = FusedAdamW([p], state_bits=8, seed=9)
    for i, gr in enumerate(steps):
        if i == 2:
            saved, copy = opt.state_dict(), torch.nn.Parameter(p.detach().clone())
            import copy as c
            saved = c.deepcopy(saved)
        p.grad = gr
        opt.step()
    other = FusedAdamW([copy], state_bits=8)
    other.load_state_dict(saved)
    for gr in steps[2:]:
        copy.grad = gr
        other.step()
    assert torch.equal(p, copy)
    for k in ("exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_scale"):
        assert torch.equal(opt.state[p][k].view(torch.uint8), other.state[copy][k].view(torch.uint8))
    with pytest.raises(ValueError, match="8-bit moments"):
        q = torch.nn.Parameter(start.to(dev))
        full = FusedAdamW([q])
        q.grad = steps[0]
        full.step()
        FusedAdamW([torch.nn.Parameter(start.to(dev))], state_bits=8).load_state_dict(full.state_dict())


def test_unaligned_bucket_takes_the_packed_gradients_all_the_same(dev):
    print("[case] FusedAdamW(state_bits=8) without aligned starts", flush=True)
    g = torch.Generator().manual_seed(6)
    n, offs, nums = 150, [0, 50], [50, 100]
    grads = [torch.randn(k, generator=g).to(dev) for k in nums]
    sides = []
    for packed in (True, False):
        p = torch.nn.Parameter(torch.randn(n, generator=torch.Generator().manual_seed(7)).to(dev))
        opt = FusedAdamW([p], state_bits=8)
        if packed:
            opt.step_packed(p, grads, offs, nums)
        else:
            p.grad = torch.cat(grads)
            opt.step()
        sides.append(p.detach())
    assert torch.equal(*sides)


def test_captured_and_replayed(dev):
    print("[case] adamw8 in a graph", flush=True)
    n = 3000
    g = torch.Generator().manual_seed(8)
    p0 = torch.randn(n, generator=g).to(dev)
    p, m8, grad = p0.clone(), ops.adamw8_state(n, dev), torch.zeros(n, device=dev)
    how = dict(HOW, step=5, seed=3)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.adamw8_fused(p.clone(), *ops.adamw8_state(n, dev), grad, **how)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.adamw8_fused(p, *m8, grad, **how)
    q, w8 = p0.clone(), ops.adamw8_state(n, dev)
    for rep in range(4):
        grad.copy_(torch.randn(n, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        ops.adamw8_fused(q, *w8, grad, **how)
        assert torch.equal(p, q) and all(torch.equal(a, b) for a, b in zip(_bytes(m8), _bytes(w8))), rep


def test_refusals(dev):
    n = 128
    p, m8, g = torch.zeros(n, device=dev), ops.adamw8_state(n, dev), torch.zeros(n, device=dev)
    how = dict(HOW, step=1, seed=0)
    with pytest.raises(ValueError, match="e8m0 scale"):
        ops.adamw8_fused(p, m8[0], m8[1][:1], m8[2], m8[3], g, **how)
    with pytest.raises(ValueError, match="e8m0 scale"):
        ops.adamw8_fused(p, m8[2], m8[1], m8[0], m8[3], g, **how)
    with pytest.raises(ValueError, match="fp32 contiguous"):
        ops.adamw8_fused(p, *m8, g[:64], **how)
    with pytest.raises(RuntimeError, match="invalid argument"):
        ops.adamw8_fused(p, *m8, g, **dict(how, step=0))
    with pytest.raises(ValueError, match="multiples of 64"):
        ops.adamw8_fused_packed(p, *m8, None, [g[:10]], [32], [10], **how)
    with pytest.raises(ValueError, match="outside the bucket"):
        ops.adamw8_fused_packed(p, *m8, None, [g[:100]], [64], [100], **how)
    with pytest.raises(ValueError, match="none over another"):
        ops.adamw8_fused_packed(p, *m8, None, [g[:100], g[:10]], [0, 64], [100, 10], **how)
    with pytest.raises(ValueError, match="size differs"):
        ops.adamw8_fused_packed(p, *m8, None, [g[:100]], [0], [99], **how)
    with pytest.raises(TypeError, match="float32 and bfloat16"):
        ops.adamw8_fused_packed(p, *m8, None, [g[:10].half()], [0], [10], **how)
    with pytest.raises(ValueError, match="32 or 8"):
        FusedAdamW([torch.nn.Parameter(p)], state_bits=4)
