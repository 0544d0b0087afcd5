"""FusedMuon on the GPU: by itself, over a bucket, saved and loaded, in a graph, and as the optimizer of a layer with a balance loss.

Weights of one step: the update's error (tests/test_gpu_orthogonalize.py) times the step, and a rounding of the weight; several steps add
their errors up, and an update's input differs by the steps before, so each step is compared from the state it began with."""
import copy
import io

import pytest
import torch

from oracle import bucket as OB
from oracle import orthogonalize as O
from piper_amd import functional as F_, ops
from piper_amd.bucket import BucketState, ParamStorage, StageStore, flatten_params
from piper_amd.moe import AnnotatedMoE, MoEArgs
from piper_amd.optim import FusedMuon

pytestmark = pytest.mark.gpu
HYPER = dict(lr=0.01, momentum=0.9, weight_decay=0.1, adjust_lr="match_rms_adamw")
SHAPES = [(40, 96), (7,), (3, 64, 24), (130, 50), (33,), (1,), (2, 2, 16, 16)]


def make(shape, seed, dtype, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def off(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    return ((a - b).norm() / b.norm().clamp_min(1e-300)).item()


def check_matrix(w1, m1, w0, m0, g, **hyper):
    want_w, want_m = O.muon_step(w0.double().cpu(), m0.double().cpu(), g.double().cpu(), **hyper)
    plain_w, _ = O.muon_step(w0.float().cpu(), m0.float().cpu(), g.float().cpu(), **hyper)
    assert (m1.cpu().double() - want_m).abs().max() <= 2.0 ** -22 * max(m0.abs().max().item(), g.abs().max().item())
    rows, cols = w0.shape[-2:]
    step = hyper["lr"] * O.rate(rows, cols, hyper["adjust_lr"]) * (want_w.numel() / (rows * cols) * min(rows, cols)) ** 0.5
    assert off(w1, want_w) <= 2 * off(plain_w, want_w) + 2.0 ** -23 + 5 * 2.0 ** -22 * step / want_w.norm().item()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_parameters_by_themselves(dev, dtype):
    params = [torch.nn.Parameter(make(s, i, dtype).to(dev)) for i, s in enumerate(SHAPES)]
    opt = FusedMuon(params, adamw=dict(lr=0.002, betas=(0.8, 0.9), eps=1e-6, weight_decay=0.3), **HYPER)
    masters = [p.detach().float().clone() for p in params]
    firsts, seconds = ([torch.zeros_like(m) for m in masters] for _ in range(2))
    for step in range(1, 4):
        grads = [make(s, 100 * step + i, dtype, 1e-2).to(dev) for i, s in enumerate(SHAPES)]
        for p, g in zip(params, grads):
            p.grad = g
        opt.step()
        for p, g, w0, m0, v0 in zip(params, grads, masters, firsts, seconds):
            st = opt.state[p]
            if p.dim() >= 2:
                check_matrix(st["master"].view(p.shape), st["momentum"].view(p.shape), w0, m0, g, **HYPER)
            else:
                want, m, v = OB.adamw_step_torch(w0.cpu(), g.float().cpu(), m0.cpu(), v0.cpu(), step, 0.002, (0.8, 0.9), 1e-6, 0.3)
                assert (st["master"].cpu() - want).abs().max() <= 1e-6 and (st["momentum"].cpu() - m).abs().max() <= 1e-8
                v0.copy_(st["exp_avg_sq"][:p.numel()])
            assert st["step"] == step and torch.equal(p.detach().reshape(-1), st["master"].to(dtype))
            w0.copy_(st["master"].view(p.shape))
            m0.copy_(st["momentum"].view(p.shape))


def a_bucket(dev, dtype, align=256, **kw):
    params = [torch.nn.Parameter(make(s, i, dtype).to(dev)) for i, s in enumerate(SHAPES)]
    bucket = flatten_params(BucketState(), params, optim_class=lambda ps: FusedMuon(ps, **HYPER, **kw), align_bytes=align)
    store = StageStore(buckets={0: bucket}, zero_managed_ubids={0})
    return params, bucket, ParamStorage(store)


def put_grads(params, seed, dev, missing=()):
    for i, p in enumerate(params):
        p.grad = None if i in missing else make(p.shape, seed + i, p.dtype, 1e-2).to(dev)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("align", [256, 1])
@pytest.mark.parametrize("zero", [False, True])
def test_bucket_packed_and_held(dev, dtype, align, zero):
    """Two microbatches; the second one's gradients packed too, or held for the step: the same bits, and the definition's."""
    got = []
    for hold in (False, True):
        params, bucket, storage = a_bucket(dev, dtype, align, zero_grad_in_step=zero)
        opt = bucket.shard_optimizer
        for step in range(2):
            if not zero or step == 0:
                storage.zero_grad_buffers()
            before = copy.deepcopy(opt.state[bucket.shard_param]) if opt.state.get(bucket.shard_param) else None
            put_grads(params, 1000 * step, dev, missing=(3,))
            storage.accumulate_zero_param_grads_to_flat(0)
            put_grads(params, 1000 * step + 500, dev, missing=(4,))
            (storage.hold_param_grads if hold else storage.accumulate_zero_param_grads_to_flat)(0)
            flat = bucket.flat_grads.clone()
            w0 = torch.cat([p.detach().reshape(-1) for p in params])
            storage.step_zero_shard_optimizers()
            if zero:
                assert not any(bucket.flat_grads[o:o + n].any() for _, o, n, _ in bucket.param_view_specs)
            else:
                assert torch.equal(bucket.flat_grads, flat)
            st = opt.state[bucket.shard_param]
            if not hold and before is not None:
                for _, o, n, s in bucket.param_view_specs:
                    if len(s) >= 2:
                        cut = lambda t: t[o:o + n].view(s)  # noqa: E731
                        check_matrix(cut(st["master"]), cut(st["momentum"]), cut(before["master"]), cut(before["momentum"]), cut(flat), **HYPER)
            for p, o, n, s in bucket.param_view_specs:
                assert torch.equal(p.detach().reshape(-1), st["master"][o:o + n].to(dtype))
            assert not torch.equal(w0, torch.cat([p.detach().reshape(-1) for p in params]))
        got.append((bucket.flat_params.clone(), *(st[k].clone() for k in ("master", "momentum", "exp_avg_sq"))))
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_saved_and_loaded_state_continues_bit_for_bit(dev, dtype):
    params, bucket, storage = a_bucket(dev, dtype)
    for step in range(4):
        if step == 2:
            file = io.BytesIO()
            torch.save((bucket.flat_params, bucket.shard_optimizer.state_dict()), file)
        storage.zero_grad_buffers()
        put_grads(params, 10 * step, dev)
        storage.accumulate_zero_param_grads_to_flat(0)
        storage.step_zero_shard_optimizers()
    file.seek(0)
    flat, saved = torch.load(file, weights_only=True)
    params2, bucket2, storage2 = a_bucket(dev, dtype)
    with torch.no_grad():
        bucket2.flat_params.copy_(flat)
    bucket2.shard_optimizer.load_state_dict(saved)
    for step in (2, 3):
        storage2.zero_grad_buffers()
        put_grads(params2, 10 * step, dev)
        storage2.accumulate_zero_param_grads_to_flat(0)
        storage2.step_zero_shard_optimizers()
    assert torch.equal(bucket.flat_params, bucket2.flat_params)
    a, b = bucket.shard_optimizer.state[bucket.shard_param], bucket2.shard_optimizer.state[bucket2.shard_param]
    assert all(torch.equal(a[k], b[k]) for k in ("master", "momentum", "exp_avg_sq")) and a["step"] == b["step"] == 4


def test_more_shapes_than_a_launch_takes(dev):
    """Ninety matrices of thirty shapes, an empty one among them: each as by itself."""
    shapes = [(17 + 5 * (i % 30), 130 - 4 * (i % 30)) for i in range(90)]
    shapes[50] = (0, 8)
    w, m, g = ([make(s, k + i, torch.float32, 0.1).to(dev) for i, s in enumerate(shapes)] for k in (0, 200, 400))
    alone = []
    for a, b, c in zip(w, m, g):
        a, b = a.clone(), b.clone()
        ops.muon_fused([a], [b], [c], lr=0.1)
        alone.append((a, b))
    ops.muon_fused(w, m, g, lr=0.1)
    for (a, b), x, y in zip(alone, w, m):
        assert torch.equal(a, x) and torch.equal(b, y)


@pytest.mark.parametrize("half", [False, True])
def test_streams_and_a_graph(dev, half):
    shapes = [(4, 200, 150), (129, 257)]
    fresh = lambda: ([make(s, i, torch.float32).to(dev) for i, s in enumerate(shapes)], [torch.zeros(s, device=dev) for s in shapes],  # noqa: E731
                     [torch.zeros(s, dtype=torch.bfloat16, device=dev) for s in shapes])
    grads = [[make(s, 10 * k + i, torch.bfloat16, 1e-2).to(dev) for i, s in enumerate(shapes)] for k in range(4)]
    w, m, sh = fresh()
    for g in grads:
        ops.muon_fused(w, m, g, shadows=sh, lr=0.1, half_products=half)
    side = torch.cuda.Stream()
    w2, m2, sh2 = fresh()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for g in grads:
            ops.muon_fused(w2, m2, g, shadows=sh2, lr=0.1, half_products=half)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(w + m + sh, w2 + m2 + sh2))
    w3, m3, sh3 = fresh()
    fixed = [torch.zeros_like(g) for g in grads[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.muon_fused(w3, m3, fixed, shadows=sh3, lr=0.1, half_products=half)
    for g in grads:
        for a, b in zip(fixed, g):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        ops.orthogonalize(fixed[0])       # other work between the replays
    assert all(torch.equal(a, b) for a, b in zip(w + m + sh, w3 + m3 + sh3))


def test_a_gradient_that_is_not_finite_reaches_its_own_matrix_only(dev):
    w, m, g = ([make(s, k, torch.float32).to(dev) for s in [(5, 40, 60), (70, 70)]] for k in (0, 1, 2))
    w1, m1 = [t.clone() for t in w], [t.clone() for t in m]
    ops.muon_fused(w1, m1, g, lr=0.1)
    g[0][2, 3, 4] = float("inf")
    ops.muon_fused(w, m, g, lr=0.1)
    assert w[0][2].isnan().all()
    for e in (0, 1, 3, 4):
        assert torch.equal(w[0][e], w1[0][e])
    assert torch.equal(w[1], w1[1])


def test_refusals(dev):
    w, m, g = (torch.zeros(4, 6, device=dev) for _ in range(3))
    for bad in (dict(masters=[w.bfloat16()]), dict(masters=[w[0]]), dict(masters=[w.t()]), dict(momenta=[m[:2]]), dict(grads=[g[:2]]), dict(flat_grads=[g.bfloat16()]),
                dict(shadows=[w]), dict(grads=[g, g]), dict(momenta=[m.cpu()])):
        args = dict(masters=[w], momenta=[m], grads=[g]) | bad
        with pytest.raises(ValueError):
            ops.muon_fused(args.pop("masters"), args.pop("momenta"), args.pop("grads"), lr=0.1, **args)
    with pytest.raises(TypeError):
        ops.muon_fused([w], [m], [g.double()], lr=0.1)
    with pytest.raises(TypeError):
        ops.orthogonalize(w.double())
    with pytest.raises(ValueError, match="dimensions"):
        ops.orthogonalize(w[0])
    with pytest.raises(ValueError, match="32768"):
        ops.orthogonalize(torch.empty(1, 32769, device=dev))
    with pytest.raises(ValueError, match="eps"):
        ops.orthogonalize(w, eps=0.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_layer_trained_with_both(dev, dtype):
    """The balance loss and the Muon step together, as a stage uses them: forward, backward into a bucket, step; the router's gate,
    fp32 in a bucket of its own, by AdamW."""
    moe = AnnotatedMoE(MoEArgs(num_experts=8, top_k=2, route_norm=True, balance_loss_coeff=0.1), 64, 48, dtype=dtype).to(dev)
    moe.init_weights(std=0.1, generator=torch.Generator(device=dev).manual_seed(0))
    gate = moe.router.gate.weight
    flatten = lambda ps: flatten_params(BucketState(), ps, optim_class=lambda q: FusedMuon(q, matrices=lambda p: p is not gate, **HYPER))  # noqa: E731
    experts, router = flatten([moe.experts.w1, moe.experts.w2, moe.experts.w3]), flatten([gate])
    experts.companions = [router]
    storage = ParamStorage(StageStore(buckets={0: experts}, zero_managed_ubids={0}))
    gen = torch.Generator(device=dev).manual_seed(1)
    losses = []
    for step in range(3):
        storage.zero_grad_buffers()
        for mb in range(2):
            x, d = (torch.randn(2, 32, 64, device=dev, generator=gen).to(dtype) for _ in range(2))
            with F_.accumulate_weight_grads():
                moe(x).backward(d * 1e-2)
            assert moe.tokens_per_expert.shape == (8,) and int(moe.tokens_per_expert.sum()) == 128
            (storage.accumulate_zero_param_grads_to_flat if mb == 0 else storage.hold_param_grads)(0)
        w0 = experts.flat_params.clone()
        storage.step_zero_shard_optimizers()
        losses.append(moe.balance_loss.item())
        assert not torch.equal(w0, experts.flat_params) and experts.flat_params.isfinite().all() and router.flat_params.isfinite().all()
        assert gate.grad is None and moe.experts.w1.grad is None
    assert all(0 < v < 10 for v in losses)
    assert experts.shard_optimizer.state[experts.shard_param]["exp_avg_sq"].numel() == 0
    assert router.shard_optimizer.state[router.shard_param]["exp_avg_sq"].numel() == gate.numel()


def test_a_tensor_given_twice_is_refused(dev):
    w, m, g = (torch.zeros(3, 4, 6, device=dev) for _ in range(3))
    sh = torch.zeros(4, 6, dtype=torch.bfloat16, device=dev)
    for args in (dict(masters=[w[0], w[0]]), dict(momenta=[m[1], m[1]]), dict(momenta=[m[0], w[1]]), dict(shadows=[sh, sh]), dict(flat_grads=[g[0], g[0]], zero_grad=True),
                 dict(masters=[w.view(-1)[:24].view(4, 6), w.view(-1)[20:44].view(4, 6)])):
        args = dict(masters=[w[0], w[1]], momenta=[m[0], m[1]], grads=[g[0], g[0]]) | args
        with pytest.raises(ValueError, match="overlap"):
            ops.muon_fused(args.pop("masters"), args.pop("momenta"), args.pop("grads"), lr=0.1, **args)
    ops.muon_fused([w[0], w[1], w[2, :0]], [m[0], m[1], m[2, :0]], [g[0], g[0], None], flat_grads=[g[2], g[2], None], lr=0.1)      # read, not written
