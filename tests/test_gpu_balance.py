"""The router's balance loss on the GPU against its definition in 64 bits: by itself, behind the router, inside the fused region and in the
module.

Tolerances.  An element of the gradient adds up products of a softmax, a table value and a factor.  A softmax in fp32 is off by half a
step (2^-24) of its exponent's argument, up to 16 here, and by a few more roundings: 2^-19 of the summands' magnitudes
(oracle.balance.gradient_scale) in all.  The loss is a mean of such softmaxes with positive weights: 2^-19 of itself."""
import pytest
import torch

from oracle import balance as O
from piper_amd import _lib, functional as F_, ops
from piper_amd.moe import AnnotatedMoE, MoEArgs, MoEFeedForwardBlock

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TOL = 2.0 ** -19


def inputs(T, E, K, seed, skew=0.0):
    gen = torch.Generator().manual_seed(seed)
    logits = torch.randn(T, E, generator=gen) - skew * torch.log(torch.arange(1, E + 1).float())
    return logits, torch.topk(logits, K, dim=1).indices.to(torch.int32)


def check(T, E, K, cb, cz, sequences, seed=0, skew=0.0, logits=None, idx=None, d_loss=1.7):
    if logits is None:
        logits, idx = inputs(T, E, K, seed, skew)
    x = logits.to(DEV).requires_grad_(True)
    off = None if sequences is None else torch.tensor(sequences, dtype=torch.int32, device=DEV)
    loss, counts = F_.balance_loss(x, idx.to(DEV), balance_coeff=cb, z_coeff=cz, sequences=off)
    d, = torch.autograd.grad(loss, x, torch.tensor(d_loss, device=DEV))
    e = logits.double().requires_grad_(True)
    want, want_counts = O.balance_loss(e, idx, cb, cz, sequences)
    want_d, = torch.autograd.grad(want, e, torch.tensor(d_loss, dtype=torch.float64))
    assert loss.dtype == torch.float32 and loss.shape == () and counts.dtype == torch.int32 and not counts.requires_grad
    assert torch.equal(counts.cpu().long(), want_counts if sequences is not None else want_counts[0])
    assert abs(loss.item() - want.item()) <= TOL * abs(want.item())
    scale = O.gradient_scale(logits, want_counts, K, cb, cz, sequences) * abs(d_loss)
    assert ((d.cpu().double() - want_d).abs() <= TOL * scale + 1e-30).all()
    return d


@pytest.mark.parametrize("E,K", [(1, 1), (2, 1), (7, 3), (8, 2), (9, 2), (16, 4), (17, 4), (32, 8), (33, 8), (60, 4), (64, 8), (65, 8), (128, 8), (129, 8),
                                 (256, 8), (300, 8), (1000, 16), (1024, 64)])
@pytest.mark.parametrize("T", [1, 63, 200])
def test_sizes(T, E, K):
    check(T, E, K, 1.0, 1e-3, None, seed=E)


@pytest.mark.parametrize("sequences", [[0, 300], [0, 0, 300, 300], [0, 1, 2, 3, 300], [5, 64, 64, 128, 129, 290], [40, 40, 40], [0, 63, 64, 65, 127, 128, 191, 257],
                                       [299, 300], list(range(0, 301, 2))])
@pytest.mark.parametrize("E,K", [(8, 2), (20, 3), (128, 8)])
def test_sequences(sequences, E, K):
    """Empty ones, single tokens, bounds beside a chunk's, tokens in front of the first and behind the last one."""
    d = check(300, E, K, 0.5, 1e-2, sequences, skew=1.0)
    assert not d[:sequences[0]].any() and not d[sequences[-1]:].any()


@pytest.mark.parametrize("T,E,K,S", [(40000, 60, 4, 61), (33000, 128, 8, 1), (70001, 8, 2, 700)])
def test_long_inputs(T, E, K, S):
    """More than one piece of 64 tokens to a chunk."""
    gen = torch.Generator().manual_seed(1)
    cuts = sorted(torch.randint(0, T - 100, (S - 1,), generator=gen).tolist())
    check(T, E, K, 1.0, 1e-3, [0, *cuts, T - 100], seed=2, skew=1.0)


def test_coefficients_and_no_tokens():
    for cb, cz in ((0.0, 1.0), (1.0, 0.0), (0.0, 0.0), (-0.5, 2.0)):
        check(100, 12, 3, cb, cz, None)
    loss, counts = F_.balance_loss(torch.empty(0, 8, device=DEV), torch.empty(0, 2, dtype=torch.int32, device=DEV))
    assert loss.item() == 0 and counts.tolist() == [0] * 8
    x = torch.empty(0, 8, device=DEV, requires_grad=True)
    loss, _ = F_.balance_loss(x, torch.empty(0, 2, dtype=torch.int32, device=DEV))
    assert torch.autograd.grad(loss, x)[0].shape == (0, 8)


def test_balanced_choices_have_no_gradient_at_all():
    """All experts chosen equally often: exactly zero, not what is left of cancelled sums."""
    logits, _ = inputs(64, 4, 1, 3)
    idx = (torch.arange(64) % 4).to(torch.int32).view(64, 1)
    x = logits.to(DEV).requires_grad_(True)
    loss, counts = F_.balance_loss(x, idx.to(DEV))
    assert counts.tolist() == [16] * 4 and not torch.autograd.grad(loss, x)[0].any()
    check(640, 4, 1, 1.0, 0.0, None, logits=logits.repeat(10, 1), idx=torch.cat([idx.repeat(9, 1), idx.clamp(max=2)]))     # nearly


def test_rows_that_are_masked_or_not_finite():
    """-inf logits are experts out of reach; a row that is not finite makes the loss so, and its own gradient."""
    logits, _ = inputs(130, 12, 2, 4)
    logits[:, 5] = float("-inf")
    logits[7, 1:] = float("-inf")
    idx = torch.topk(logits, 2, dim=1).indices.to(torch.int32)
    x = logits.to(DEV).requires_grad_(True)
    loss, counts = F_.balance_loss(x, idx.to(DEV), z_coeff=0.1)
    d, = torch.autograd.grad(loss, x)
    e = logits.double().requires_grad_(True)
    want, _ = O.balance_loss(e, idx, 1.0, 0.1)
    assert abs(loss.item() - want.item()) <= TOL * want.item()
    assert not d[:, 5].any() and not d.isnan().any()
    bad = logits.clone()
    bad[9] = float("nan")
    y = bad.to(DEV).requires_grad_(True)
    loss, _ = F_.balance_loss(y, idx.to(DEV), z_coeff=0.1)
    d2, = torch.autograd.grad(loss, y)
    rest = torch.arange(130) != 9
    assert loss.isnan() and d2[9].isnan().all() and torch.equal(d2[rest], d[rest])


def test_ids_out_of_range_are_not_counted():
    logits, idx = inputs(70, 6, 2, 5)
    idx[3, 0], idx[4, 1] = 6, -1
    _, counts = F_.balance_loss(logits.to(DEV), idx.to(DEV))
    keep = (idx >= 0) & (idx < 6)
    assert counts.cpu().tolist() == torch.bincount(idx[keep].long(), minlength=6).tolist()


def test_strides_streams_and_a_graph_with_its_backward():
    logits, idx = inputs(500, 24, 4, 6, 1.0)
    off = torch.tensor([0, 100, 333, 480], dtype=torch.int32, device=DEV)

    def run(x, i, o):
        loss, counts = F_.balance_loss(x, i, z_coeff=1e-2, sequences=o)
        d, = torch.autograd.grad(loss, x)
        return loss.detach(), counts, d

    x0, i0 = logits.to(DEV).requires_grad_(True), idx.to(DEV)
    want = run(x0, i0, off)
    wide = torch.zeros(500, 50, device=DEV)
    wide[:, 3:27] = logits.to(DEV)
    turned = i0.t().contiguous().t()
    both = torch.stack([off, off], 1)[:, 0]
    x1 = wide[:, 3:27].detach().requires_grad_(True)
    for a, b in zip(run(x1, turned, both), want):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(x0, i0, off)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del got
    # a capture with its backward (of a leaf that no eager graph holds), replayed with other inputs in between
    leaf, ids, at = logits.to(DEV).requires_grad_(True), i0.clone(), off.clone()
    with torch.cuda.stream(side):
        run(leaf, ids, at)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(leaf, ids, at)
    for seed in (6, 7, 6, 8):
        l2, i2 = inputs(500, 24, 4, seed, 1.0)
        with torch.no_grad():
            leaf.copy_(l2)
            ids.copy_(i2)
        graph.replay()
        torch.cuda.synchronize()
        eager = run(l2.to(DEV).requires_grad_(True), i2.to(DEV), off)
        for a, b in zip(out, eager):
            assert torch.equal(a, b)


def test_refusals():
    logits, idx = (t.to(DEV) for t in inputs(8, 4, 2, 0))
    for bad in (dict(logits=logits.double()), dict(logits=logits.bfloat16()), dict(logits=logits[0]), dict(top_idx=idx.long()), dict(top_idx=idx[:4]),
                dict(top_idx=idx[:, :0]), dict(sequences=torch.tensor([0, 8], device=DEV)), dict(sequences=torch.tensor([0], dtype=torch.int32, device=DEV)),
                dict(sequences=torch.tensor([0, 8], dtype=torch.int32))):
        args = dict(logits=logits, top_idx=idx) | bad
        with pytest.raises(ValueError):
            F_.balance_loss(args.pop("logits"), args.pop("top_idx"), **args)
    with pytest.raises(RuntimeError, match="shape"):
        F_.balance_loss(torch.zeros(2, 1025, device=DEV), torch.zeros(2, 1, dtype=torch.int32, device=DEV))


# ------------------------------------------------------------------------------------------------ with the router and the experts
def layer(T, H, E, I, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=gen)  # noqa: E731
    t = dict(x=r(T, H).to(dtype), w_gate=r(E, H) * 0.1, w1=(r(E, I, H) * 0.05).to(dtype), w2=(r(E, H, I) * 0.05).to(dtype), w3=(r(E, I, H) * 0.05).to(dtype))
    return {k: v.to(DEV).requires_grad_(True) for k, v in t.items()}, r(T, H).to(dtype).to(DEV)


def rel(a, b):
    a, b = a.double(), b.double()
    return ((a - b).abs().max() / b.abs().max().clamp_min(1e-30)).item()


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 1e-5), (torch.bfloat16, 2e-2)])
@pytest.mark.parametrize("T,H,E,I,K", [(300, 64, 8, 32, 2), (96, 128, 20, 64, 4), (1, 64, 8, 32, 2), (2048, 256, 16, 256, 4)])
@pytest.mark.parametrize("sequences", [None, "some"])
def test_region_is_the_region_and_the_loss(dtype, tol, T, H, E, I, K, sequences):
    """out as without the loss, bit for bit; the gradients are those of both by themselves, added."""
    t, d_out = layer(T, H, E, I, dtype, 9)
    off = None if sequences is None else torch.tensor([0, T // 3, T // 3, T - T // 5], dtype=torch.int32, device=DEV)
    kw = dict(top_k=K, route_norm=True, route_scale=1.5)
    args = (t["x"], t["w_gate"], None, t["w1"], t["w2"], t["w3"])
    d_loss = torch.tensor(300.0, device=DEV)
    out, loss, counts = F_.expert_region_balanced(*args, **kw, balance_coeff=0.5, z_coeff=0.02, sequences=off)
    got = torch.autograd.grad([out, loss], [v for v in t.values()], [d_out, d_loss])
    out0 = F_.expert_region(*args, **kw)
    plain = torch.autograd.grad(out0, [v for v in t.values()], d_out)
    assert torch.equal(out, out0)
    logits = ops.gate_logits(t["x"].detach(), t["w_gate"].detach()).requires_grad_(True)
    idx = ops.route_topk(logits.detach(), K, True, 1.5)[1]
    loss1, counts1 = F_.balance_loss(logits, idx, balance_coeff=0.5, z_coeff=0.02, sequences=off)
    assert torch.equal(counts, counts1) and torch.equal(loss, loss1)
    dl, = torch.autograd.grad(loss1, logits, d_loss)
    want = dict(zip(t, (p.double() for p in plain)))
    want["x"] += dl.double() @ t["w_gate"].detach().double()
    want["w_gate"] += dl.double().t() @ t["x"].detach().double()
    for (k, w), g in zip(want.items(), got):
        assert g.dtype == t[k].dtype and rel(g, w) <= tol, k
    # without the loss's gradient, and without the output's
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(F_.expert_region_balanced(*args, **kw, sequences=off)[0], list(t.values()), d_out), plain))
    alone = torch.autograd.grad(F_.expert_region_balanced(*args, **kw, balance_coeff=0.5, z_coeff=0.02, sequences=off)[1], [t["w_gate"], t["w1"]], d_loss)
    assert rel(alone[0], dl.double().t() @ t["x"].detach().double()) <= 1e-5 and not alone[1].any()
    with torch.no_grad():
        out2, loss2, counts2 = F_.expert_region_balanced(*args, **kw, balance_coeff=0.5, z_coeff=0.02, sequences=off)
    assert rel(out2, out) <= tol and torch.equal(loss2, loss) and torch.equal(counts2, counts)


def test_router_with_the_loss():
    t, _ = layer(200, 64, 12, 8, torch.bfloat16, 10)
    bias = torch.randn(12, device=DEV).requires_grad_(True)
    d_s = torch.randn(200, 3, device=DEV)
    leaves = [t["x"], t["w_gate"], bias]
    scores, idx, per_expert, loss, counts = F_.router_balanced(t["x"], t["w_gate"], bias, top_k=3, route_norm=True, balance_coeff=2.0, z_coeff=0.1)
    s0, i0, c0 = F_.router(t["x"], t["w_gate"], bias, top_k=3, route_norm=True)
    assert torch.equal(scores, s0) and torch.equal(idx, i0) and torch.equal(per_expert, c0) and torch.equal(counts, c0)
    got = torch.autograd.grad([scores, loss], leaves, [d_s, torch.tensor(3.0, device=DEV)])
    plain = torch.autograd.grad(s0, leaves, d_s)
    logits = ops.gate_logits(t["x"].detach(), t["w_gate"].detach(), bias.detach()).requires_grad_(True)
    l1, _ = F_.balance_loss(logits, idx, balance_coeff=2.0, z_coeff=0.1)
    dl, = torch.autograd.grad(l1, logits, torch.tensor(3.0, device=DEV))
    assert torch.equal(loss, l1)
    want = [dl.double() @ t["w_gate"].detach().double(), dl.double().t() @ t["x"].detach().double(), dl.double().sum(0)]
    for g, p, w, tol in zip(got, plain, want, (2e-2, 1e-5, 1e-5)):
        assert rel(g, p.double() + w) <= tol
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(F_.router_balanced(t["x"], t["w_gate"], bias, top_k=3, route_norm=True)[0], leaves, d_s), plain))


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("block", [False, True])
def test_module_trains_its_router_on_it(fused, block):
    """The loss's gradient arrives through the output alone; weight gradients may be put off and added up."""
    kw = dict(num_experts=8, top_k=2, route_norm=True)
    make = lambda **more: (MoEFeedForwardBlock if block else AnnotatedMoE)(MoEArgs(**kw, **more), 64, 32).to(DEV)  # noqa: E731
    plain, with_it = make(), make(balance_loss_coeff=0.5, router_z_loss_coeff=0.1)
    moe0, moe1 = (plain.moe, with_it.moe) if block else (plain, with_it)
    moe0.init_weights(std=0.1, generator=torch.Generator(device=DEV).manual_seed(0))
    with_it.load_state_dict(plain.state_dict())
    moe0.fused = moe1.fused = fused
    gen = torch.Generator(device=DEV).manual_seed(1)
    x, d = (torch.randn(2, 50, 64, device=DEV, generator=gen) for _ in range(2))
    off = torch.tensor([0, 50, 100], dtype=torch.int32, device=DEV)
    if block and not fused:
        plain, with_it = (lambda x, m=m, **k: x + m.moe(m.ffn_norm(x), **k) for m in (plain, with_it))
    a, b = plain(x), with_it(x, sequences=off)
    assert rel(a, b) <= 1e-6 and moe1.tokens_per_expert.shape == (2, 8) and int(moe1.tokens_per_expert.sum()) == 200
    a.backward(d)
    with F_.accumulate_weight_grads():
        b.backward(d)
    g0, g1 = moe0.router.gate.weight.grad, moe1.router.gate.weight.grad
    xn = F_.rmsnorm(x.reshape(-1, 64), with_it.ffn_norm.weight) if block and fused else None
    if not block:
        xn = x.reshape(-1, 64)
    if xn is not None:
        logits = ops.gate_logits(xn.detach(), moe1.router.gate.weight.detach()).requires_grad_(True)
        loss, _ = F_.balance_loss(logits, ops.route_topk(logits.detach(), 2, True)[1], balance_coeff=0.5, z_coeff=0.1, sequences=off)
        assert rel(moe1.balance_loss, loss.detach()) <= 1e-6 and not moe1.balance_loss.requires_grad
        dl, = torch.autograd.grad(loss, logits)
        assert rel(g1, g0.double() + dl.double().t() @ xn.detach().double()) <= 1e-5
    for n in ("w1", "w2", "w3"):
        assert rel(getattr(moe1.experts, n).grad, getattr(moe0.experts, n).grad) <= 1e-5
    if fused and not block:      # a second microbatch with the weight gradients put off
        first = g1.clone()
        with F_.defer_weight_grads() as queue:
            with_it(x, sequences=off).backward(d)
        assert torch.equal(moe1.router.gate.weight.grad, first)
        queue.run()
        assert rel(moe1.router.gate.weight.grad, 2 * first.double()) <= 1e-6


def test_through_the_dispatcher():
    t, d_out = layer(64, 64, 8, 32, torch.float32, 12)
    args = (t["x"], t["w_gate"], None, t["w1"], t["w2"], t["w3"])
    direct = F_.expert_region_balanced(*args, top_k=2, route_norm=True)
    op = torch.ops.piper_amd.expert_region_balanced(*args, 2, True, 1.0, None, None, 1.0, 0.0)
    assert all(torch.equal(a, b) for a, b in zip(op, direct))
    g = [torch.autograd.grad([r[0], r[1]], list(t.values()), [d_out, torch.ones((), device=DEV)]) for r in (direct, op)]
    assert all(torch.equal(a, b) for a, b in zip(*g))

    @torch.compile(fullgraph=True, backend="eager")
    def step(x, w):
        return F_.expert_region_balanced(x, w, None, t["w1"], t["w2"], t["w3"], top_k=2, route_norm=True)
    assert all(torch.equal(a, b) for a, b in zip(step(t["x"], t["w_gate"]), direct))


@pytest.mark.parametrize("E,K", [(200, 8), (300, 8), (600, 8)])
@pytest.mark.parametrize("S,T", [(3, 400), (150, 1500), (1025, 3000)])
def test_many_and_few_sequences_of_many_experts(E, K, S, T):
    """Five, three and one of a workgroup's sequences at once; ragged lengths, a third of them nothing, padding at both ends."""
    gen = torch.Generator().manual_seed(S + E)
    cuts = torch.randint(7, T - 7, (S + 1,), generator=gen)
    cuts[::3] = cuts[1::3][0]
    check(T, E, K, 1.0, 1e-3, sorted(cuts.tolist()), seed=S, skew=0.5)


def test_two_losses_at_once_and_a_captured_one():
    """On two streams at the same time, and in a graph that is replayed with other inputs between other work: the same bits each time."""
    cases = [(*inputs(2000, 60, 4, s, 0.5), torch.tensor([0, 100 + s, 700, 700, 1900], dtype=torch.int32)) for s in range(4)]

    def run(x, idx, off):
        loss, counts = F_.balance_loss(x, idx, z_coeff=1e-3, sequences=off)
        return loss.detach(), counts, torch.autograd.grad(loss, x)[0]
    on = [(x.to(DEV).requires_grad_(True), i.to(DEV), o.to(DEV)) for x, i, o in cases]
    want = [run(*c) for c in on]
    streams = [torch.cuda.Stream() for _ in on]
    got = [None] * len(on)
    for k, s in enumerate(streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got[k] = run(*on[k])
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    fixed = (torch.zeros_like(on[0][0]).requires_grad_(True), torch.zeros_like(on[0][1]), torch.zeros_like(on[0][2]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(*fixed)
    for c, w in zip(on, want):
        with torch.no_grad():
            for a, b in zip(fixed, c):
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, w))
        run(*c)
