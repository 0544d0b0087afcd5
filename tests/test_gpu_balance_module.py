"""The modules with a balance loss on the GPU: what a program does with their outputs, in training and without gradients.

Gradients of the gate: two sums of the same fp32 terms in different orders, 1e-5 of the largest (as tests/test_gpu_balance.py)."""
import pytest
import torch

from piper_amd import _lib, functional as F_, ops
from piper_amd.bucket import BucketState, ParamStorage, StageStore, flatten_params
from piper_amd.moe import AnnotatedMoE, MoEArgs, MoEFeedForwardBlock
from piper_amd.optim import FusedMuon

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ARGS = dict(num_experts=8, top_k=2, route_norm=True)
LOSS = dict(balance_loss_coeff=0.5, router_z_loss_coeff=0.1)


def rel(a, b):
    a, b = a.detach().double(), b.detach().double()
    return ((a - b).abs().max() / b.abs().max().clamp_min(1e-30)).item()


def pair(cls, dtype=None, seed=0, dims=(64, 32), **args):
    """The module without and with a balance loss, of the same weights."""
    args = ARGS | args
    plain, with_it = (cls(MoEArgs(**args, **more), *dims, dtype=dtype).to(DEV) for more in ({}, LOSS))
    moe = plain.moe if cls is MoEFeedForwardBlock else plain
    moe.init_weights(std=0.1, generator=torch.Generator(device=DEV).manual_seed(seed))
    with_it.load_state_dict(plain.state_dict())
    return plain, with_it


def tokens(*shape, seed=1, dtype=torch.float32):
    return torch.randn(*shape, device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed)).to(dtype)


def loss_gradient(moe, x2, sequences=None):
    """The loss's gradient of the gate, formed apart."""
    logits = ops.gate_logits(x2.detach(), moe.router.gate.weight.detach()).requires_grad_(True)
    idx = ops.route_topk(logits.detach(), moe.router.top_k, True)[1]
    loss, _ = F_.balance_loss(logits, idx, balance_coeff=LOSS["balance_loss_coeff"], z_coeff=LOSS["router_z_loss_coeff"], sequences=sequences)
    d, = torch.autograd.grad(loss, logits)
    return d.double().t() @ x2.detach().double()


@pytest.mark.parametrize("fused", [True, False])
def test_output_changed_in_place(fused):
    plain, with_it = pair(AnnotatedMoE)
    plain.fused = with_it.fused = fused
    x = tokens(2, 30, 64)
    for moe in (plain, with_it):
        out = moe(x)
        out += x
        out.mul_(2).sum().backward()
    want = plain.router.gate.weight.grad.double() + loss_gradient(with_it, x.reshape(-1, 64))
    assert rel(with_it.router.gate.weight.grad, want) <= 1e-5


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("scale", [1024.0, torch.tensor(1024.0)])
def test_a_scaled_loss(fused, scale):
    """The factor of the program's loss, taken off the gradients afterwards: the gradients without it."""
    _, moe = pair(AnnotatedMoE)
    moe.fused = fused
    x, d = tokens(2, 30, 64), tokens(2, 30, 64, seed=2)
    moe(x).backward(d)
    want = moe.router.gate.weight.grad.clone()
    moe.zero_grad()
    moe.balance_loss_scale = scale.to(DEV) if isinstance(scale, torch.Tensor) else scale
    moe(x).backward(d * 1024)
    assert torch.equal(moe.router.gate.weight.grad / 1024, want)      # (a power of two)


@pytest.mark.parametrize("cls", [AnnotatedMoE, MoEFeedForwardBlock])
@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("dtype,dims,experts", [(torch.bfloat16, (512, 256), 16), (torch.float32, (64, 32), 8)])
@pytest.mark.parametrize("T", [1, 3, 200])
def test_without_gradients_it_is_the_module_without_the_loss(cls, fused, dtype, dims, experts, T):
    """The same launches and bits, single tokens among them, and no value of a loss that was not formed."""
    plain, with_it = pair(cls, dtype, dims=dims, num_experts=experts)
    of = lambda m: m.moe if cls is MoEFeedForwardBlock else m  # noqa: E731
    of(plain).fused = of(with_it).fused = fused
    x = tokens(1, T, dims[0], dtype=dtype)
    off = torch.tensor([0, T], dtype=torch.int32, device=DEV)
    with_it(x, sequences=off)
    assert of(with_it).balance_loss is not None and of(with_it).tokens_per_expert.shape == (1, experts)
    launches = []
    with torch.no_grad():
        for m, more in ((plain, {}), (with_it, dict(sequences=off))):
            m(x, **more)
            torch.cuda.synchronize()
            _lib.timing_enable(True)
            try:
                out = m(x, **more)
                torch.cuda.synchronize()
                launches.append([name for name, _ in _lib.timing_collect()])
            finally:
                _lib.timing_enable(False)
            if m is plain:
                want = out
    assert torch.equal(out, want) and launches[0] == launches[1] and len(launches[0]) > 0
    assert of(with_it).balance_loss is None and of(with_it).tokens_per_expert is None
    of(with_it).balance_loss_without_grad = True
    with torch.no_grad():
        again = with_it(x, sequences=off)
    assert rel(again, want) <= (2e-2 if dtype == torch.bfloat16 else 1e-5)
    assert of(with_it).balance_loss.shape == () and int(of(with_it).tokens_per_expert.sum()) == T * 2


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,I", [(128, 512), (130, 515)])
def test_region_without_gradients_writes_no_pre_activations(dtype, H, I):
    """The region with the loss under no_grad: the bits of the one without it, in as little memory (and the loss's own)."""
    T, E = 2048, 8
    gen = torch.Generator(device=DEV).manual_seed(3)
    r = lambda *s: torch.randn(*s, device=DEV, generator=gen)  # noqa: E731
    args = (r(T, H).to(dtype), r(E, H) * 0.1, None, *((r(*s) * 0.05).to(dtype) for s in ((E, I, H), (E, H, I), (E, I, H))))
    peaks, outs = [], []
    with torch.no_grad():
        for run in (F_.expert_region, lambda *a, **k: F_.expert_region_balanced(*a, **k)[0]):
            run(*args, top_k=2, route_norm=True)
            torch.cuda.synchronize()
            torch.cuda.empty_cache()
            torch.cuda.reset_peak_memory_stats()
            before = torch.cuda.memory_allocated()
            outs.append(run(*args, top_k=2, route_norm=True))
            peaks.append(torch.cuda.max_memory_allocated() - before)
    assert torch.equal(*outs)
    # one of the two pre-activations alone would be more than the loss's workspace (33 chunks of 8 experts) and roundings of allocations
    assert peaks[1] <= peaks[0] + 2 * T * I * args[0].element_size() // 2


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("sequences", [False, True])
def test_block_trains_its_gate_on_the_loss(fused, sequences):
    """The block as it is, with the residual in its experts' last kernel or added by the unfused path."""
    plain, with_it = pair(MoEFeedForwardBlock)
    plain.moe.fused = with_it.moe.fused = fused
    x, d = tokens(2, 50, 64), tokens(2, 50, 64, seed=2)
    off = torch.tensor([0, 30, 30, 90], dtype=torch.int32, device=DEV) if sequences else None
    more = dict(sequences=off) if sequences else {}
    a, b = plain(x), with_it(x, **more)
    assert rel(b, a) <= 1e-6
    a.backward(d)
    b.backward(d)
    xn = F_.rmsnorm(x.reshape(-1, 64), with_it.ffn_norm.weight).detach()
    extra = loss_gradient(with_it.moe, xn, off)
    g0, g1 = (m.moe.router.gate.weight.grad for m in (plain, with_it))
    assert rel(g1, g0.double() + extra) <= 1e-5 and extra.abs().max() > 1e-3 * g0.abs().max()      # (and it is not nothing)
    for n in ("w1", "w2", "w3"):
        assert rel(getattr(with_it.moe.experts, n).grad, getattr(plain.moe.experts, n).grad) <= 1e-5
    assert int(with_it.moe.tokens_per_expert.sum()) == (180 if sequences else 200)


def test_experts_in_8_bits_train_the_gate_on_the_loss():
    plain, with_it = pair(AnnotatedMoE, torch.bfloat16, dims=(128, 64))
    x, d = tokens(2, 40, 128, dtype=torch.bfloat16), tokens(2, 40, 128, seed=2, dtype=torch.bfloat16)
    for m in (plain, with_it):
        m(x, experts_fp8=m.experts.quantize()).backward(d)
    g0, g1 = (m.router.gate.weight.grad for m in (plain, with_it))
    extra = loss_gradient(with_it, x.reshape(-1, 128))
    assert rel(g1 - g0, extra) <= 1e-5 * (1 + (g0.abs().max() / extra.abs().max()).item()) and rel(with_it.experts.w1.grad, plain.experts.w1.grad) == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("hold", [False, True])
def test_a_step_of_the_gate_takes_the_loss(dtype, hold):
    """Two microbatches into a bucket and FusedMuon's step over it: the gate's momentum holds what the loss adds to its gradient."""
    momenta, extra = [], 0
    for moe in pair(AnnotatedMoE, dtype):
        gate = moe.router.gate.weight
        router = flatten_params(BucketState(), [gate], optim_class=lambda q: FusedMuon(q, matrices=lambda p: p is not gate, adamw=dict(betas=(0.5, 0.9))))  # noqa: B023
        storage = ParamStorage(StageStore(buckets={0: router}, zero_managed_ubids={0}))
        for mb in range(2):
            x, d = (tokens(2, 32, 64, seed=10 * mb + k, dtype=dtype) for k in (1, 2))
            if moe.balanced:
                extra = extra + loss_gradient(moe, x.reshape(-1, 64))
            moe(x).backward(d * 1e-2)
            (storage.hold_param_grads if hold and mb else storage.accumulate_zero_param_grads_to_flat)(0)
        storage.step_zero_shard_optimizers()
        momenta.append(router.shard_optimizer.state[router.shard_param]["momentum"][:gate.numel()].view(gate.shape).clone())
    assert rel(momenta[1], momenta[0].double() + 0.5 * extra) <= 1e-5 and extra.abs().max() > 1e-2 * momenta[0].abs().max()
