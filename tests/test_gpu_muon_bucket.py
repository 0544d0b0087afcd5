"""FusedMuon over buckets on the GPU: every matrix, vector and empty tensor against the definitions of their steps, packed and held.

AdamW's tolerances are those of tests/test_gpu_muon.py: 1e-6 of the weights (of size 1), 1e-8 of first moments (gradients of 1e-2), and second
moments, sums of 1e-4 times 0.1 and less, to 1e-10: four roundings of 2^-24 and less of 1e-4 each, 2.4e-11."""
import pytest
import torch

from oracle import bucket as OB
from piper_amd import ops
from piper_amd.bucket import BucketState, ParamStorage, StageStore, flatten_params
from piper_amd.optim import FusedMuon
from test_gpu_muon import HYPER, check_matrix, make, put_grads

pytestmark = pytest.mark.gpu
ADAMW = dict(lr=0.002, betas=(0.8, 0.9), eps=1e-6, weight_decay=0.3)
# an empty tensor shares its place with the one behind it
SHAPES = [(0, 8), (40, 96), (7,), (3, 0, 24), (3, 64, 24), (0,), (33,), (1,), (130, 50), (2, 5, 0), (1030,), (5,)]


def a_bucket(dev, dtype, align):
    params = [torch.nn.Parameter(make(s, i, dtype).to(dev)) for i, s in enumerate(SHAPES)]
    bucket = flatten_params(BucketState(), params, optim_class=lambda ps: FusedMuon(ps, adamw=ADAMW, **HYPER), align_bytes=align)
    return params, bucket, ParamStorage(StageStore(buckets={0: bucket}, zero_managed_ubids={0}))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("align", [256, 1])
@pytest.mark.parametrize("hold", [False, True])
def test_everything_in_a_bucket_takes_its_own_step(dev, dtype, align, hold):
    params, bucket, storage = a_bucket(dev, dtype, align)
    opt, p = bucket.shard_optimizer, bucket.shard_param
    second = {i: torch.zeros(torch.Size(s).numel()) for i, s in enumerate(SHAPES) if len(s) == 1}
    before = {k: v.clone() for k, v in opt._init_state(p).items() if isinstance(v, torch.Tensor)}
    for step in (1, 2, 3):
        storage.zero_grad_buffers()
        total = [torch.zeros(s) for s in SHAPES]
        for mb in range(2):
            put_grads(params, 1000 * step + 500 * mb, dev, missing=(4, 6) if mb else (1, 2))
            for t, q in zip(total, params):
                if q.grad is not None:
                    t += q.grad.float().cpu()
            (storage.hold_param_grads if hold and mb else storage.accumulate_zero_param_grads_to_flat)(0)
        storage.step_zero_shard_optimizers()
        st = opt.state[p]
        assert st["step"] == step
        at = 0
        for i, ((q, o, n, s), g) in enumerate(zip(bucket.param_view_specs, total)):
            cut = lambda t: t[o:o + n].view(s)  # noqa: E731
            if len(s) >= 2 and n:
                check_matrix(cut(st["master"]), cut(st["momentum"]), cut(before["master"]), cut(before["momentum"]), g, **HYPER)
            elif n:
                want, m, v = OB.adamw_step_torch(cut(before["master"]).cpu(), g, cut(before["momentum"]).cpu(), second[i].clone(), step, ADAMW["lr"], ADAMW["betas"],
                                                 ADAMW["eps"], ADAMW["weight_decay"])
                got_v = st["exp_avg_sq"][at:at + n].cpu()
                at += -(-n // 4) * 4
                assert (cut(st["master"]).cpu() - want).abs().max() <= 1e-6, s
                assert (cut(st["momentum"]).cpu() - m).abs().max() <= 1e-8 and (got_v - v).abs().max() <= 1e-10, s
                second[i] = got_v
            assert torch.equal(q.detach(), cut(st["master"]).to(dtype))
        assert at == st["exp_avg_sq"].numel()
        before = {k: st[k].clone() for k in before}


@pytest.mark.parametrize("align", [256, 1])
def test_held_and_packed_steps_are_the_same_bits(dev, align):
    got = []
    for hold in (False, True):
        params, bucket, storage = a_bucket(dev, torch.bfloat16, align)
        for step in range(2):
            storage.zero_grad_buffers()
            put_grads(params, 7 * step, dev, missing=(0, 3))
            (storage.hold_param_grads if hold else storage.accumulate_zero_param_grads_to_flat)(0)
            storage.step_zero_shard_optimizers()
        got.append((bucket.flat_params, *(bucket.shard_optimizer.state[bucket.shard_param][k] for k in ("master", "momentum", "exp_avg_sq"))))
    assert all(torch.equal(a, b) for a, b in zip(*got))


def test_a_gradient_in_a_buffer_that_is_written_is_refused(dev):
    room = torch.zeros(8, 4, 6, device=dev)
    w, m, g, f = room[:2], room[2:4], room[4:6], room[6:8]
    half = w[0].view(-1).view(torch.bfloat16)[:24].view(4, 6)
    for bad in (dict(grads=[m[0], g[1]]), dict(grads=[g[0], w[0]]), dict(grads=[room.view(-1)[36:60].view(4, 6), g[1]]), dict(flat_grads=[w[1], f[1]]),
                dict(flat_grads=[f[0], f[1]], grads=[g[0], f[0]], zero_grad=True), dict(grads=[half, None])):
        args = dict(grads=[g[0], g[1]], flat_grads=[f[0], f[1]]) | bad
        with pytest.raises(ValueError, match="overlap"):
            ops.muon_fused([w[0], w[1]], [m[0], m[1]], args.pop("grads"), lr=0.1, **args)
    # read twice, neighbours
    ops.muon_fused([w[0], w[1]], [m[0], m[1]], [g[0], g[0]], flat_grads=[g[0], f[1]], lr=0.1)
    ops.muon_fused([w[0], w[1]], [m[0], m[1]], [g[0], g[1]], flat_grads=[f[0], f[1]], lr=0.1, zero_grad=True)
