"""FusedMuon on the CPU: what it takes for matrices, what it refuses, which saved states it loads."""
import copy

import pytest
import torch

from piper_amd.optim import FusedMuon


def bucket(seed=0, dtype=torch.bfloat16):
    """A flat parameter with a matrix, a vector and a stack of matrices in it, some steps on (made up: a step itself needs a GPU)."""
    g = torch.Generator().manual_seed(seed)
    p = torch.nn.Parameter(torch.randn(600, generator=g).to(dtype))
    params = [torch.empty(10, 20), torch.empty(7), torch.empty(2, 5, 8)]
    specs = [(params[0], 0, 200, (10, 20)), (params[1], 256, 7, (7,)), (params[2], 512, 80, (2, 5, 8))]
    opt = FusedMuon([p], lr=0.01)
    opt.bind_views(p, specs)
    st = opt._init_state(p)
    st["step"] = 4 + seed
    for k in ("momentum", "exp_avg_sq"):
        st[k].copy_(torch.rand(st[k].shape, generator=g))
    return p, opt, specs


def test_places_and_state():
    p, opt, specs = bucket()
    assert opt._places(p) == [(0, 200, (10, 20), True), (256, 7, (7,), False), (512, 80, (2, 5, 8), True)]
    st = opt.state[p]
    assert st["master"].numel() == st["momentum"].numel() == 600 and st["exp_avg_sq"].numel() == 8
    assert all(st[k].dtype == torch.float32 for k in ("master", "momentum", "exp_avg_sq"))
    w, v = torch.nn.Parameter(torch.zeros(4, 6)), torch.nn.Parameter(torch.zeros(4))
    opt = FusedMuon([w, v])
    assert opt._places(w) == [(0, 24, (4, 6), True)] and opt._places(v) == [(0, 4, (4,), False)]
    opt = FusedMuon([w, v], matrices=lambda t: t is not w)
    assert not opt._places(w)[0][3] and not opt._places(v)[0][3]      # a vector is no matrix whoever says so


def test_views_that_are_none():
    p, opt, specs = bucket()
    with pytest.raises(RuntimeError, match="stepped already"):
        opt.bind_views(p, specs)
    q = torch.nn.Parameter(torch.zeros(100))
    opt = FusedMuon([q])
    for bad in ((None, 50, 60, (6, 10)), (None, -1, 4, (2, 2)), (None, 0, 10, (2, 6))):
        with pytest.raises(ValueError, match="no view"):
            opt.bind_views(q, [(torch.empty(2, 2), *bad[1:])])
    with pytest.raises(ValueError, match="flat"):
        opt.bind_views(torch.zeros(3, 3), [])
    opt.bind_views(q, [(torch.empty(2, 5), 0, 10, (2, 5))])
    with pytest.raises(RuntimeError, match="in their order"):
        opt.step_packed(q, [None], [4], [10])


@pytest.mark.parametrize("bad", [dict(lr=-1), dict(momentum=1.0), dict(weight_decay=-0.1), dict(eps=0), dict(ns_steps=101), dict(ns_coefficients=(1, 2)),
                                 dict(adjust_lr="no"), dict(adamw=dict(lr=-1)), dict(adamw=dict(betas=(1.0, 0.9))), dict(adamw=dict(beta=0.9)),
                                 dict(lr=0.0, adamw=dict(lr=0.1))])
def test_hyper_parameters(bad):
    with pytest.raises(ValueError):
        FusedMuon([torch.nn.Parameter(torch.zeros(2, 2))], **bad)


def test_the_others_lr_follows_a_schedule():
    w = torch.nn.Parameter(torch.zeros(2, 2))
    opt = FusedMuon([w], lr=0.1, adamw=dict(lr=0.01))
    schedule = torch.optim.lr_scheduler.LambdaLR(opt, lambda step: 0.5 ** step)
    opt.zero_grad()
    opt.step()
    schedule.step()
    g = opt.param_groups[0]
    assert g["lr"] == 0.05 and abs(g["lr"] * g["adamw_lr_ratio"] - 0.005) < 1e-12


def same(a, b):
    return a.keys() == b.keys() and all(torch.equal(a[k], b[k]) and a[k].dtype == b[k].dtype if isinstance(a[k], torch.Tensor) else a[k] == b[k] for k in a)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_saved_states(dtype):
    p, opt, _ = bucket(1, dtype)
    q, other, _ = bucket(2, dtype)
    other.load_state_dict(copy.deepcopy(opt.state_dict()))
    want = dict(opt.state[p])
    if dtype == torch.float32:
        want["master"] = q.detach().reshape(-1)
        assert other.state[q]["master"].data_ptr() == q.data_ptr()
    assert same(other.state[q], want)
    before = copy.deepcopy(other.state[q])
    plain = torch.nn.Parameter(torch.zeros(600, dtype=dtype))
    stranger = FusedMuon([plain])                    # the same size, no matrix in it
    stranger._init_state(plain)["step"] = 1
    for broken in (stranger.state_dict(), *({**s, "state": {0: {k: v for k, v in s["state"][0].items() if k != gone}}}
                                            for s in [opt.state_dict()] for gone in ("momentum", "step", "exp_avg_sq", "master"))):
        with pytest.raises(ValueError, match="FusedMuon: the saved state"):
            other.load_state_dict(broken)
        assert same(other.state[q], before)
