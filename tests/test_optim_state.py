"""FusedAdamW's saved states: which ones it takes, and that a refused one changes nothing."""
import copy

import pytest
import torch

from piper_amd.optim import FusedAdamW


def _optimizer(bits, dtype=torch.float32, sizes=(130, 64), seed=0):
    """An optimizer some steps on, its state made up (a step itself needs a GPU)."""
    g = torch.Generator().manual_seed(seed)
    params = [torch.nn.Parameter(torch.randn(n, generator=g).to(dtype)) for n in sizes]
    opt = FusedAdamW(params, state_bits=bits)
    for p in params:
        st = opt._init_state(p)
        st["step"] = 3 + seed
        for name in ("exp_avg", "exp_avg_sq"):
            st[name].view(torch.uint8 if bits == 8 else torch.int32).random_(1, 100, generator=g)
        if bits == 8:
            for name in ("exp_avg_scale", "exp_avg_sq_scale"):
                st[name].view(torch.uint8).random_(90, 120, generator=g)
        elif dtype != torch.float32:
            st["master"] += torch.rand(p.numel(), generator=g) * 2.0 ** -12
    return params, opt


def _bits(t):
    return t.detach().contiguous().view(torch.uint8)


def _same(a, b):
    return a.keys() == b.keys() and all(torch.equal(_bits(a[k]), _bits(b[k])) and a[k].dtype == b[k].dtype if isinstance(a[k], torch.Tensor) else a[k] == b[k]
                                        for k in a)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("to,what", [(32, "8-bit moments"), (8, "no 8-bit moments")])
def test_states_of_the_other_width_are_refused_and_change_nothing(to, what, dtype):
    _, source = _optimizer(40 - to, dtype, seed=1)
    params, opt = _optimizer(to, dtype)
    before = [copy.deepcopy(opt.state[p]) for p in params]
    groups = copy.deepcopy([{k: v for k, v in g.items() if k != "params"} for g in opt.param_groups])
    source.param_groups[0]["lr"] = 0.5
    with pytest.raises(ValueError, match=what):
        opt.load_state_dict(source.state_dict())
    assert all(_same(opt.state[p], b) for p, b in zip(params, before))
    assert [{k: v for k, v in g.items() if k != "params"} for g in opt.param_groups] == groups
    assert not opt._optimizer_load_state_dict_pre_hooks


@pytest.mark.parametrize("bits", [8, 32])
def test_incomplete_states_and_other_sizes_are_refused(bits):
    params, opt = _optimizer(bits)
    before = [copy.deepcopy(opt.state[p]) for p in params]
    with pytest.raises(ValueError, match="a parameter of 130 elements"):
        opt.load_state_dict(_optimizer(bits, sizes=(131, 64))[1].state_dict())
    for gone in ("master", "exp_avg_sq", "step"):
        broken = copy.deepcopy(_optimizer(bits, seed=2)[1].state_dict())
        del broken["state"][1][gone]
        with pytest.raises(ValueError):
            opt.load_state_dict(broken)
    with pytest.raises(ValueError):
        opt.load_state_dict(_optimizer(bits, sizes=(130,))[1].state_dict())
    assert all(_same(opt.state[p], b) for p, b in zip(params, before))
    empty = FusedAdamW([torch.nn.Parameter(torch.zeros(n)) for n in (130, 64)], state_bits=bits)
    opt.load_state_dict(empty.state_dict())      # saved before the first step
    assert not any(opt.state.get(p) for p in params)


def test_a_hook_of_the_program_comes_first():
    """A pre-hook that takes the 8-bit state out: what is loaded is what it returns."""
    _, eight = _optimizer(8, seed=1)
    params, opt = _optimizer(32)
    opt.register_load_state_dict_pre_hook(lambda _, sd: dict(sd, state={}))
    opt.load_state_dict(eight.state_dict())
    assert not any(opt.state.get(p) for p in params)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [8, 32])
def test_what_is_loaded_is_what_was_saved(bits, dtype):
    theirs, source = _optimizer(bits, dtype, seed=1)
    params, opt = _optimizer(bits, dtype)
    with torch.no_grad():
        for p, q in zip(params, theirs):
            p.copy_(q)
    saved = copy.deepcopy(source.state_dict())
    seen = []
    opt.register_load_state_dict_post_hook(lambda o: seen.append(o.state[params[0]]["master"].dtype))
    opt.load_state_dict(saved)
    assert seen == [torch.float32] and len(opt._optimizer_load_state_dict_post_hooks) == 1
    for i, (p, q) in enumerate(zip(params, theirs)):
        st = opt.state[p]
        assert _same(st, source.state[q]) and st["master"].dtype == torch.float32
        assert (st["master"].data_ptr() == p.data_ptr()) == (dtype == torch.float32)      # a step of the master is one of the parameter
        for name in ("exp_avg", "exp_avg_sq"):
            assert st[name].data_ptr() != saved["state"][i][name].data_ptr()
