"""What FusedMuon hands to the kernels, on the CPU with the two entry points recorded in their place."""
import pytest
import torch

from piper_amd import ops
from piper_amd.optim import FusedMuon


@pytest.fixture()
def calls(monkeypatch):
    made = []

    def muon(masters, momenta, grads, *, flat_grads, shadows, **kw):
        for i, w in enumerate(masters):
            assert grads[i] is None or grads[i].numel() == w.numel()
            made.append(("muon", tuple(w.shape), w.data_ptr(), momenta[i].data_ptr(), grads[i], None if flat_grads[i] is None else flat_grads[i].data_ptr()))

    def adamw(master, exp_avg, exp_avg_sq, flat, grads, offsets, numels, **kw):
        assert offsets == [0] and numels == [master.numel()] and exp_avg_sq.numel() == master.numel()
        made.append(("adamw", (master.numel(),), master.data_ptr(), exp_avg.data_ptr(), grads[0], exp_avg_sq.data_ptr()))
    monkeypatch.setattr(ops, "muon_fused", muon)
    monkeypatch.setattr(ops, "adamw_fused_packed", adamw)
    return made


# an empty tensor shares its offset with the one behind it
SHAPES = [(0, 8), (10, 20), (0,), (7,), (2, 0, 4), (5,), (3, 4, 8), (0, 3)]


def bucket():
    offsets, end = ops.bucket_plan([torch.Size(s).numel() for s in SHAPES], 4, 256)
    p = torch.nn.Parameter(torch.randn(end))
    opt = FusedMuon([p], lr=0.01)
    params = [torch.empty(s) for s in SHAPES]
    opt.bind_views(p, [(t, o, t.numel(), tuple(t.shape)) for t, o in zip(params, offsets)])
    return p, opt, offsets, [t.numel() for t in params]


@pytest.mark.parametrize("order", [1, -1])
def test_gradients_reach_their_own_parameters(calls, order):
    global SHAPES
    shapes, SHAPES = SHAPES, SHAPES[::order]
    try:
        p, opt, offsets, numels = bucket()
        assert len(set(offsets)) < len(offsets)
        grads = [torch.randn(s) for s in SHAPES]
        flat = torch.zeros_like(p)
        opt.step_packed(p, grads, offsets, numels, flat)
        st = opt.state[p]
        assert st["step"] == 1
        got = {c[2]: c for c in calls}
        seconds = set()
        for s, o, n, g in zip(SHAPES, offsets, numels, grads):
            if n == 0:
                continue
            c = got.pop(st["master"][o:].data_ptr())
            assert c[0] == ("muon" if len(s) >= 2 else "adamw") and c[4].reshape(-1).data_ptr() == g.data_ptr() and c[3] == st["momentum"][o:].data_ptr()
            if c[0] == "muon":
                assert c[1] == s and c[5] == flat[o:].data_ptr()
            else:
                at = (c[5] - st["exp_avg_sq"].data_ptr()) // 4
                assert at % 4 == 0 and not seconds & set(range(at, at + n)) and at + n <= st["exp_avg_sq"].numel()
                seconds |= set(range(at, at + n))
        assert not got
    finally:
        SHAPES = shapes


def test_parameters_of_other_types_are_refused_before_anything_changes(calls):
    for shape in ((4, 6), (5,)):
        p = torch.nn.Parameter(torch.randn(shape).half())
        p.grad = torch.randn(shape).half()
        opt = FusedMuon([p])
        with pytest.raises(ValueError, match="float32 or bfloat16"):
            opt.step()
        assert not calls and not opt.state.get(p)


def test_gradients_of_any_iterable(calls):
    p, opt, offsets, numels = bucket()
    opt.step_packed(p, (torch.zeros(s) for s in SHAPES), iter(offsets), iter(numels))
    assert len(calls) == sum(n > 0 for n in numels)


def broken(grads, flat):
    yield [None] * 7, flat
    for i, g in ((1, torch.zeros(199)), (1, torch.zeros(10, 20, dtype=torch.float64)), (1, grads[1].to("meta")), (5, torch.zeros(6)), (1, grads[1].bfloat16())):
        yield [*grads[:i], g, *grads[i + 1:]], flat
    yield grads, flat[:-1]
    yield grads, flat.double()


def test_a_refused_step_leaves_everything_as_it_was(calls):
    p, opt, offsets, numels = bucket()
    grads, flat = [torch.randn(s) for s in SHAPES], torch.zeros_like(p)
    for bad, f in broken(grads, flat):
        with pytest.raises(ValueError, match="FusedMuon"):
            opt.step_packed(p, bad, offsets, numels, f)
        assert not calls and not opt.state.get(p)
    opt.step_packed(p, grads, offsets, numels, flat)
    made = len(calls)
    for bad, f in broken(grads, flat):
        with pytest.raises(ValueError, match="FusedMuon"):
            opt.step_packed(p, bad, offsets, numels, f)
        assert len(calls) == made and opt.state[p]["step"] == 1
