"""The balance loss with more sequences than are looked at together, most of them without tokens, in all of its forms.  Tolerances as in
tests/test_gpu_balance.py."""
import pytest
import torch

from piper_amd import functional as F_, ops
from test_gpu_balance import DEV, check, inputs, layer, rel

pytestmark = pytest.mark.gpu


def offsets(T, S, kind, seed=0):
    gen = torch.Generator().manual_seed(seed)
    if kind == "short":           # a few tokens each
        cuts = torch.randint(3, T - 3, (S + 1,), generator=gen).sort().values
    elif kind == "one place":     # all but two of them empty, side by side
        cuts = torch.full((S + 1,), T // 3)
        cuts[0], cuts[-1] = 1, T - 2
    elif kind == "ends":          # in front of the tokens and behind them
        cuts = torch.full((S + 1,), T)
        cuts[:S // 2] = 0
        cuts[S // 2] = T // 2
    else:                         # clusters of empty ones between those with tokens
        cuts = (torch.randint(0, 40, (S + 1,), generator=gen).sort().values * T) // 40
    return cuts.to(torch.int32)


KINDS = ["short", "one place", "ends", "clusters"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T,E,K,S", [(2000, 8, 2, 127), (2000, 8, 2, 128), (2000, 20, 3, 129), (3000, 8, 2, 1023), (3000, 8, 2, 1025), (3000, 60, 4, 1030),
                                     (700, 8, 2, 5000), (40000, 8, 2, 9000)])
def test_loss_and_gradient(T, E, K, S, kind):
    check(T, E, K, 0.7, 1e-2, offsets(T, S, kind, S).tolist(), seed=S, skew=0.5)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("S", [63, 64, 127, 128, 129, 200, 4097, 9000])
def test_behind_the_router_and_in_the_region(kind, S):
    t, d_out = layer(600, 64, 8, 32, torch.float32, 9)
    off = offsets(600, S, kind, S).to(DEV)
    kw = dict(top_k=2, route_norm=True, balance_coeff=0.5, z_coeff=0.02, sequences=off)
    d_loss = torch.tensor(300.0, device=DEV)
    logits = ops.gate_logits(t["x"].detach(), t["w_gate"].detach()).requires_grad_(True)
    idx = ops.route_topk(logits.detach(), 2, True)[1]
    loss, counts = F_.balance_loss(logits, idx, balance_coeff=0.5, z_coeff=0.02, sequences=off)
    dl, = torch.autograd.grad(loss, logits, d_loss)
    want = dl.double().t() @ t["x"].detach().double()
    for got in (F_.expert_region_balanced(t["x"], t["w_gate"], None, t["w1"], t["w2"], t["w3"], **kw)[1:],
                F_.router_balanced(t["x"], t["w_gate"], **kw)[3:]):
        assert torch.equal(got[0], loss) and torch.equal(got[1], counts)
        g, = torch.autograd.grad(got[0], t["w_gate"], d_loss)
        assert rel(g, want) <= 1e-5


def test_cost_does_not_grow_with_tokens_times_sequences():
    """131,072 tokens and half a million sequences: 7e10 offsets if every token looked at all of them, tens of milliseconds and more; with a
    search forward and backward stay far below 20 ms, by themselves and behind the router."""
    T, E, S = 131072, 8, 1 << 19
    logits, idx = (v.to(DEV) for v in inputs(T, E, 2, 1))
    off = (torch.arange(S + 1, device=DEV) // 4).to(torch.int32)
    x = torch.randn(T, 64, device=DEV)
    w = (torch.randn(E, 64, device=DEV) * 0.1).requires_grad_(True)
    leaf = logits.requires_grad_(True)

    def alone():
        torch.autograd.grad(F_.balance_loss(leaf, idx, sequences=off)[0], leaf)

    def behind():
        torch.autograd.grad(F_.router_balanced(x, w, top_k=2, route_norm=True, sequences=off)[3], w)
    for run in (alone, behind):
        run()
        times = []
        for _ in range(3):
            begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            begin.record()
            run()
            end.record()
            end.synchronize()
            times.append(begin.elapsed_time(end))
        assert min(times) < 20.0, times
