"""What the balance loss refuses, on the CPU, and its oracle."""
import ctypes as C

import pytest
import torch

from oracle import balance as O
from piper_amd import _lib, functional as F_
from piper_amd.moe import AnnotatedMoE, MoEArgs


@pytest.fixture()
def p():
    buf = C.create_string_buffer(1 << 16)
    yield (C.addressof(buf) + 255) // 256 * 256


def refused(rc, word):
    assert rc < 0 and word in _lib.status_string(rc)


def test_forward_refuses(p):
    lib = _lib.load()

    def run(logits=p, idx=p, seq=None, T=4, E=8, K=2, S=1, loss=p, counts=p, table=p, ws=p, bytes_=1 << 15):
        return lib.pk_balance_loss(logits, idx, seq, T, E, K, S, 1.0, 0.0, loss, counts, table, ws, bytes_, None)

    for bad in (dict(logits=None), dict(idx=None), dict(loss=None), dict(counts=None), dict(table=None), dict(T=-1), dict(E=0), dict(K=0), dict(S=0),
                dict(S=2)):
        refused(run(**bad), "argument")
    for bad in (dict(E=1025), dict(K=65), dict(T=1 << 31)):
        refused(run(**bad), "shape")
    for bad in (dict(ws=None), dict(ws=p + 4), dict(bytes_=100)):
        refused(run(**bad), "workspace")
    refused(lib.pk_balance_workspace_bytes(-1, 8, 1), "argument")
    assert lib.pk_balance_workspace_bytes(0, 8, 1) > 0
    # no chunk belongs to two sequences: as many more of them as there are sequences
    assert lib.pk_balance_workspace_bytes(64 * 512, 64, 1) >= 2 * 512 * 64 * 4


def test_backward_refuses(p):
    lib = _lib.load()

    def run(logits=p, seq=None, table=p, d_loss=p, d=p, T=4, E=8, S=1):
        return lib.pk_balance_loss_bwd(logits, seq, table, d_loss, d, T, E, S, None)

    for bad in (dict(logits=None), dict(table=None), dict(d_loss=None), dict(d=None), dict(T=-1), dict(E=0), dict(S=0), dict(S=3)):
        refused(run(**bad), "argument")
    refused(run(E=1025), "shape")
    assert run(T=0, logits=None) == 0
    args = [p, p, p, 4, 8, 2, 1, 1.0, p, None]
    assert lib.pk_route_topk_balanced_bwd(p, None, 1, p, *args[:3], 0, *args[4:]) == 0
    for first in ((None, None, 1, p), (p, None, 1, None), (p, None, 2, p), (p, None, 0, p)):
        refused(lib.pk_route_topk_balanced_bwd(*first, *args), "argument")
    region = [p, p, p, None, 0, p, 1, 1.0, p, 1, p, p, p, None, None, 0, p, 4, 64, 8, 2, None, 0, None]
    refused(lib.pk_region_router_balanced_bwd(p, None, 2, p, *region), "argument")
    refused(lib.pk_region_router_balanced_bwd(p, None, 1, None, *region), "argument")
    refused(lib.pk_region_router_balanced_bwd(p, None, 1, p, *region), "workspace")


def test_tensors_on_the_cpu_are_refused_and_fake_ones_get_shapes():
    logits, idx = torch.zeros(6, 4), torch.zeros(6, 2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU only"):
        F_.balance_loss(logits, idx)
    loss, counts = F_.balance_loss(logits.to("meta"), idx.to("meta"))
    assert loss.shape == () and counts.shape == (4,) and counts.dtype == torch.int32
    loss, counts = F_.balance_loss(logits.to("meta"), idx.to("meta"), sequences=torch.empty(4, dtype=torch.int32, device="meta"))
    assert counts.shape == (3, 4)
    w = [torch.empty(s, device="meta") for s in ((4, 8), (4, 16, 8), (4, 8, 16), (4, 16, 8))]
    out, loss, counts = F_.expert_region_balanced(torch.empty(6, 8, device="meta"), w[0], None, *w[1:], top_k=2, route_norm=True)
    assert out.shape == (6, 8) and loss.shape == () and counts.shape == (4,)


def test_a_loss_is_trained_beside_an_output():
    x = torch.tensor([2.0, 3.0], requires_grad=True)
    out = F_.with_loss(x * 5, (x * x).sum())
    assert torch.equal(out, torch.tensor([10.0, 15.0]))
    out.sum().backward()
    assert torch.equal(x.grad, 5 + 2 * x.detach())


def test_modules_ask_for_it_by_their_arguments():
    assert not AnnotatedMoE(MoEArgs(), 8, 8).balanced
    moe = AnnotatedMoE(MoEArgs(balance_loss_coeff=0.01), 8, 8)
    assert moe.balanced and AnnotatedMoE(MoEArgs(router_z_loss_coeff=0.01), 8, 8).balanced
    assert moe.balance_loss is None and moe.tokens_per_expert is None

    class Args:      # another framework's, which knows nothing of it
        num_experts, top_k, score_func, route_norm, route_scale, gate_bias, score_before_experts, num_shared_experts = 4, 2, "softmax", True, 1.0, False, False, 0
    assert not AnnotatedMoE(Args, 8, 8).balanced


def test_oracle_against_a_hand_worked_case_and_differences():
    # two tokens, two experts, both choose expert 0: f = (2, 0), P = mean softmax
    logits = torch.tensor([[1.0, 0.0], [2.0, 0.0]], dtype=torch.float64)
    p = torch.sigmoid(torch.tensor([1.0, 2.0], dtype=torch.float64))
    loss, counts = O.balance_loss(logits, torch.zeros(2, 1, dtype=torch.int64))
    assert torch.allclose(loss, 2 * p.mean()) and counts.tolist() == [[2, 0]]
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(9, 5, dtype=torch.float64, generator=gen).requires_grad_(True)
    idx = torch.topk(x.detach(), 2, dim=1).indices
    assert torch.autograd.gradcheck(lambda t: O.balance_loss(t, idx, 0.7, 0.3, [1, 4, 4, 8])[0], (x,))
    _, counts = O.balance_loss(x, idx, 1.0, 0.0, [1, 4, 4, 8])
    assert counts.sum(1).tolist() == [6, 0, 8]
    g, = torch.autograd.grad(O.balance_loss(x, idx, 0.7, 0.3, [1, 4, 4, 8])[0], x)
    assert (g.abs() <= O.gradient_scale(x.detach(), counts, 2, 0.7, 0.3, [1, 4, 4, 8]) * (1 + 1e-9)).all() and not g[0].any() and not g[8].any()
