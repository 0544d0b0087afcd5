"""The fused region with tensors that start anywhere, where its weight gradients come from transposed copies."""
import pytest
import torch

from piper_amd import _lib
from piper_amd import functional as F_

pytestmark = pytest.mark.gpu


def _odd(t):
    """The same values two bytes behind a 16-byte boundary."""
    t = t.detach()
    v = torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape)
    assert v.data_ptr() % 16 == 2
    return v


def test_rows_and_gradients_that_start_anywhere(dev):
    T, H, E, I, K = 200, 2048, 6, 1024, 2
    print("[case] region, views at odd offsets", flush=True)
    assert _lib.load().pk_region_transposed_pays(T * K, H, I, E, _lib.PK_BF16) == 1 and T * K > 40 * E
    g = torch.Generator().manual_seed(0)
    mk = lambda *shape, unit=0.05: (torch.randn(shape, generator=g) * unit).bfloat16().to(dev).requires_grad_(True)  # noqa: E731
    x, w1, w2, w3, d_out = mk(T, H, unit=1.0), mk(E, I, H), mk(E, H, I), mk(E, I, H), mk(T, H, unit=1.0).detach()
    gate = (torch.randn(E, H, generator=g) * 0.05).to(dev).requires_grad_(True)

    def close(a, b):
        # the same sums of bf16 operands in another order and, of an unaligned x, by other kernels: a bf16 step of what is rounded
        # on the way (g, u and the gradients behind them) moves a result by no more than a few steps of the largest of its kind
        return all((p.double() - q.double()).norm() <= 2.0 ** -7 * q.double().norm() for p, q in zip(a, b))

    def grads(x_, d):
        x_ = x_.requires_grad_(True)
        y = F_.expert_region(x_, gate, None, w1, w2, w3, top_k=K, route_norm=True)
        return torch.autograd.grad(y, (w1, w2, w3, x_), d)

    want = grads(x, d_out)
    assert all(torch.equal(a, b) for a, b in zip(grads(x, _odd(d_out)), want))
    assert close(grads(_odd(x), d_out), want)
    with F_.accumulate_weight_grads():
        sides = []
        for place in (lambda t: t.clone(), _odd):
            for p, t in zip((w1, w2, w3), want):
                p.grad = place(t)
            at = [p.grad for p in (w1, w2, w3)]
            F_.expert_region(x, gate, None, w1, w2, w3, top_k=K, route_norm=True).backward(d_out)
            assert all(p.grad is a for p, a in zip((w1, w2, w3), at))
            sides.append([a.clone() for a in at])
    assert all(torch.equal(a, b) for a, b in zip(*sides))
    for p in (w1, w2, w3):
        p.grad = None
    odd = [_odd(w).requires_grad_(True) for w in (w1, w2, w3)]
    y = F_.expert_region(x, gate, None, *odd, top_k=K, route_norm=True)
    assert close(torch.autograd.grad(y, (*odd, x), d_out), want)
