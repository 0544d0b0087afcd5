"""A row of the output's gradient that is not finite, where the region's weight gradients come from transposed copies."""
import pytest
import torch

from piper_amd import _lib
from piper_amd import functional as F_

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_weight_gradients_see_their_own_experts_rows_only(dev, value):
    T, H, E, I, K = 200, 2048, 6, 1024, 2
    print(f"[case] region, d_out holds {value}", flush=True)
    assert _lib.load().pk_region_transposed_pays(T * K, H, I, E, _lib.PK_BF16) == 1 and T * K > 40 * E
    g = torch.Generator().manual_seed(0)
    mk = lambda *shape, unit=0.05: (torch.randn(shape, generator=g) * unit).bfloat16().to(dev).requires_grad_(True)  # noqa: E731
    x, w1, w2, w3, d_out = mk(T, H, unit=1.0), mk(E, I, H), mk(E, H, I), mk(E, I, H), mk(T, H, unit=1.0).detach()
    gate = torch.zeros(E, H)
    gate[torch.arange(E), torch.arange(E)] = 4.0
    gate = gate.to(dev).requires_grad_(True)
    with torch.no_grad():      # token t goes to experts t % 3 and 3 + t % 3
        x[:, :E] = 0.0
        for j in (0, 3):
            x[torch.arange(T), j + torch.arange(T) % 3] = 1.0 + j

    def grads(d):
        y = F_.expert_region(x, gate, None, w1, w2, w3, top_k=K, route_norm=True)
        return torch.autograd.grad(y, (w1, w2, w3), d)

    want = grads(d_out)
    assert all(torch.isfinite(t).all() for t in want)
    for t in (0, 1, 2, T - 3, T - 2, T - 1):              # the first and the last rows of all six
        bad = d_out.clone()
        bad[t, ::7] = value
        for a, b in zip(grads(bad), want):
            for e in range(E):
                assert not torch.isfinite(a[e]).all() if e % 3 == t % 3 else torch.equal(a[e], b[e]), (t, e)
