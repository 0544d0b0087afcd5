"""The balance loss's gradient as a whole is neither too large nor too small.

Every element has the factor d_loss / S' (S' sequences with tokens).  Rounded by itself it would move them all together, by what the first
test computes for the numbers taken here.  All other roundings differ from token to token or from expert to expert, and the projection on the
exact gradient averages over them: eight of 2^-24 / sqrt(3) for each of 20,000 tokens, a thousand of which at least count, 3e-9 (rms);
one for each of at least 61 * 8 table entries, a hundred of which at least count, 3.4e-9.  2^-26 = 1.5e-8 is three times both together."""
import numpy as np
import pytest
import torch

from oracle import balance as O
from piper_amd import _lib, functional as F_
from test_gpu_balance import DEV, inputs

CASES = [(61, 1.1), (61, 1.3), (401, 0.7), (491, 1.3)]
TOL = 2.0 ** -26


def rounded_factor(S, d_loss):
    f = np.float32(d_loss) * np.float32(1 / S)
    return float(f) / (float(np.float32(d_loss)) / S) - 1


def test_numbers_whose_rounded_factor_shows():
    assert all(abs(rounded_factor(S, d)) > 2 * TOL for S, d in CASES)


def moved(got, want):
    got, want = got.double().cpu(), want.double().cpu()
    return ((got * want).sum() / (want * want).sum() - 1).item()


@pytest.mark.gpu
@pytest.mark.parametrize("S,d_loss", CASES)
def test_gradient_is_not_moved_as_a_whole(S, d_loss):
    T, E = 20000, 8
    off = torch.linspace(0, T, S + 1).round().int()
    logits, idx = inputs(T, E, 2, S, 0.5)
    e = logits.double().requires_grad_(True)
    d = torch.tensor(d_loss)
    want, = torch.autograd.grad(O.balance_loss(e, idx, 1.0, 0.0, off.tolist())[0], e, d.double())
    x = logits.to(DEV).requires_grad_(True)
    got, = torch.autograd.grad(F_.balance_loss(x, idx.to(DEV), sequences=off.to(DEV))[0], x, d.to(DEV))
    assert abs(moved(got, want)) <= TOL
    # behind the router: its kernel's gradient of the logits, without one of the scores
    lib, dev = _lib.load(), lambda *a, **k: torch.empty(*a, device=DEV, **k)
    oc, ic, dl, xc = off.to(DEV), idx.to(DEV), d.to(DEV), x.detach()
    bytes_ = int(lib.pk_balance_workspace_bytes(T, E, S))
    loss, counts, table, ws = dev(()), dev(S, E, dtype=torch.int32), dev(S * E + 2), dev(bytes_, dtype=torch.uint8)
    _lib.call("pk_balance_loss", xc.data_ptr(), ic.data_ptr(), oc.data_ptr(), T, E, 2, S, 1.0, 0.0, loss.data_ptr(), counts.data_ptr(), table.data_ptr(),
              ws.data_ptr(), bytes_, _lib.current_stream())
    got, scores = dev(T, E), torch.zeros(T, 2, device=DEV)
    _lib.call("pk_route_topk_balanced_bwd", table.data_ptr(), oc.data_ptr(), S, dl.data_ptr(), xc.data_ptr(), ic.data_ptr(), scores.data_ptr(), T, E, 2, 1, 1.0,
              got.data_ptr(), _lib.current_stream())
    assert abs(moved(got, want)) <= TOL
