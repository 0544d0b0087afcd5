"""FusedAdamW with 32-bit moments, saved and loaded: the run goes on bit for bit."""
import copy
import io

import pytest
import torch

from piper_amd.optim import FusedAdamW

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("model_first", [True, False])
def test_saved_and_loaded_state_continues_bit_for_bit(dev, dtype, model_first):
    print(f"[case] FusedAdamW state_dict {dtype} model_first={model_first}", flush=True)
    g = torch.Generator().manual_seed(4)
    steps = [torch.randn(300, generator=g).to(dtype).to(dev) for _ in range(5)]
    p = torch.nn.Parameter(torch.randn(300, generator=g).to(dtype).to(dev))
    opt = FusedAdamW([p], lr=1e-2)
    for i, gr in enumerate(steps):
        if i == 2:
            file = io.BytesIO()
            torch.save((p.detach(), opt.state_dict()), file)
        p.grad = gr
        opt.step()
    file.seek(0)
    weights, saved = torch.load(file, weights_only=True)
    q = torch.nn.Parameter(torch.zeros_like(p))
    other = FusedAdamW([q], lr=1e-2)
    for what in (0, 1) if model_first else (1, 0):
        if what == 0:
            with torch.no_grad():
                q.copy_(weights)
        else:
            other.load_state_dict(copy.deepcopy(saved))
    for gr in steps[2:]:
        q.grad = gr
        other.step()
    assert torch.equal(p, q)
    for k in ("master", "exp_avg", "exp_avg_sq"):
        assert torch.equal(opt.state[p][k], other.state[q][k]) and other.state[q][k].dtype == torch.float32
