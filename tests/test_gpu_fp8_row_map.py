"""Rows that a map names, in 8-bit blocks: entries outside of x are not followed."""
import pytest
import torch

from piper_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("div", [1, 3])
def test_entries_that_name_no_row_make_rows_of_nan(dev, div, dtype):
    print(f"[case] quantize rows, a map that leaves x, divisor {div} {dtype}", flush=True)
    x = torch.randn(5, 200, generator=torch.Generator().manual_seed(div)).to(dtype).to(dev)
    entries = [0, 5 * div - 1, -1, 5 * div, 2, 2 ** 31 - 1, -2 ** 31, 7 * div]
    q, s = ops.quantize_rows_fp8(x, torch.tensor(entries, dtype=torch.int32, device=dev), div)
    for r, entry in enumerate(entries):
        if 0 <= entry < 5 * div:
            want, scale = ops.quantize_rows_fp8(x[entry // div:entry // div + 1])
            assert torch.equal(q[r].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(s[r].view(torch.uint8), scale[0].view(torch.uint8))
        else:
            assert torch.isnan(q[r].float()).all()
    none = ops.quantize_rows_fp8(x, torch.empty(0, dtype=torch.int32, device=dev), div)
    assert none[0].shape == (0, 256) and none[1].shape == (0, 2)
