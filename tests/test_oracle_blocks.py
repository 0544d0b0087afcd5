"""The restatement of the 8-bit block formats against torch's own 8-bit types and against closed forms (CPU)."""
import math

import pytest
import torch

from oracle import blocks as B


@pytest.mark.parametrize("mantissa,bias,dtype,top", [(3, 7, torch.float8_e4m3fn, 448.0), (2, 15, torch.float8_e5m2, 57344.0)])
def test_nearest_is_the_types_own_rounding(mantissa, bias, dtype, top):
    codes = torch.arange(0, 128, dtype=torch.uint8).view(dtype).double()
    codes = codes[torch.isfinite(codes)]
    assert codes.max() == top and torch.equal(B.nearest(codes, mantissa, bias), codes)
    between = torch.cat([(codes[1:] + codes[:-1]) / 2, codes[:-1] + (codes[1:] - codes[:-1]) * 0.499, codes[:-1] + (codes[1:] - codes[:-1]) * 0.501])
    for t in (between, -between, torch.linspace(-top, top, 4001, dtype=torch.float64)):
        assert torch.equal(B.nearest(t.float().double(), mantissa, bias), t.float().to(dtype).double())


def test_scale_exponent_is_the_smallest_that_fits():
    for largest in (448.0, 57344.0):
        for k in range(-126, 100, 7):
            at = largest * 2.0 ** k
            for a, want in ((at, k), (at * (1 + 2.0 ** -40), k + 1), (at * (1 - 2.0 ** -40), k), (at / 2, max(k - 1, -126)), (at * 0.75, k)):
                assert B.scale_exponent(torch.tensor([a], dtype=torch.float64), largest).item() == want
        assert B.scale_exponent(torch.tensor([0.0, 1e-300], dtype=torch.float64), largest).tolist() == [-126, -126]


def test_blocks_round_trip_and_poison_only_themselves():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(5, 300, generator=g) * torch.tensor([1e-20, 1.0, 1e20, 1e-3, 7.0])[:, None]
    err = (B.rounded_rows(x) - x.double()).abs()
    blocks = torch.nn.functional.pad(x.double().abs(), (0, 84)).view(5, 3, 128).amax(2).repeat_interleave(128, 1)[:, :300]
    # half a step of a normal value, or of the subnormals, whose step is 2^-9 of the scale and the scale at most amax / 224
    assert (err <= torch.maximum(2.0 ** -4 * x.double().abs(), blocks / 224 * 2.0 ** -10)).all()
    x[2, 130] = math.inf
    x[3, 299] = math.nan
    q, k = B.rows(x)
    assert torch.isnan(q.view(5, 3, 128)).all(2).tolist() == [[False] * 3, [False] * 3, [False, True, False], [False, False, True], [False] * 3]
    w = torch.randn(2, 130, 257, generator=g)
    assert (B.rounded_weights(w) - w.double()).abs().max() <= w.abs().max() * 2.0 ** -4


def test_stochastic_rounding_is_unbiased_and_keeps_positive_values():
    n = 64 * 64
    bits = B.random_bits(n, 12345)
    assert len(set(bits.tolist())) == n                     # the mix is a permutation of the index
    for half in (bits >> 16, bits & 0xFFFF):
        u = half.double() / 65536
        # mean and variance of n uniform numbers, within five deviations
        assert abs(u.mean() - 0.5) < 5 / math.sqrt(12 * n) and abs(u.var() - 1 / 12) < 5 * math.sqrt(1 / 180 / n)
    for mantissa, value in ((3, 3.3e-4), (2, 1.7e-7)):
        x = torch.full((n,), value, dtype=torch.float64)
        v, k = B.encode(x, bits >> 16, mantissa)
        got = v * B.two_to(k).repeat_interleave(64)
        step = B.grid_step(x / B.two_to(k[0]), mantissa, 7 if mantissa == 3 else 15) * B.two_to(k[0])
        assert (got - x).abs().max() < step[0]
        assert abs((got - x).mean()) < 5 * step[0] / 2 / math.sqrt(n)
    tiny = torch.cat([torch.tensor([1.0]), torch.full((63,), 1e-30)]).double()
    v, _ = B.encode(tiny, bits[:64] >> 16, 2)
    assert (v > 0).all()
    bad = torch.tensor([math.nan, -math.inf, 2.0, 0.0]).double()
    v, k = B.encode(bad, bits[:4] >> 16, 3)
    assert torch.isnan(v[:2]).all() and (v * B.two_to(k))[2:].tolist() == [2.0, 0.0]


def test_adamw_step_is_torchs():
    g = torch.Generator().manual_seed(1)
    p0 = torch.randn(50, generator=g, dtype=torch.float64)
    p = torch.nn.Parameter(p0.clone())
    opt = torch.optim.AdamW([p], lr=1e-2, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)
    q, m, v = p0, torch.zeros(50).double(), torch.zeros(50).double()
    for step in range(1, 5):
        p.grad = torch.randn(50, generator=g, dtype=torch.float64)
        q, m, v = B.adamw8_step(q, p.grad, m, v, step, 1e-2, 0.9, 0.95, 1e-8, 0.1)
        opt.step()
        assert torch.allclose(p.detach(), q, rtol=1e-12, atol=1e-14)


def test_errors_of_the_experts_cover_a_computation_in_fp32():
    g = torch.Generator().manual_seed(2)
    E, H, I, counts = 2, 160, 136, [3, 4]
    w1, w3 = (torch.randn(E, I, H, generator=g) * 0.1 for _ in range(2))
    w2 = torch.randn(E, H, I, generator=g) * 0.1
    x, d_y = (torch.randn(7, H, generator=g).bfloat16() for _ in range(2))
    exact = B.experts(w1, w2, w3, x, counts, d_y)
    for (name, (value, err, deviation)), want in zip(B.experts_between(w1, w2, w3, x, counts, d_y).items(), exact):
        assert torch.allclose(value, want, rtol=1e-9, atol=1e-12), name
        # a fraction of the size of what is tested, or the bounds would test nothing
        assert err.norm() < 0.4 * value.norm() and deviation.norm() < 0.06 * value.norm(), name
