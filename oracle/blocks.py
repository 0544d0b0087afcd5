"""8-bit block formats, the experts' products and the AdamW step on them, restated in float64 on the CPU (test infrastructure;
no counterpart in the reference).  Values, not codes: a quantized tensor is what its codes and scales stand for."""
from __future__ import annotations

import functools
import math

import torch

BLOCK, STATE_BLOCK = 128, 64


def two_to(k: torch.Tensor) -> torch.Tensor:
    return torch.ldexp(torch.ones_like(k, dtype=torch.float64), k.to(torch.int32))


def scale_exponent(amax: torch.Tensor, largest: float) -> torch.Tensor:
    """Smallest integer k >= -126 with amax <= largest * 2^k (amax float64, largest 1.75 times a power of two)."""
    m, e = torch.frexp(amax / largest)                     # exact up to the division; corrected below
    k = e.to(torch.int64)
    for d in (1, 0, -1, -2):                               # largest candidate first
        k = torch.where(amax <= largest * two_to(e + d), e + d, k)
    return torch.where(amax == 0, torch.full_like(k, -126), k).clamp(min=-126)


def grid_step(t: torch.Tensor, mantissa: int, bias: int) -> torch.Tensor:
    """Distance of neighbouring values of the format at magnitude t."""
    _, e = torch.frexp(t)
    return two_to(torch.clamp(e.to(torch.int64) - 1, min=1 - bias) - mantissa)


def nearest(x: torch.Tensor, mantissa: int = 3, bias: int = 7) -> torch.Tensor:
    step = grid_step(x.abs(), mantissa, bias)
    return torch.round(x / step) * step                    # torch.round: ties to even, as the formats do


def quantize(x: torch.Tensor, dims) -> tuple[torch.Tensor, torch.Tensor]:
    """x already cut into blocks (the dimensions `dims`): (values in units of the scale, exponents)."""
    amax = x.abs().amax(dims, keepdim=True)
    k = scale_exponent(torch.where(torch.isfinite(amax), amax, torch.zeros_like(amax)), 448.0)
    bad = ~torch.isfinite(amax)
    q = nearest(x / two_to(k))
    return torch.where(bad, torch.full_like(q, math.nan), q), torch.where(bad, torch.zeros_like(k), k)


def rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [R,K] -> (codes as values [R,K'], exponents [R,K'/128])."""
    R, K = x.shape
    pad = torch.nn.functional.pad(x.double(), (0, -K % BLOCK)).view(R, -1, BLOCK)
    q, k = quantize(pad, (2,))
    return q.view(R, -1), k.view(R, -1)


def rounded_rows(x: torch.Tensor) -> torch.Tensor:
    q, k = rows(x)
    return (q.view(*k.shape, BLOCK) * two_to(k)[..., None]).view(x.shape[0], -1)[:, :x.shape[1]]


def weights(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """w [E,N,K] -> (codes as values [E,N',K'], exponents [E,N'/128,K'/128])."""
    E, N, K = w.shape
    p = torch.nn.functional.pad(w.double(), (0, -K % BLOCK, 0, -N % BLOCK))
    n, k = p.shape[1] // BLOCK, p.shape[2] // BLOCK
    q, e = quantize(p.view(E, n, BLOCK, k, BLOCK), (2, 4))
    return q.view(E, n * BLOCK, k * BLOCK), e.view(E, n, k)


def rounded_weights(w: torch.Tensor) -> torch.Tensor:
    q, e = weights(w)
    s = two_to(e).repeat_interleave(BLOCK, 1).repeat_interleave(BLOCK, 2)
    return (q * s)[:, :w.shape[1], :w.shape[2]]


def experts(w1, w2, w3, x, counts, d_y=None):
    """y, or with d_y (y, d_x, d_w1, d_w2, d_w3), in float64; gate, up and their gradients are held in bfloat16."""
    held = lambda t: t.to(torch.bfloat16).double()  # noqa: E731
    v1, v2, v3 = (rounded_weights(w) for w in (w1, w2, w3))
    y = torch.zeros(x.shape[0], x.shape[1], dtype=torch.float64)
    d_x, g1, g2, g3 = torch.zeros_like(y), *(torch.zeros(w.shape, dtype=torch.float64) for w in (w1, w2, w3))
    start = 0
    for e, n in enumerate(int(c) for c in counts):
        r = slice(start, start + n)
        start += n
        if n == 0:
            continue
        xr = rounded_rows(x[r])
        g, u = held(xr @ v1[e].t()), held(xr @ v3[e].t())
        sg = torch.sigmoid(g)
        h = g * sg * u
        y[r] = rounded_rows(h) @ v2[e].t()
        if d_y is None:
            continue
        d_h = rounded_rows(d_y[r]) @ v2[e]
        d_g, d_u = held(d_h * u * sg * (1 + g * (1 - sg))), held(d_h * g * sg)
        d_x[r] = rounded_rows(d_g) @ v1[e] + rounded_rows(d_u) @ v3[e]
        g1[e], g2[e], g3[e] = d_g.t() @ x[r].double(), d_y[r].double().t() @ held(h), d_u.t() @ x[r].double()
    return y if d_y is None else (y, d_x, g1, g2, g3)


# ------------------------------------------------------------------------------ AdamW with 8-bit moments
def random_bits(n: int, seed: int, first: int = 0) -> torch.Tensor:
    out = []
    for i in range(first, first + n):
        h = (i * 0x6A09E667 + seed) % 2 ** 32
        h ^= h >> 16
        h = h * 0xBB67AE85 % 2 ** 32
        h ^= h >> 15
        h = h * 0x9E3779B1 % 2 ** 32
        out.append(h ^ (h >> 16))
    return torch.tensor(out, dtype=torch.int64)


def encode(x: torch.Tensor, random16: torch.Tensor, mantissa: int) -> tuple[torch.Tensor, torch.Tensor]:
    """x [n] (float64) in blocks of 64 -> (codes as values [n], exponents): rounded up where the part below a step exceeds
    1 - random16 / 65536.  Elements that are not finite become NaN and do not count for the scale."""
    bias, largest = (7, 448.0) if mantissa == 3 else (15, 57344.0)
    n = x.numel()
    finite = torch.isfinite(x)
    a = torch.where(finite, x.abs(), torch.zeros_like(x))
    k = scale_exponent(torch.nn.functional.pad(a, (0, -n % STATE_BLOCK)).view(-1, STATE_BLOCK).amax(1), largest)
    t = a / two_to(k).repeat_interleave(STATE_BLOCK)[:n]
    step = grid_step(t, mantissa, bias)
    c = torch.floor(t / step + random16.double() / 65536)
    if mantissa == 2:
        c = torch.where((t > 0) & (c == 0), torch.ones_like(c), c)
    v = c * step * torch.where(torch.signbit(x), -1.0, 1.0)
    return torch.where(finite, v, torch.full_like(v, math.nan)), k


def adamw8_step(p, g, m, v, step, lr, beta1, beta2, eps, weight_decay):
    """(p, m, v) after one step in float64, the moments before they are stored."""
    p, g, m, v = (t.double() for t in (p, g, m, v))
    m = beta1 * m + (1 - beta1) * g
    v = beta2 * v + (1 - beta2) * g * g
    p = p * (1 - lr * weight_decay)
    return p - lr * (m / (1 - beta1 ** step)) / (torch.sqrt(v / (1 - beta2 ** step)) + eps), m, v


# ------------------------------------------------------------------------------ how far a computation in fp32 may be off
# Every function takes and gives (value, error): the value in float64 and what a computation in fp32 can differ by.  A rounding
# is monotonous, so what it makes of a value that is off by at most `err` lies between what it makes of value - err and value + err.
U32, U16 = 2.0 ** -24, 2.0 ** -8          # half a step of fp32 and of bfloat16, relative


def held_between(x, err):
    h = lambda t: t.to(torch.float32).to(torch.bfloat16).double()  # noqa: E731  (the oracle's values fit fp32 well enough: err covers it)
    v = h(x)
    return v, torch.maximum((h(x + err + U32 * x.abs()) - v).abs(), (v - h(x - err - U32 * x.abs())).abs())


def rounded_rows_between(x, err):
    """(value, error, 2^-6 of the scale: the least exponent of a normal code)."""
    R, K = x.shape
    pad = lambda t: torch.nn.functional.pad(t, (0, -K % BLOCK)).view(R, -1, BLOCK)  # noqa: E731
    x, err = pad(x), pad(err)
    k = scale_exponent(x.abs().amax(2, keepdim=True), 448.0)
    least = scale_exponent((x.abs() - err).clamp(min=0).amax(2, keepdim=True), 448.0)
    most = scale_exponent((x.abs() + err).amax(2, keepdim=True), 448.0)
    v = nearest(x / two_to(k)) * two_to(k)
    off = torch.zeros_like(v)
    for kk in (least, k, most):
        for t in (x - err, x + err):
            off = torch.maximum(off, (nearest(t / two_to(kk)) * two_to(kk) - v).abs())
    return tuple(t.reshape(R, -1)[:, :K] for t in (v, off, two_to(most - 6).expand_as(v)))


def weights_with_floor(w):
    """([E,N,K] values, 2^-6 of their scales)."""
    _, e = weights(w)
    s = two_to(e - 6).repeat_interleave(BLOCK, 1).repeat_interleave(BLOCK, 2)
    return rounded_weights(w), s[:, :w.shape[1], :w.shape[2]]


GROUP, GROUP_BITS = 8, 13


def product_between(a, b, decoded=False):
    """a @ b for a = (value, error, floor), b = (value, floor), as the matrix instructions form it.  Those for codes align the products
    of GROUP neighbouring values to the largest exponent among them and keep GROUP_BITS bits below it, which loses at most
    2^-GROUP_BITS of that power of two for each (a code below the normal ones counts with the least normal exponent), and add
    such sums up in fp32 in some order.  Those for decoded values add exact products up in fp32."""
    (v, err, floor), (w, w_floor) = a, b
    K = v.shape[1]
    size = v.abs() @ w.abs() + err @ w.abs()
    lost = K * U32 * size
    top, w_top = torch.maximum(v.abs() + err, floor), torch.maximum(w.abs(), w_floor)
    for k in range(0, 0 if decoded else K, GROUP):
        lost += GROUP * 2.0 ** -GROUP_BITS * (top[:, k:k + GROUP, None] * w_top[None, k:k + GROUP]).amax(1)
    # and the deviation if the errors of the summands have nothing to do with each other
    return v @ w, err @ w.abs() + lost, (err.square() @ w.square() + lost.square()).sqrt()


def exactly(x):
    """Rows of codes that are known exactly, as product_between takes them."""
    return rounded_rows_between(x.double(), torch.zeros(x.shape, dtype=torch.float64))


def experts_between(w1, w2, w3, x, counts, d_y=None, decoded=False):
    """experts() with the error of every output: {name: (value, error, deviation)}, names y, d_x, d_w1, d_w2, d_w3.  The error is what a
    value can be off by if every uncertain rounding falls the wrong way with the same sign; the deviation takes the summands'
    errors as unrelated, and bounds the 2-norm over a whole output.  decoded: see product_between."""
    product = functools.partial(product_between, decoded=decoded)
    zero = torch.zeros_like
    (v1, f1), (v2, f2), (v3, f3) = (weights_with_floor(w) for w in (w1, w2, w3))
    names = ("y",) if d_y is None else ("y", "d_x", "d_w1", "d_w2", "d_w3")
    shapes = dict(y=x.shape, d_x=x.shape, d_w1=w1.shape, d_w2=w2.shape, d_w3=w3.shape)
    out = {n: tuple(torch.zeros(shapes[n], dtype=torch.float64) for _ in range(3)) for n in names}

    def put(name, at, value, err, dev):                     # the last rounding, to bfloat16
        out[name][0][at], out[name][1][at] = value, err + U16 * (value.abs() + err)
        out[name][2][at] = (dev.square() + (U16 * (value.abs() + dev)).square()).sqrt()

    start = 0
    for e, n in enumerate(int(c) for c in counts):
        r = slice(start, start + n)
        start += n
        if n == 0:
            continue
        xr = exactly(x[r])
        g, ge = held_between(*product(xr, (v1[e].t(), f1[e].t()))[:2])
        u, ue = held_between(*product(xr, (v3[e].t(), f3[e].t()))[:2])
        sg = torch.sigmoid(g)
        # silu has a slope of at most 1.1; exponential, sum, reciprocal and two products are within 12 half steps together, and an
        # exponential's argument of size |g| moves it by |g| half steps
        h = g * sg * u
        he = 1.1 * ge * (u.abs() + ue) + (g * sg).abs() * ue + (12 + g.abs()) * U32 * h.abs()
        put("y", r, *product(rounded_rows_between(h, he), (v2[e].t(), f2[e].t())))
        if d_y is None:
            continue
        d_h, de, _ = product(exactly(d_y[r]), (v2[e], f2[e]))
        slope = sg * (1 + g * (1 - sg))
        # slope is within 1.1 and has a slope of at most 1/2; its parts are at most 1 + |g| and rounded a dozen times
        rough = (16 + g.abs()) * U32 * (1 + g.abs())
        d_g = d_h * u * slope
        dge = 1.1 * (de * (u.abs() + ue) + d_h.abs() * ue) + (d_h * u).abs() * (0.5 * ge + rough)
        d_u = d_h * g * sg
        due = de * ((g * sg).abs() + 1.1 * ge) + d_h.abs() * (1.1 * ge) + (d_h * g).abs() * (16 + g.abs()) * U32
        d_g, dge = held_between(d_g, dge)
        d_u, due = held_between(d_u, due)
        a, ae, ad = product(rounded_rows_between(d_g, dge), (v1[e], f1[e]))
        b, be, bd = product(rounded_rows_between(d_u, due), (v3[e], f3[e]))
        sums = I_SUMS * U32 * (a.abs() + b.abs())
        put("d_x", r, a + b, ae + be + sums, (ad.square() + bd.square() + sums.square()).sqrt())
        xd = x[r].double()
        hb, hbe = held_between(h, he)
        for name, (left, le, right, re) in dict(d_w1=(d_g, dge, xd, zero(xd)), d_w3=(d_u, due, xd, zero(xd)),
                                                d_w2=(d_y[r].double(), zero(d_y[r].double()), hb, hbe)).items():
            sums = n * U32 * (left.abs().t() @ right.abs())
            put(name, e, left.t() @ right, le.t() @ right.abs() + left.abs().t() @ re + sums,
                (le.t().square() @ right.square() + left.t().square() @ re.square() + sums.square()).sqrt())
    return out


I_SUMS = 8        # d_x adds its two products' partial sums in one accumulator: a few more roundings of the whole
