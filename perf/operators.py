"""The eight-bit operators of a training stage, as cases that can be timed and compared.

Four operators, each through the entry points that a program calls:

* ``serve``: the SwiGLU experts on expert-sorted rows with weights and activations in 8-bit floating point
  and a scale for each block of 128, without a backward;
* ``train``: the same with its backward: the gradient of the rows through 8-bit products, those of the three
  weights from the rows as they came;
* ``quantize``: the weights of a layer's experts into those blocks (row-major and transposed);
* ``adamw``: one AdamW step over the tensors of a bucket with both moments in 8-bit floating point, from the
  bucket's fp32 gradients (``packed`` false) or from the tensors' own gradients (``packed`` true).

Where ``own`` is false they are computed from elementary torch operations in 32 bits.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
WIDE = dict(hidden=2048, experts=128, top_k=8, inter=768)      # the benchmark's expert region
BLOCK = 128                                                    # values of a row that share a scale (weights: 128 x 128)
STATE_BLOCK = 64                                               # values of an AdamW moment that share a scale
ADAMW = dict(lr=1e-3, beta1=0.9, beta2=0.95, eps=1e-8, weight_decay=0.1)

# what the largest listed cases cost; no drawn case costs more
_MAX_ROW_FLOPS = 18 * 2048 * 768 * 65536
_MAX_WEIGHTS = 3 * 128 * 768 * 2048
_MAX_ELEMENTS = 170e6


def listed() -> list[dict]:
    return [
        # one sequence being decoded: launches and the weights of eight experts
        dict(name="serve_1", kind="serve", tokens=1, spare=0, skew=0.0, dtype="bf16", **WIDE),
        # a decode batch: every expert has a row or two, so the weights are the traffic
        dict(name="serve_24", kind="serve", tokens=24, spare=0, skew=0.0, dtype="bf16", **WIDE),
        # the prompt of one request, of no particular length
        dict(name="serve_1777", kind="serve", tokens=1777, spare=0, skew=0.0, dtype="bf16", **WIDE),
        # the benchmark's microbatch, evenly routed
        dict(name="train_4096", kind="train", tokens=4096, spare=0, skew=0.0, dtype="bf16", **WIDE),
        # a long microbatch with Zipf-distributed expert popularity
        dict(name="train_8192_skewed", kind="train", tokens=8192, spare=0, skew=0.45, dtype="bf16", **WIDE),
        # widths that are no multiple of a block, and rows that no expert owns
        dict(name="train_ragged_widths", kind="train", tokens=1030, spare=37, skew=0.0, dtype="bf16", hidden=1000, experts=24, top_k=4,
             inter=360),
        # a layer's expert weights after an optimizer step
        dict(name="quantize_layer", kind="quantize", dtype="bf16", hidden=2048, experts=128, inter=768),
        # those of a small fp32 model with odd widths
        dict(name="quantize_odd_f32", kind="quantize", dtype="f32", hidden=1000, experts=24, inter=363),
        # a small stage: launches count
        dict(name="adamw_small", kind="adamw", packed=True, tensors=24, elements=300_000, grad="bf16"),
        # two decoder layers' worth of bf16 parameters, the last gradients not packed
        dict(name="adamw_bucket", kind="adamw", packed=True, tensors=96, elements=160_000_000, grad="bf16"),
        # fp32 parameters whose gradients are a flat buffer
        dict(name="adamw_flat_f32", kind="adamw", packed=False, tensors=40, elements=30_000_000, grad="f32"),
    ]


def _log(rng: random.Random, lo: float, hi: float) -> float:
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["serve", "serve", "train", "train", "quantize", "adamw"])
    if kind == "adamw":
        return dict(kind=kind, packed=rng.random() < 0.6, tensors=rng.randint(1, 150), elements=int(_log(rng, 20_000, 160e6)),
                    grad=rng.choice(["bf16", "bf16", "f32"]))
    hidden = rng.choice([8 * rng.randint(16, 384), 128 * rng.randint(2, 24), rng.randint(130, 2100)])
    inter = rng.choice([8 * rng.randint(16, 192), 128 * rng.randint(1, 12), rng.randint(130, 1100)])
    experts = rng.choice([4, 8, 16, 24, 64, 128])
    experts = max(1, min(experts, int(_MAX_WEIGHTS / (3 * hidden * inter))))
    if kind == "quantize":
        return dict(kind=kind, dtype=rng.choice(["bf16", "bf16", "f32"]), hidden=hidden, experts=experts, inter=inter)
    top_k = rng.randint(1, min(8, experts))
    most = min(4096.0 if kind == "serve" else 8192.0, _MAX_ROW_FLOPS / (18 * hidden * inter * top_k), 65536 / top_k)
    tokens = int(_log(rng, 1, max(2.0, most)))
    return dict(kind=kind, tokens=tokens, spare=rng.choice([0, 0, rng.randint(1, 90)]), skew=rng.choice([0.0, 0.0, rng.uniform(0.2, 0.6)]),
                dtype="bf16", hidden=hidden, experts=experts, top_k=top_k, inter=inter)


# ------------------------------------------------------------------------------------------------ inputs
def _up(n: int, m: int) -> int:
    return -(-n // m) * m


def _shapes(case: dict) -> list[int]:
    """Element counts of a bucket's tensors: matrices of two widths, vectors, and odd ones."""
    share = [(1.0, 0.4, 0.004, 0.07, 0.7)[i % 5] for i in range(case["tensors"])]
    unit = case["elements"] / sum(share)
    return [max(1, int(unit * s) // (128 if i % 3 else 1) * (128 if i % 3 and int(unit * s) >= 128 else 1)) for i, s in enumerate(share)]


def _counts(case: dict, gen: torch.Generator, dev) -> torch.Tensor:
    """Rows of every expert: top_k different experts for each token, the first experts the more popular with a skew."""
    E = case["experts"]
    popular = -2.4 * case["skew"] * torch.log(torch.arange(1, E + 1, device=dev, dtype=torch.float32))
    noise = -torch.log(-torch.log(torch.rand((case["tokens"], E), generator=gen, device=dev).clamp(1e-6, 1 - 1e-6)))
    chosen = torch.topk(popular + noise, case["top_k"], dim=1).indices
    return torch.bincount(chosen.reshape(-1), minlength=E).to(torch.int32)


def prepare(case: dict, seed: int):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    if case["kind"] == "adamw":
        return _prepare_adamw(case, seed, gen, dev)
    dt = DTYPES[case["dtype"]]
    E, I, H = case["experts"], case["inter"], case["hidden"]
    w1, w3 = ((torch.randn((E, I, H), generator=gen, device=dev) * 0.02).to(dt) for _ in range(2))
    w2 = (torch.randn((E, H, I), generator=gen, device=dev) * 0.02).to(dt)
    if case["kind"] == "quantize":
        return dict(case=case, w=(w1, w2, w3))
    train = case["kind"] == "train"
    counts = _counts(case, gen, dev)
    rows = case["tokens"] * case["top_k"] + case["spare"]
    x = torch.randn((rows, H), generator=gen, device=dev).to(dt)
    state = dict(case=case, counts=counts, x=x, w=(w1, w2, w3), blocks=_blocks_of_weights((w1, w2, w3), train))
    # where a row sits if every expert gets as many rows as the largest one, over the experts that have any
    host = counts.cpu()
    state["active"] = torch.nonzero(host).reshape(-1).to(dev)
    state["most"], state["owned"] = max(1, int(host.max())), int(host.sum())
    if train:
        state["d_y"] = torch.randn((rows, H), generator=gen, device=dev).to(dt)
        for t in (x, w1, w2, w3):
            t.requires_grad_(True)
    return state


def _prepare_adamw(case, seed, gen, dev):
    numels = _shapes(case)
    gdt = DTYPES[case["grad"]]
    offsets, end = [], 0
    for n in numels:
        offsets.append(end)
        end = _up(end + n, 128)
    live = torch.zeros(end, dtype=torch.bool, device=dev)
    grads = []
    for o, n in zip(offsets, numels):
        live[o:o + n] = True
        grads.append((torch.randn(n, generator=gen, device=dev) * 1e-3).to(gdt))
    master = torch.randn(end, generator=gen, device=dev) * 0.02 * live
    m = torch.randn(end, generator=gen, device=dev) * 3e-4 * live
    v = (torch.randn(end, generator=gen, device=dev) * 1e-3).square() * live
    half = torch.full((end,), 0x8000, dtype=torch.int64, device=dev)
    m8, ms = _encode(m, half, 3)
    v8, vs = _encode(v, half, 2)
    state = dict(case=case, master=master, exp_avg=m8, exp_avg_scale=ms, exp_avg_sq=v8, exp_avg_sq_scale=vs, offsets=offsets,
                 numels=numels, step=100, seed=seed & 0xFFFF, flat=None, grads=None, shadow=None)
    if case["packed"]:
        state["grads"], state["shadow"] = grads, master.to(torch.bfloat16)
    else:
        flat = torch.zeros(end, device=dev)
        for o, n, g in zip(offsets, numels, grads):
            flat[o:o + n] = g.float()
        state["flat"] = flat
    return state


# ------------------------------------------------------------------------------------------------ block formats
# A scale is a power of two, held as its biased exponent in 8 bits: the smallest with which the block's largest
# magnitude is at most 1.75 * 2^top, the largest value of the format (e4m3: 448, top 8; e5m2: 57344, top 15).
def _scale_byte(amax: torch.Tensor, top: int) -> torch.Tensor:
    bits = amax.contiguous().view(torch.int32).to(torch.int64)
    return ((bits >> 23) - top + ((bits & 0x7FFFFF) > 0x600000)).clamp(min=1)


def _power(byte: torch.Tensor) -> torch.Tensor:
    """2^(byte - 127) as fp32, for bytes of 1 to 254."""
    return (byte.to(torch.int32) << 23).view(torch.float32)


def _quantize(blocks: torch.Tensor, dims) -> tuple[torch.Tensor, torch.Tensor]:
    """(e4m3 values, scale bytes) of fp32 values whose blocks are the dimensions `dims`."""
    byte = _scale_byte(blocks.abs().amax(dims, keepdim=True), 8)
    return (blocks * _power(254 - byte)).to(torch.float8_e4m3fn), byte


def _e8m0(byte: torch.Tensor) -> torch.Tensor:
    return byte.to(torch.uint8).view(torch.float8_e8m0fnu)


def _rows_in_blocks(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """A row's values in blocks of 128: (values as fp32 with the scale left out, their scale bytes)."""
    R, K = x.shape
    x = torch.nn.functional.pad(x.float(), (0, _up(K, BLOCK) - K)).view(R, -1, BLOCK)
    q, byte = _quantize(x, (2,))
    return q, byte


def _rounded_rows(x: torch.Tensor) -> torch.Tensor:
    """What the 8-bit blocks of x's rows stand for, in fp32."""
    q, byte = _rows_in_blocks(x)
    return (q.float() * _power(byte)).view(x.shape[0], -1)[:, :x.shape[1]]


def _weight_in_blocks(w: torch.Tensor):
    """w [E, N, K] in blocks of 128 x 128: row-major [E, N, K'] and transposed [E, K, N'] (rows padded with zeros to whole
    blocks), scales [E, N / 128, K / 128]."""
    E, N, K = w.shape
    n, k = _up(N, BLOCK), _up(K, BLOCK)
    p = torch.nn.functional.pad(w.detach().float(), (0, k - K, 0, n - N)).view(E, n // BLOCK, BLOCK, k // BLOCK, BLOCK)
    q, byte = _quantize(p, (2, 4))
    q = q.view(torch.uint8).view(E, n, k)
    return (q[:, :N].contiguous().view(torch.float8_e4m3fn), q.transpose(1, 2)[:, :K].contiguous().view(torch.float8_e4m3fn),
            _e8m0(byte.view(E, n // BLOCK, k // BLOCK)))


def _blocks_of_weights(ws, transposed: bool):
    got = [_weight_in_blocks(w) for w in ws]
    return dict(q=[g[0] for g in got], t=[g[1] if transposed else None for g in got], s=[g[2] for g in got])


def _values(q: torch.Tensor, s: torch.Tensor, rows: int, cols: int) -> torch.Tensor:
    """fp32 values of row-major weight blocks."""
    scale = _power(s.view(torch.uint8)).repeat_interleave(BLOCK, 1).repeat_interleave(BLOCK, 2)
    return q.float()[:, :, :cols] * scale[:, :rows, :cols]


# ------------------------------------------------------------------------------------------------ the experts
def _places(state):
    """Row and column of every owned row in [active experts, most rows]."""
    counts = state["counts"].to(torch.int64)[state["active"]]
    starts = counts.cumsum(0) - counts
    e = torch.repeat_interleave(torch.arange(counts.numel(), device=counts.device), counts, output_size=state["owned"])
    return e, torch.arange(state["owned"], device=counts.device) - starts[e]


def _spread(x, at, state):
    out = x.new_zeros((state["active"].numel(), state["most"], x.shape[1]))
    out[at] = x[:state["owned"]]
    return out


def _plain_experts(state):
    """y and, for the backward, what it needs: every row times its expert's three matrices, fp32 sums of the values that the
    8-bit blocks stand for; gate and up are held in the rows' type."""
    x, active, case = state["x"].detach(), state["active"], state["case"]
    H, I, dt = case["hidden"], case["inter"], x.dtype
    q, s = state["blocks"]["q"], state["blocks"]["s"]
    v1, v2, v3 = (_values(q[i][active], s[i][active], *shape) for i, shape in enumerate(((I, H), (H, I), (I, H))))
    at = _places(state)
    xs = _spread(_rounded_rows(x), at, state)
    g = torch.bmm(xs, v1.transpose(1, 2).contiguous())[at].to(dt).float()
    u = torch.bmm(xs, v3.transpose(1, 2).contiguous())[at].to(dt).float()
    h = g / (1 + torch.exp(-g)) * u
    hs = _spread(_rounded_rows(h), at, state)
    y = torch.zeros((x.shape[0], H), dtype=dt, device=x.device)
    y[:state["owned"]] = torch.bmm(hs, v2.transpose(1, 2).contiguous())[at].to(dt)
    return y, g, u, h, at, (v1, v2, v3)


def _plain_train(state):
    y, g, u, h, at, (v1, v2, v3) = _plain_experts(state)
    x, d_y, active, n = state["x"].detach(), state["d_y"], state["active"], state["owned"]
    dt = x.dtype
    d_h = torch.bmm(_spread(_rounded_rows(d_y), at, state), v2)[at]
    sg = 1 / (1 + torch.exp(-g))
    d_g = (d_h * u * (sg * (1 + g * (1 - sg)))).to(dt)
    d_u = (d_h * (g * sg)).to(dt)
    rows = torch.bmm(_spread(_rounded_rows(d_g), at, state), v1) + torch.bmm(_spread(_rounded_rows(d_u), at, state), v3)
    d_x = torch.zeros_like(x)
    d_x[:n] = rows[at].to(dt)

    def weight_grad(like, left, right):
        out = torch.zeros(like.shape, dtype=dt, device=x.device)
        out[active] = torch.bmm(_spread(left.float(), at, state).transpose(1, 2).contiguous(), _spread(right.float(), at, state)).to(dt)
        return out

    w1, w2, w3 = state["w"]
    return y, d_x, weight_grad(w1, d_g, x), weight_grad(w2, d_y, h.to(dt)), weight_grad(w3, d_u, x)


# ------------------------------------------------------------------------------------------------ AdamW with 8-bit moments
_MASK = 0xFFFFFFFF


def _random_bits(n: int, seed: int, dev) -> torch.Tensor:
    """32 bits for each element of a bucket, from its index and the seed of the step."""
    h = (torch.arange(n, dtype=torch.int64, device=dev) * 0x6A09E667 + seed) & _MASK
    h = h ^ (h >> 16)
    h = (h * 0xBB67AE85) & _MASK
    h = h ^ (h >> 15)
    h = (h * 0x9E3779B1) & _MASK
    return h ^ (h >> 16)


def _encode(x: torch.Tensor, random16: torch.Tensor, mantissa: int):
    """fp32 [n] in blocks of 64: e4m3 (mantissa 3) or e5m2 (mantissa 2), rounded down or up with random16 / 65536 as the
    threshold, so that the mean is x; a positive e5m2 value (a second moment) does not become zero."""
    bias, top, drop = (7, 8, 20) if mantissa == 3 else (15, 15, 21)
    n = x.numel()
    byte = _scale_byte(torch.nn.functional.pad(x.abs(), (0, _up(n, STATE_BLOCK) - n)).view(-1, STATE_BLOCK).amax(1), top)
    t = x.abs() * _power(254 - byte).repeat_interleave(STATE_BLOCK)[:n]
    bits = t.view(torch.int32).to(torch.int64)
    normal = ((bits + (random16 << (drop - 16))) >> drop) - ((127 - bias) << mantissa)
    small = torch.floor(t * 2.0 ** (bias - 1 + mantissa) + random16.float() * 2.0 ** -16).to(torch.int64)
    code = torch.where(t < 2.0 ** (1 - bias), small, normal)
    if mantissa == 2:
        code = torch.where((t > 0) & (code == 0), 1, code)
    code = (code | (torch.signbit(x).to(torch.int64) << 7)).to(torch.uint8)
    return code.view(torch.float8_e4m3fn if mantissa == 3 else torch.float8_e5m2), _e8m0(byte)


def _decode(code, scale, n):
    return code.float() * _power(scale.view(torch.uint8)).repeat_interleave(STATE_BLOCK)[:n]


def _flat_grad(state):
    """The gradient of every element of the bucket in fp32 (zeros between the tensors)."""
    if state["flat"] is not None:
        return state["flat"]
    n, offsets = state["master"].numel(), state["offsets"]
    ends = offsets[1:] + [n]
    return torch.cat([torch.nn.functional.pad(g.float(), (0, e - o - k))
                      for g, o, e, k in zip(state["grads"], offsets, ends, state["numels"])])


def _plain_adamw(state):
    a, n, step = ADAMW, state["master"].numel(), state["step"]
    p = state["master"]
    g = _flat_grad(state)
    m = _decode(state["exp_avg"], state["exp_avg_scale"], n)
    v = _decode(state["exp_avg_sq"], state["exp_avg_sq_scale"], n)
    p = p * (1 - a["lr"] * a["weight_decay"])
    m = m + (g - m) * (1 - a["beta1"])
    v = v * a["beta2"] + ((1 - a["beta2"]) * g) * g
    denom = v.sqrt() * (1 / math.sqrt(1 - a["beta2"] ** step)) + a["eps"]
    p = p - (a["lr"] / (1 - a["beta1"] ** step)) * (m / denom)
    bits = _random_bits(n, state["seed"] + step, p.device)
    m8, ms = _encode(m, bits >> 16, 3)
    v8, vs = _encode(v, bits & 0xFFFF, 2)
    for name, new in (("exp_avg", m8), ("exp_avg_scale", ms), ("exp_avg_sq", v8), ("exp_avg_sq_scale", vs)):
        state[name].view(torch.uint8).copy_(new.view(torch.uint8))
    state["master"].copy_(p)
    if state["shadow"] is not None:
        state["shadow"].copy_(p)


def _updated(state):
    out = {k: state[k] for k in ("master", "exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_scale")}
    if state["shadow"] is not None:
        out["shadow"] = state["shadow"]
    return out


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    kind = state["case"]["kind"]
    if own:
        return _run_own(state, kind)
    if kind == "quantize":
        got = _blocks_of_weights(state["w"], True)
        return got["q"] + got["t"] + got["s"]
    if kind == "serve":
        return _plain_experts(state)[0]
    if kind == "train":
        return _plain_train(state)
    state["step"] += 1
    _plain_adamw(state)
    return _updated(state)


def _run_own(state, kind):
    from piper_amd import functional as F_
    from piper_amd import ops

    if kind == "quantize":
        e = F_.quantize_experts(*state["w"])
        return [e.q1, e.q2, e.q3, e.t1, e.t2, e.t3, e.s1, e.s2, e.s3]
    if kind in ("serve", "train"):
        (w1, w2, w3), b = state["w"], state["blocks"]
        experts = F_.Fp8Experts(w1, w2, w3, *b["q"], *b["s"], *b["t"])
        y = F_.bmm_experts_fp8(experts, state["x"], state["counts"])
        if kind == "serve":
            return y
        return (y.detach(), *torch.autograd.grad(y, (state["x"], w1, w2, w3), state["d_y"]))
    state["step"] += 1
    moments = [state[k] for k in ("exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_scale")]
    how = dict(ADAMW, step=state["step"], seed=state["seed"] + state["step"], shadow=state["shadow"])
    if state["grads"] is not None:
        ops.adamw8_fused_packed(state["master"], *moments, None, state["grads"], state["offsets"], state["numels"], **how)
    else:
        ops.adamw8_fused(state["master"], *moments, state["flat"], **how)
    return _updated(state)


def work(case: dict) -> dict:
    kind = case["kind"]
    if kind == "adamw":
        n = sum(_shapes(case))
        grad = 4 if case["grad"] == "f32" or not case["packed"] else 2
        return dict(bytes=n * (8 + 4 + 4 / STATE_BLOCK + grad + (2 if case["packed"] else 0)), flops=20.0 * n)
    E, I, H = case["experts"], case["inter"], case["hidden"]
    e = 4 if case["dtype"] == "f32" else 2
    if kind == "quantize":
        return dict(bytes=3 * E * I * H * (e + 2 + 1 / BLOCK ** 2), flops=3.0 * E * I * H)
    rows = case["tokens"] * case["top_k"]
    active = E * (1 - (1 - case["top_k"] / E) ** case["tokens"])
    if kind == "serve":
        return dict(bytes=active * 3 * I * H + 2 * rows * H * e, flops=6.0 * rows * H * I)
    return dict(bytes=active * 6 * I * H + 3 * E * I * H * e + 4 * rows * H * e, flops=18.0 * rows * H * I)


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def _two_to(k: torch.Tensor) -> torch.Tensor:
    """2^k exactly (a general power may be a rounding off, and a value on the border of two scales then gets the wrong one)."""
    return ((k.to(torch.int64) + 1023) << 52).view(torch.float64)


def _codes64(mantissa: int, bias: int, top: float) -> torch.Tensor:
    """The values of an 8-bit format that are not negative, by code."""
    codes = torch.arange(128, dtype=torch.float64)
    e, f = torch.floor(codes / 2 ** mantissa), codes % 2 ** mantissa
    v = torch.where(e == 0, f * 2.0 ** (1 - bias - mantissa), (1 + f / 2 ** mantissa) * _two_to(e - bias))
    return v[v <= top]


def _exponent64(amax: torch.Tensor, largest: float, least: int) -> torch.Tensor:
    """The smallest k with amax <= largest * 2^k, from `least` on."""
    k = torch.ceil(torch.log2(amax.clamp(min=1e-300) / largest))
    k = torch.where(amax > largest * _two_to(k), k + 1, k)
    k = torch.where(amax <= largest * _two_to(k - 1), k - 1, k)
    return k.clamp(min=least)


def _nearest64(x: torch.Tensor) -> torch.Tensor:
    """The nearest e4m3 value, ties to the even code."""
    v = _codes64(3, 7, 448.0).to(x.device)
    a = x.abs().contiguous()
    i = torch.bucketize(a, (v[1:] + v[:-1]) / 2)           # of a tie: the lower one
    tie = (i + 1 < v.numel()) & (a == (v[i] + v[(i + 1).clamp(max=v.numel() - 1)]) / 2) & (i % 2 == 1)
    return torch.sign(x) * v[i + tie.to(torch.int64)]


def _rows64(x: torch.Tensor) -> torch.Tensor:
    out = torch.empty_like(x)
    for c in range(0, x.shape[1], BLOCK):
        part = x[:, c:c + BLOCK]
        s = _two_to(_exponent64(part.abs().amax(1, keepdim=True), 448.0, -126))
        out[:, c:c + BLOCK] = _nearest64(part / s) * s
    return out


def _weight64(w: torch.Tensor):
    """Of one expert's matrix in 64 bits: (values with the scales left out, exponents of the scales)."""
    N, K = w.shape
    q = torch.empty_like(w)
    k = torch.empty((-(-N // BLOCK), -(-K // BLOCK)), dtype=w.dtype, device=w.device)
    for i in range(k.shape[0]):
        for j in range(k.shape[1]):
            at = (slice(i * BLOCK, (i + 1) * BLOCK), slice(j * BLOCK, (j + 1) * BLOCK))
            k[i, j] = _exponent64(w[at].abs().amax(), 448.0, -126)
            q[at] = w[at] / _two_to(k[i, j])
    return _nearest64(q), k


def _exact_experts(case, state):
    dt, I, H = state["x"].dtype, case["inter"], case["hidden"]
    train = case["kind"] == "train"
    x, (w1, w2, w3) = state["x"].detach(), (w.detach() for w in state["w"])
    q, s = state["blocks"]["q"], state["blocks"]["s"]

    def value(i, e, n, k):
        scale = _two_to(s[i][e].view(torch.uint8).to(torch.int64) - 127)
        return q[i][e].double()[:n, :k] * scale.repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]

    held = lambda t: t.to(dt).double()  # noqa: E731
    y = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    d_x, grads = torch.zeros_like(y), [torch.zeros(w.shape, dtype=dt, device=x.device) for w in (w1, w2, w3)] if train else []
    start = 0
    for e, n in enumerate(state["counts"].tolist()):
        if n == 0:
            continue
        r = slice(start, start + n)
        start += n
        a1, a2, a3 = value(0, e, I, H), value(1, e, H, I), value(2, e, I, H)
        xr = _rows64(x[r].double())
        g, u = held(xr @ a1.t()), held(xr @ a3.t())
        h = g * torch.sigmoid(g) * u
        y[r] = _rows64(h) @ a2.t()
        if not train:
            continue
        dy = state["d_y"][r].double()
        d_h = _rows64(dy) @ a2
        sg = torch.sigmoid(g)
        d_g, d_u = held(d_h * u * sg * (1 + g * (1 - sg))), held(d_h * g * sg)
        d_x[r] = _rows64(d_g) @ a1 + _rows64(d_u) @ a3
        grads[0][e] = (d_g.t() @ x[r].double()).to(dt)
        grads[1][e] = (dy.t() @ held(h)).to(dt)
        grads[2][e] = (d_u.t() @ x[r].double()).to(dt)
    return (y, d_x, *grads) if train else y


def _stochastic64(x: torch.Tensor, random16: torch.Tensor, mantissa: int, bias: int, largest: float):
    """(values in units of the scale, exponents) of blocks of 64."""
    n = x.numel()
    pad = torch.zeros(_up(n, STATE_BLOCK), dtype=x.dtype, device=x.device)
    pad[:n] = x.abs()
    k = _exponent64(pad.view(-1, STATE_BLOCK).amax(1), largest, -126)
    t = pad / _two_to(k).repeat_interleave(STATE_BLOCK)
    t = t[:n]
    e = torch.floor(torch.log2(t.clamp(min=1e-300)))
    e = torch.where(_two_to(e) > t, e - 1, torch.where(_two_to(e + 1) <= t, e + 1, e)).clamp(min=1 - bias)
    unit = _two_to(e - mantissa)
    c = torch.floor(t / unit + random16.double() / 65536)
    if mantissa == 2:
        c = torch.where((t > 0) & (c == 0), torch.ones_like(c), c)
    return torch.sign(x) * c * unit, k


def _exact_adamw(state):
    a, n, step = ADAMW, state["master"].numel(), state["step"] + 1
    p = state["master"].double()
    g = torch.zeros(n, dtype=torch.float64, device=p.device)
    if state["flat"] is not None:
        g += state["flat"]
    else:
        for o, k, t in zip(state["offsets"], state["numels"], state["grads"]):
            g[o:o + k] = t.double()

    def value(code, scale):
        s = _two_to(scale.view(torch.uint8).to(torch.int64) - 127)
        return code.double() * s.repeat_interleave(STATE_BLOCK)[:n]

    m = a["beta1"] * value(state["exp_avg"], state["exp_avg_scale"]) + (1 - a["beta1"]) * g
    v = a["beta2"] * value(state["exp_avg_sq"], state["exp_avg_sq_scale"]) + (1 - a["beta2"]) * g * g
    p = p * (1 - a["lr"] * a["weight_decay"])
    p = p - a["lr"] * (m / (1 - a["beta1"] ** step)) / (torch.sqrt(v / (1 - a["beta2"] ** step)) + a["eps"])
    bits = _random_bits(n, state["seed"] + step, p.device)
    m8, mk = _stochastic64(m, bits >> 16, 3, 7, 448.0)
    v8, vk = _stochastic64(v, bits & 0xFFFF, 2, 15, 57344.0)
    out = dict(master=p, exp_avg=m8, exp_avg_scale=_two_to(mk), exp_avg_sq=v8, exp_avg_sq_scale=_two_to(vk))
    if state["shadow"] is not None:
        out["shadow"] = p
    return out


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    if case["kind"] == "adamw":
        return _exact_adamw(state)
    if case["kind"] in ("serve", "train"):
        return _exact_experts(case, state)
    qs, ts, ss = [], [], []
    for w in state["w"]:
        E, N, K = w.shape
        q = torch.zeros((E, N, _up(K, BLOCK)), dtype=torch.float32, device=w.device)
        t = torch.zeros((E, K, _up(N, BLOCK)), dtype=torch.float32, device=w.device)
        s = torch.zeros((E, -(-N // BLOCK), -(-K // BLOCK)), dtype=torch.float32, device=w.device)
        for e in range(E):
            v, k = _weight64(w[e].double())
            q[e, :, :K], t[e, :, :N], s[e] = v.float(), v.t().float(), _two_to(k).float()
        qs.append(q)
        ts.append(t)
        ss.append(s)
    return qs + ts + ss
