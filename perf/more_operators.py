"""What the training of an expert layer takes beside its forward and backward, as cases that can be timed and compared.

Three operators, each through the entry points that a program calls:

* ``balance``: the router's balance loss over packed sequences, with the tokens that every expert gets in each of them, and
  the gradient of its logits;
* ``orthogonalize``: the Newton-Schulz products that bring a matrix, or a stack of them, near the closest semi-orthogonal one;
* ``muon``: an optimizer step over the matrices of a bucket: momentum, orthogonalization, decay and update of the fp32
  weights and of the copy that the model reads.

Where ``own`` is false they are computed from elementary torch operations in 32 bits (sums over tokens in 64).
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
STEPS, COEFFICIENTS, EPS = 5, (3.4445, -4.775, 2.0315), 1e-7
MUON = dict(lr=1e-3, momentum=0.95, weight_decay=0.1)

# what the largest listed cases cost; no drawn case costs more
_MAX_LOGITS = 131072 * 128
_MAX_VALUES = 128 * 768 * 2048
_MAX_FLOPS = 128 * STEPS * (3 * 768 * 768 * 2048 + 768 ** 3)


def listed() -> list[dict]:
    return [
        # one microbatch of the tiny fp32 region, two sequences: launches
        dict(name="balance_256", kind="balance", tokens=256, experts=8, top_k=2, sequences=2, padding=0, z=0.0, skew=0.0),
        # one microbatch of the benchmark's region as one sequence
        dict(name="balance_4096", kind="balance", tokens=4096, experts=128, top_k=8, sequences=1, padding=0, z=1e-3, skew=0.0),
        # packed sequences of different lengths (some empty) with padding behind the last one, popular experts
        dict(name="balance_packed", kind="balance", tokens=16411, experts=60, top_k=4, sequences=61, padding=203, z=1e-3, skew=0.45),
        # all microbatches of an iteration at once
        dict(name="balance_131072", kind="balance", tokens=131072, experts=128, top_k=8, sequences=512, padding=0, z=1e-3, skew=0.45),
        # the router's own matrix: one small one, which latency bounds
        dict(name="orthogonalize_gate", kind="orthogonalize", batch=1, rows=128, cols=2048, dtype="f32"),
        # experts of odd widths, taller than wide
        dict(name="orthogonalize_odd", kind="orthogonalize", batch=24, rows=1000, cols=363, dtype="bf16"),
        # one weight of all experts of the benchmark's layer
        dict(name="orthogonalize_experts", kind="orthogonalize", batch=128, rows=768, cols=2048, dtype="bf16"),
        # one dense matrix, in fp32: few tiles, long reductions
        dict(name="orthogonalize_dense", kind="orthogonalize", batch=1, rows=2048, cols=4096, dtype="f32"),
        # the tiny fp32 region's experts
        dict(name="muon_small", kind="muon", layers=1, hidden=256, q=0, kv=0, experts=8, inter=512, stacked=True, dtype="f32", packed=False),
        # the matrices of the benchmark's bucket: two layers, 92 of them, the last gradients as the backward left them (bf16) and those of
        # earlier microbatches in the bucket (fp32)
        dict(name="muon_bucket", kind="muon", layers=2, hidden=2048, q=4096, kv=512, experts=14, inter=768, stacked=False, dtype="bf16", packed=True),
        # a layer with its experts in three stacks
        dict(name="muon_layer", kind="muon", layers=1, hidden=2048, q=4096, kv=512, experts=32, inter=768, stacked=True, dtype="bf16", packed=False),
    ]


def _log(rng: random.Random, lo: float, hi: float) -> float:
    return math.exp(rng.uniform(math.log(lo), math.log(hi)))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(["balance", "orthogonalize", "muon"])
    if kind == "balance":
        experts = rng.choice([2, 8, 60, 64, 128, 256, rng.randint(3, 400)])
        tokens = max(1, int(_log(rng, 1, min(131072, _MAX_LOGITS / experts))))
        return dict(kind=kind, tokens=tokens, experts=experts, top_k=rng.randint(1, min(8, experts - 1)),
                    sequences=max(1, int(_log(rng, 1, max(2.0, min(512.0, tokens))))), padding=rng.choice([0, 0, rng.randint(0, min(300, tokens))]),
                    z=rng.choice([0.0, 1e-3]), skew=rng.choice([0.0, rng.uniform(0.1, 0.6)]))
    if kind == "orthogonalize":
        rows, cols = (rng.choice([8 * rng.randint(4, 300), 128 * rng.randint(1, 18), rng.randint(17, 2100)]) for _ in range(2))
        most = min(_MAX_VALUES / (rows * cols), _MAX_FLOPS / _flops(rows, cols), 128.0)
        return dict(kind=kind, batch=max(1, int(_log(rng, 1, max(2.0, most)))), rows=rows, cols=cols, dtype=rng.choice(["bf16", "bf16", "f32"]))
    hidden = rng.choice([8 * rng.randint(8, 256), 128 * rng.randint(1, 16), rng.randint(65, 2048)])
    inter = rng.choice([8 * rng.randint(8, 128), 128 * rng.randint(1, 8), rng.randint(65, 1024)])
    q = rng.choice([0, hidden, 2 * hidden])
    layers = rng.randint(1, 3)
    dense = layers * 2 * _flops(hidden, q) if q else 0
    experts = max(1, int(min((_MAX_FLOPS - dense) / (3 * _flops(hidden, inter) * layers), 64)))
    return dict(kind=kind, layers=layers, hidden=hidden, q=q, kv=hidden // 4 if q else 0, experts=rng.randint(1, experts), inter=inter,
                stacked=rng.random() < 0.5, dtype=rng.choice(["bf16", "bf16", "f32"]), packed=rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------ inputs
def _flops(rows: int, cols: int) -> int:
    """Products of one matrix's steps: two symmetric results, of which half is needed, and the update."""
    m, n = min(rows, cols), max(rows, cols)
    return STEPS * (m * m * n + m ** 3 + 2 * m * m * n)


def _shapes(case: dict) -> list[tuple[int, ...]]:
    H, I, E = case["hidden"], case["inter"], case["experts"]
    layer = [(case["q"], H), (case["kv"], H), (case["kv"], H), (H, case["q"])] if case["q"] else []
    if case["stacked"]:
        layer += [(E, I, H), (E, I, H), (E, H, I)]
    else:
        layer += [(I, H), (I, H), (H, I)] * E
    return layer * case["layers"]


def _gradients(shape, gen, dev) -> torch.Tensor:
    """Matrices with a few strong directions over noise, as gradients of a layer's weights are."""
    *batch, r, c = shape
    strong = torch.matmul(torch.randn((*batch, r, 8), generator=gen, device=dev), torch.randn((*batch, 8, c), generator=gen, device=dev))
    return (torch.randn(shape, generator=gen, device=dev) + 0.05 * strong) * 1e-3


def _offsets(case: dict, gen: torch.Generator, dev) -> torch.Tensor:
    """Where the sequences begin and end: cuts of the tokens in front of the padding, some of them at the same place."""
    owned = case["tokens"] - case["padding"]
    cuts = torch.randint(0, owned + 1, (case["sequences"] - 1,), generator=gen, device=dev).sort().values
    return torch.cat([cuts.new_zeros(1), cuts, cuts.new_full((1,), owned)]).to(torch.int32)


def prepare(case: dict, seed: int):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    if case["kind"] == "balance":
        T, E = case["tokens"], case["experts"]
        popular = -2.4 * case["skew"] * torch.log(torch.arange(1, E + 1, device=dev, dtype=torch.float32))
        logits = torch.randn((T, E), generator=gen, device=dev) + popular
        chosen = torch.topk(logits, case["top_k"], dim=1).indices.to(torch.int32)
        return dict(case=case, logits=logits.requires_grad_(True), chosen=chosen, sequences=_offsets(case, gen, dev),
                    d_loss=torch.rand((), generator=gen, device=dev) + 0.5)
    if case["kind"] == "orthogonalize":
        return dict(case=case, x=_gradients((case["batch"], case["rows"], case["cols"]), gen, dev).to(DTYPES[case["dtype"]]))
    shapes = _shapes(case)
    offsets, end = [], 0
    for s in shapes:
        offsets.append(end)
        end = -(-(end + math.prod(s)) // 128) * 128
    places = [(slice(o, o + math.prod(s)), s) for o, s in zip(offsets, shapes)]
    master, momentum = torch.zeros(end, device=dev), torch.zeros(end, device=dev)
    flat = torch.zeros(end, device=dev) if case["packed"] else None
    grads = []
    for at, s in places:
        master[at] = torch.randn(math.prod(s), generator=gen, device=dev) * 0.02
        momentum[at] = _gradients(s, gen, dev).reshape(-1)
        grads.append(_gradients(s, gen, dev).to(DTYPES[case["dtype"]]))
        if flat is not None:
            flat[at] = _gradients(s, gen, dev).reshape(-1)
    shadow = master.to(torch.bfloat16) if case["dtype"] == "bf16" else None
    return dict(case=case, places=places, master=master, momentum=momentum, flat=flat, grads=grads, shadow=shadow)


# ------------------------------------------------------------------------------------------------ balance
# For each sequence s of L tokens: f_e = (times that expert e was chosen) E / (K L), P_e = mean over its tokens of
# softmax(logits)_e.  loss = mean over the sequences with tokens of sum_e f_e P_e + z mean over the tokens of logsumexp(logits)^2.
def _plain_balance(state):
    case, logits, off = state["case"], state["logits"].detach(), state["sequences"].to(torch.int64)
    T, E, K, S = case["tokens"], case["experts"], case["top_k"], case["sequences"]
    owned = off[-1]
    t = torch.arange(T, device=logits.device)
    seq = torch.searchsorted(off, t, right=True) - 1                   # S: behind the last sequence
    live = (t < owned).float().unsqueeze(1)
    mx = logits.amax(1, keepdim=True)
    p = torch.exp(logits - mx)
    total = p.sum(1, keepdim=True)
    p, lse = p / total, mx + torch.log(total)
    chosen = (seq.unsqueeze(1) * E + state["chosen"].to(torch.int64)).reshape(-1)
    counts = torch.zeros((S + 1) * E, dtype=torch.int64, device=p.device).scatter_add_(0, chosen, torch.ones_like(chosen))[:S * E].view(S, E)
    length = (off[1:] - off[:-1]).double().unsqueeze(1)
    some = (length > 0).sum()
    sums = torch.nn.functional.pad(p.t().contiguous().double().cumsum(1), (1, 0))      # [E, T + 1]
    sums = (sums[:, off[1:]] - sums[:, off[:-1]]).t()
    slope = torch.where(length > 0, counts * (E / K) / length.clamp(min=1) ** 2 / some.clamp(min=1), 0.0)
    loss = (slope * sums).sum() + case["z"] * (lse * lse * live).double().sum() / owned.clamp(min=1)
    g = torch.nn.functional.pad(slope, (0, 0, 0, 1))[seq]              # close to its mean over p where the experts are balanced
    d = p * (g - (g * p).sum(1, keepdim=True) + 2 * case["z"] / owned.clamp(min=1) * lse * live)
    return loss.float(), counts.to(torch.int32), (d * state["d_loss"]).float()


def _own_balance(state):
    from piper_amd import functional

    loss, counts = functional.balance_loss(state["logits"], state["chosen"], balance_coeff=1.0, z_coeff=state["case"]["z"],
                                           sequences=state["sequences"])
    d, = torch.autograd.grad(loss, state["logits"], state["d_loss"])
    return loss, counts, d


# ------------------------------------------------------------------------------------------------ orthogonalization
def _orthogonal(u: torch.Tensor) -> torch.Tensor:
    """X = U / max(|U|, eps), STEPS times X <- a X + (b A + c A A) X with A = X X^T, over the shorter side; fp32 [.., r, c]."""
    tall = u.shape[-2] > u.shape[-1]
    x = u.transpose(-2, -1).contiguous() if tall else u
    x = x / x.square().sum((-2, -1), keepdim=True).sqrt().clamp(min=EPS)
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        g = torch.matmul(x, x.transpose(-2, -1).contiguous())
        x = a * x + torch.matmul(b * g + c * torch.matmul(g, g), x)
    return x.transpose(-2, -1) if tall else x


def _plain_orthogonalize(state):
    return _orthogonal(state["x"].float()).contiguous().to(state["x"].dtype)


def _own_orthogonalize(state):
    from piper_amd import ops

    return ops.orthogonalize(state["x"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)


# ------------------------------------------------------------------------------------------------ the optimizer step
# m <- m + (1 - mu) (g - m), u = g + mu (m - g), w <- w (1 - lr decay) - lr 0.2 sqrt(max(rows, cols)) orthogonal(u)
def _plain_muon(state):
    lr, mu, decay = MUON["lr"], MUON["momentum"], MUON["weight_decay"]
    for (at, s), grad in zip(state["places"], state["grads"]):
        g = grad.float()
        if state["flat"] is not None:
            g = state["flat"][at].view(s) + g
        m = state["momentum"][at].view(s)
        m += (1 - mu) * (g - m)
        o = _orthogonal(g + mu * (m - g))
        w = state["master"][at].view(s)
        w.copy_(w * (1 - lr * decay) - lr * 0.2 * math.sqrt(max(s[-2:])) * o)
    if state["shadow"] is not None:
        state["shadow"].copy_(state["master"])
    return state["master"], state["momentum"], state["shadow"]


def _own_muon(state):
    from piper_amd import ops

    def views(flat):
        return None if flat is None else [flat[at].view(s) for at, s in state["places"]]

    ops.muon_fused(views(state["master"]), views(state["momentum"]), state["grads"], flat_grads=views(state["flat"]),
                   shadows=views(state["shadow"]), lr=MUON["lr"], momentum=MUON["momentum"], weight_decay=MUON["weight_decay"], steps=STEPS,
                   coefficients=COEFFICIENTS, eps=EPS, adjust_lr="match_rms_adamw")
    return state["master"], state["momentum"], state["shadow"]


def run(state):
    kind = state["case"]["kind"]
    if own:
        return (_own_balance if kind == "balance" else _own_orthogonalize if kind == "orthogonalize" else _own_muon)(state)
    return (_plain_balance if kind == "balance" else _plain_orthogonalize if kind == "orthogonalize" else _plain_muon)(state)


def work(case: dict) -> dict:
    if case["kind"] == "balance":
        T, E = case["tokens"], case["experts"]
        # the logits read and their gradient written, the choices read; exp, sums, products
        return dict(bytes=8 * T * E + 4 * T * case["top_k"] + 8 * case["sequences"] * E, flops=20 * T * E)
    if case["kind"] == "orthogonalize":
        n = case["batch"] * case["rows"] * case["cols"]
        return dict(bytes=2 * n * (2 if case["dtype"] == "bf16" else 4), flops=case["batch"] * _flops(case["rows"], case["cols"]))
    shapes = _shapes(case)
    n = sum(math.prod(s) for s in shapes)
    # weights and momentum read and written, gradients read (and in bf16 the model's copy written), those of the bucket read
    return dict(bytes=n * (20 + (4 if case["packed"] else 0)), flops=sum(math.prod(s[:-2]) * _flops(*s[-2:]) for s in shapes))


# ------------------------------------------------------------------------------------------------ in 64 bits
def _exact_balance(case, state):
    logits = state["logits"].detach().double().requires_grad_(True)
    off = state["sequences"].tolist()
    E, K = case["experts"], case["top_k"]
    with torch.enable_grad():
        p, lse = torch.softmax(logits, 1), torch.logsumexp(logits, 1)
        terms = [p.sum() * 0]
        for b, e in zip(off[:-1], off[1:]):
            if e > b:
                f = torch.nn.functional.one_hot(state["chosen"][b:e].long(), E).sum((0, 1)).double() * E / (K * (e - b))
                terms.append((f * p[b:e].mean(0)).sum())
        loss = sum(terms) / max(1, len(terms) - 1) + case["z"] * lse[:off[-1]].square().sum() / max(1, off[-1])
        d, = torch.autograd.grad(loss, logits, state["d_loss"].double())
    return loss.detach(), None, d


def _exact_orthogonal(u):
    if u.shape[-2] > u.shape[-1]:
        return _exact_orthogonal(u.mT.contiguous()).mT
    x = u / torch.linalg.matrix_norm(u).clamp(min=EPS)[..., None, None]
    one = torch.eye(x.shape[-2], dtype=x.dtype, device=x.device)
    for _ in range(STEPS):
        g = x @ x.mT.contiguous()
        x = (COEFFICIENTS[0] * one + g @ (COEFFICIENTS[1] * one + COEFFICIENTS[2] * g)) @ x
    return x


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    if case["kind"] == "balance":
        return _exact_balance(case, state)
    if case["kind"] == "orthogonalize":
        return torch.cat([_exact_orthogonal(x.double()) for x in state["x"].split(16)])
    master, momentum = state["master"].double(), state["momentum"].double()
    for i, (at, s) in enumerate(state["places"]):
        g = state["grads"][i].double() + (0 if state["flat"] is None else state["flat"][at].double().view(s))
        momentum[at] = MUON["momentum"] * momentum[at] + (1 - MUON["momentum"]) * g.reshape(-1)
        u = (1 - MUON["momentum"]) * g + MUON["momentum"] * momentum[at].view(s)
        rate = MUON["lr"] * 0.2 * max(s[-2:]) ** 0.5
        master[at] -= MUON["lr"] * MUON["weight_decay"] * master[at] + rate * _exact_orthogonal(u).reshape(-1)
    return master, momentum, None if state["shadow"] is None else master
