"""Newton-Schulz orthogonalization and the optimizer step built on it, from their definitions, on the CPU in any precision."""
from __future__ import annotations

import math

import torch

COEFFICIENTS = (3.4445, -4.775, 2.0315)


def orthogonalize(u: torch.Tensor, steps: int = 5, coefficients=COEFFICIENTS, eps: float = 1e-7) -> torch.Tensor:
    """u [.., r, c] in its own precision: X = u / max(|u|, eps); X <- a X + (b A + c A A) X, A = X X^T over the shorter side."""
    if u.shape[-2] > u.shape[-1]:
        return orthogonalize(u.transpose(-2, -1), steps, coefficients, eps).transpose(-2, -1)
    a, b, c = coefficients
    norm = u.double().square().sum((-2, -1), keepdim=True).sqrt()
    x = u / norm.clamp(min=eps).to(u.dtype)
    for _ in range(steps):
        g = torch.matmul(x, x.transpose(-2, -1))
        x = a * x + torch.matmul(b * g + c * torch.matmul(g, g), x)
    return x


def rate(rows: int, cols: int, adjust_lr: str) -> float:
    return 0.2 * math.sqrt(max(rows, cols)) if adjust_lr == "match_rms_adamw" else math.sqrt(max(1.0, rows / cols))


def muon_step(w, m, g, *, lr, momentum, weight_decay, nesterov=True, adjust_lr="original", steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    """(w, m) after a step, in the precision of w, m and g."""
    m = m + (1 - momentum) * (g - m)
    u = g + momentum * (m - g) if nesterov else m
    o = orthogonalize(u, steps, coefficients, eps)
    return w * (1 - lr * weight_decay) - lr * rate(*w.shape[-2:], adjust_lr) * o, m
