"""The router's balance loss from its definition, on the CPU in the precision of the logits."""
from __future__ import annotations

import torch


def balance_loss(logits: torch.Tensor, top_idx: torch.Tensor, balance_coeff: float = 1.0, z_coeff: float = 0.0, sequences=None):
    """(loss, counts [S,E]): sequences is a list of offsets (None: one sequence).  Differentiable in the logits."""
    T, E = logits.shape
    K = top_idx.shape[1]
    offsets = [0, T] if sequences is None else [int(o) for o in sequences]
    p, lse = torch.softmax(logits, 1), torch.logsumexp(logits, 1)
    counts = torch.zeros(len(offsets) - 1, E, dtype=torch.int64)
    terms, squares, tokens = logits[:0].sum(), logits[:0].sum(), 0
    some = 0
    for s, (b, e) in enumerate(zip(offsets[:-1], offsets[1:])):
        counts[s] = torch.bincount(top_idx[b:e].reshape(-1).long(), minlength=E)
        if e > b:
            some += 1
            tokens += e - b
            terms = terms + (counts[s].to(logits.dtype) * E / (K * (e - b)) * p[b:e].mean(0)).sum()
            squares = squares + lse[b:e].square().sum()
    return balance_coeff * terms / max(some, 1) + z_coeff * squares / max(tokens, 1), counts


def gradient_scale(logits: torch.Tensor, counts: torch.Tensor, K: int, balance_coeff: float, z_coeff: float, sequences=None) -> torch.Tensor:
    """What the summands of every element of the logits' gradient add up to by magnitude, [T,E] in 64 bits: a rounding of one of them is off
    by that, times half a step."""
    x = logits.double()
    T, E = x.shape
    offsets = [0, T] if sequences is None else [int(o) for o in sequences]
    p, lse = torch.softmax(x, 1), torch.logsumexp(x, 1)
    out = torch.zeros_like(x)
    some, tokens = sum(e > b for b, e in zip(offsets[:-1], offsets[1:])), max(1, offsets[-1] - offsets[0])
    for s, (b, e) in enumerate(zip(offsets[:-1], offsets[1:])):
        if e > b:
            L = e - b
            h = abs(balance_coeff) * E / (K * L * L * some) * (counts[s].double() - K * L / E).abs()
            out[b:e] = p[b:e] * (h + (p[b:e] * h).sum(1, keepdim=True) + 2 * abs(z_coeff) / tokens * lse[b:e].abs().unsqueeze(1))
    return out
