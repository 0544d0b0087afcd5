"""Fused AdamW over a flat bucket, satisfying the optimizer-factory contract of the reference's
actor: ``optim_class([shard_param])`` / ``optim_class(params, fused=True)`` returns an object whose
``.step()`` consumes ``p.grad`` (src/actor.py:573,600; src/runtime.py:470-473).

Every parameter handed in is treated as one flat buffer and updated by ONE kernel launch that
reads grad/master/exp_avg/exp_avg_sq and writes master/exp_avg/exp_avg_sq (28 B/element) plus,
for a bf16 parameter, the bf16 value the model reads (+2 B/element).  bf16 parameters get an fp32
master copy; fp32 parameters are their own master.

``state_bits=8``: both moments are held in 8-bit floating point with a power of two for each 64 elements, rounded up or down
at random so that their means are right (ops.adamw8_fused): 2 instead of 8 bytes of state an element, 18 instead of 30 B of traffic.
``seed`` chooses the random bits; runs with one seed repeat bit for bit.
"""
from __future__ import annotations

import torch

from . import ops


class FusedAdamW(torch.optim.Optimizer):
    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, fused: bool = True, zero_grad_in_step: bool = False, state_bits: int = 32,
                 seed: int = 0):
        if lr < 0 or eps < 0 or not (0 <= betas[0] < 1) or not (0 <= betas[1] < 1) or weight_decay < 0:
            raise ValueError("invalid AdamW hyper-parameters")
        if state_bits not in (8, 32):
            raise ValueError(f"FusedAdamW holds its moments in 32 or 8 bits, not {state_bits}")
        defaults = dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay)
        super().__init__(params, defaults)
        self.zero_grad_in_step = zero_grad_in_step
        self.state_bits, self.seed = state_bits, int(seed)

    def _init_state(self, p: torch.Tensor) -> dict:
        st = self.state[p]
        if not st:
            flat = p.detach().reshape(-1)
            st["step"] = 0
            st["master"] = flat if p.dtype == torch.float32 else flat.float()
            if self.state_bits == 8:
                for name, t in zip(_MOMENTS8, ops.adamw8_state(flat.numel(), flat.device)):
                    st[name] = t
                # elements of different buckets with the same index get other bits
                st["seed"] = self.seed + 0x632BE5AB * (len(self.state) - 1)
                return st
            st["exp_avg"] = torch.zeros_like(st["master"])
            st["exp_avg_sq"] = torch.zeros_like(st["master"])
        return st

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            b1, b2 = group["betas"]
            for p in group["params"]:
                if p.grad is None:
                    continue
                if not p.is_contiguous():
                    raise RuntimeError("FusedAdamW needs contiguous parameters (flatten them into a bucket)")
                st = self._init_state(p)
                st["step"] += 1
                grad = p.grad.detach().reshape(-1)
                owns_grad = grad.dtype == torch.float32 and grad.is_contiguous()
                if not owns_grad:
                    grad = grad.float().contiguous()
                shadow = None if p.dtype == torch.float32 else p.detach().reshape(-1)
                if self.state_bits == 8:
                    self._step8(st, grad, group, shadow, self.zero_grad_in_step and owns_grad)
                    continue
                ops.adamw_fused(st["master"], st["exp_avg"], st["exp_avg_sq"], grad, step=st["step"],
                                lr=group["lr"], beta1=b1, beta2=b2, eps=group["eps"],
                                weight_decay=group["weight_decay"], shadow=shadow,
                                zero_grad=self.zero_grad_in_step and owns_grad)
        return loss

    @torch.no_grad()
    def step_packed(self, p: torch.Tensor, grads, offsets, numels, flat_grad: torch.Tensor | None = None) -> None:
        """One step for the flat parameter `p` (a bucket) whose last gradients have not been packed:
        tensor i of the bucket (elements offsets[i] .. +numels[i]) has the gradient flat_grad[...] (what
        earlier microbatches packed, optional) + grads[i] (optional).  Same result as packing
        grads into flat_grad and calling step() with p.grad = flat_grad, in one launch that
        neither writes nor re-reads the fp32 gradient bucket."""
        group = next(g for g in self.param_groups if any(q is p for q in g["params"]))
        if not p.is_contiguous():
            raise RuntimeError("FusedAdamW needs contiguous parameters (flatten them into a bucket)")
        st = self._init_state(p)
        st["step"] += 1
        b1, b2 = group["betas"]
        shadow = None if p.dtype == torch.float32 else p.detach().reshape(-1)
        if self.state_bits == 8:
            clear = self.zero_grad_in_step and flat_grad is not None
            if all(o % ops.ADAMW8_BLOCK == 0 for o in offsets):
                ops.adamw8_fused_packed(st["master"], *(st[k] for k in _MOMENTS8), flat_grad, list(grads), list(offsets), list(numels),
                                        shadow=shadow, zero_grad=clear, **self._how8(st, group))
                return
            # a block of the moments may belong to two tensors (a bucket without aligned starts): packed first, into a copy
            flat = torch.zeros_like(st["master"]) if flat_grad is None else flat_grad.clone()
            ops.bucket_pack(list(grads), list(offsets), flat, accumulate=True, numels=list(numels))
            self._step8(st, flat, group, shadow, False)
            if clear:
                for o, n in zip(offsets, numels):
                    flat_grad[o:o + n].zero_()
            return
        ops.adamw_fused_packed(st["master"], st["exp_avg"], st["exp_avg_sq"], flat_grad, list(grads), list(offsets),
                               list(numels), step=st["step"], lr=group["lr"], beta1=b1, beta2=b2, eps=group["eps"],
                               weight_decay=group["weight_decay"], shadow=shadow,
                               zero_grad=self.zero_grad_in_step and flat_grad is not None)

    def _how8(self, st: dict, group: dict) -> dict:
        b1, b2 = group["betas"]
        return dict(step=st["step"], lr=group["lr"], beta1=b1, beta2=b2, eps=group["eps"], weight_decay=group["weight_decay"],
                    seed=st["seed"] + 0x9E3779B1 * st["step"])

    def _step8(self, st: dict, grad: torch.Tensor, group: dict, shadow, zero_grad: bool) -> None:
        ops.adamw8_fused(st["master"], *(st[k] for k in _MOMENTS8), grad, shadow=shadow, zero_grad=zero_grad, **self._how8(st, group))

    @torch.no_grad()
    def load_state_dict(self, state_dict) -> None:
        """torch's, which gives every floating-point state the parameter's type, a copy of its own: moments and master keep theirs here, and
        an fp32 parameter stays its own master.  A state of the other ``state_bits`` or of other sizes is a ValueError that leaves the
        optimizer as it was."""
        saved = []      # what the program's own pre-hooks make of state_dict: this one is the last to run
        hooks = (self.register_load_state_dict_pre_hook(lambda _, given: saved.extend(self._checked(given))),
                 self.register_load_state_dict_post_hook(lambda _: self._restore(saved), prepend=True))
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

    def _restore(self, saved) -> None:
        types = dict(zip(_MOMENTS8, _TYPES8)) if self.state_bits == 8 else dict(exp_avg=torch.float32, exp_avg_sq=torch.float32)
        for p, st in saved:
            own = self.state[p]
            for name, dtype in types.items():
                own[name] = st[name].to(device=p.device, dtype=dtype, copy=True)
            if p.dtype == torch.float32:
                own["master"] = p.detach().reshape(-1)
            else:
                own["master"] = st["master"].to(device=p.device, dtype=torch.float32, copy=True)

    def _checked(self, state_dict) -> list:
        """[(parameter, its saved state)] of a state dict that this optimizer can take."""
        params = [p for group in self.param_groups for p in group["params"]]
        ids = [i for group in state_dict["param_groups"] for i in group["params"]]
        found = [(p, state_dict["state"][i]) for p, i in zip(params, ids) if state_dict["state"].get(i)]
        for p, st in found:
            n, blocks = p.numel(), -(-p.numel() // ops.ADAMW8_BLOCK)
            if self.state_bits == 8:
                sizes = dict(zip(_MOMENTS8, (n, blocks, n, blocks)), master=n)
                if any(k not in st or st[k].dtype != dt for k, dt in zip(_MOMENTS8, _TYPES8)) or "seed" not in st:
                    raise ValueError("FusedAdamW(state_bits=8): the saved state has no 8-bit moments")
            else:
                sizes = dict(exp_avg=n, exp_avg_sq=n, master=n)
                if any(k in st for k in _MOMENTS8[1::2]) or any(st[k].dtype in _TYPES8 for k in _MOMENTS8[::2] if k in st):
                    raise ValueError("FusedAdamW(state_bits=32): the saved state has 8-bit moments, codes that are nothing without their scales")
            if "step" not in st or any(k not in st or st[k].numel() != size for k, size in sizes.items()):
                raise ValueError(f"FusedAdamW: the saved state is not one of a parameter of {n} elements")
        return found


_MOMENTS8 = ("exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_scale")
_TYPES8 = (torch.float8_e4m3fn, torch.float8_e8m0fnu, torch.float8_e5m2, torch.float8_e8m0fnu)
