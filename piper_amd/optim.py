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


class _FlatStateOptimizer(torch.optim.Optimizer):
    """An optimizer whose states hold flat fp32 (or narrower) buffers and a master of their parameter's weights.  Subclasses say which saved
    states they take (_checked) and how they become theirs (_restore)."""

    @torch.no_grad()
    def load_state_dict(self, state_dict) -> None:
        """torch's, which gives every floating-point state the parameter's type, a copy of its own: moments and master keep theirs here, and
        an fp32 parameter stays its own master.  A state of another kind (``state_bits``) or of other sizes is a ValueError that leaves the
        optimizer as it was."""
        saved = []      # what the program's own pre-hooks make of state_dict: this one is the last to run
        hooks = (self.register_load_state_dict_pre_hook(lambda _, given: saved.extend(self._checked(given))),
                 self.register_load_state_dict_post_hook(lambda _: self._restore(saved), prepend=True))
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

    def _restore_tensors(self, saved, types: dict) -> None:
        """The tensors `types` names in those types, copies of their own; the master of an fp32 parameter is the parameter."""
        for p, st in saved:
            own = self.state[p]
            for name, dtype in types.items():
                own[name] = st[name].to(device=p.device, dtype=dtype, copy=True)
            if p.dtype == torch.float32:
                own["master"] = p.detach().reshape(-1)
            else:
                own["master"] = st["master"].to(device=p.device, dtype=torch.float32, copy=True)

    def _found(self, state_dict) -> list:
        """[(parameter, its saved state)]"""
        params = [p for group in self.param_groups for p in group["params"]]
        ids = [i for group in state_dict["param_groups"] for i in group["params"]]
        return [(p, state_dict["state"][i]) for p, i in zip(params, ids) if state_dict["state"].get(i)]


class FusedAdamW(_FlatStateOptimizer):
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

    def _restore(self, saved) -> None:
        self._restore_tensors(saved, dict(zip(_MOMENTS8, _TYPES8)) if self.state_bits == 8 else dict(exp_avg=torch.float32, exp_avg_sq=torch.float32))

    def _checked(self, state_dict) -> list:
        """[(parameter, its saved state)] of a state dict that this optimizer can take."""
        found = self._found(state_dict)
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


class FusedMuon(_FlatStateOptimizer):
    """Every matrix by its orthogonalized momentum (ops.muon_fused), what is no matrix by AdamW, in fp32 masters, with the
    bf16 value the model reads written in the same pass.

    A parameter of two dimensions or more is a matrix, or a stack of them [.., rows, cols].  In a flat bucket the parameters are views:
    ``bucket.flatten_params(..., optim_class=FusedMuon)`` tells the optimizer where they are (``bind_views``), and one call of
    ops.muon_fused takes all of them.  Parameters outside of a bucket take a call each (92 matrices of two layers: 34.7 ms a step, in a
    bucket 11.5).  ``matrices(param)`` says which parameters are updated as matrices (a router's gate or an embedding is often left to
    AdamW); default: those of two dimensions or more.  ``adamw``: lr (a schedule of this optimizer's lr moves it in proportion), betas, eps
    and weight_decay of the others where they differ from this optimizer's lr and weight decay and AdamW's defaults.
    ``half_products``: see ops.orthogonalize.  4 bytes of state an element (4 more for AdamW's) beside the master; up to 2.5 GiB of
    workspace in a step."""

    def __init__(self, params, lr: float = 1e-3, momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.1, ns_steps: int = 5,
                 ns_coefficients=ops.NEWTON_SCHULZ, eps: float = 1e-7, adjust_lr: str = "original", half_products: bool = False,
                 adamw: dict | None = None, matrices=None, fused: bool = True, zero_grad_in_step: bool = False):
        other = dict(lr=lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=weight_decay)
        if adamw:
            unknown = set(adamw) - set(other)
            if unknown:
                raise ValueError(f"FusedMuon: adamw takes lr, betas, eps and weight_decay, not {sorted(unknown)}")
            other.update(adamw)
        b1, b2 = other["betas"]
        if lr < 0 or not 0 <= momentum < 1 or weight_decay < 0 or eps <= 0 or not 0 <= ns_steps <= 100 or len(tuple(ns_coefficients)) != 3 or \
                adjust_lr not in ("original", "match_rms_adamw"):
            raise ValueError("invalid Muon hyper-parameters")
        if not ops.newton_schulz_in_range(ns_steps, ns_coefficients):
            raise ValueError("FusedMuon: coefficients that may take singular values past 15 (ops.orthogonalize)")
        if adamw and adamw.get("lr", lr) != lr and lr == 0:
            raise ValueError("FusedMuon: adamw's lr follows lr in proportion, which has to be positive for that")
        if other["lr"] < 0 or other["eps"] < 0 or not 0 <= b1 < 1 or not 0 <= b2 < 1 or other["weight_decay"] < 0:
            raise ValueError("invalid AdamW hyper-parameters")
        defaults = dict(lr=lr, momentum=momentum, nesterov=bool(nesterov), weight_decay=weight_decay, ns_steps=int(ns_steps),
                        ns_coefficients=tuple(float(c) for c in ns_coefficients), eps=eps, adjust_lr=adjust_lr, adamw_lr_ratio=other["lr"] / lr if lr else 1.0,
                        adamw_betas=(b1, b2), adamw_eps=other["eps"], adamw_weight_decay=other["weight_decay"])
        super().__init__(params, defaults)
        self.half_products, self.zero_grad_in_step = bool(half_products), zero_grad_in_step
        self._is_matrix = matrices or (lambda p: p.dim() >= 2)
        self._views: dict = {}

    def bind_views(self, p: torch.Tensor, specs) -> None:
        """`p` is a flat buffer of the parameters ``specs``: (parameter, offset, number of elements, shape) each."""
        if self.state.get(p):
            raise RuntimeError("FusedMuon.bind_views: the parameter has been stepped already")
        if p.dim() != 1:
            raise ValueError("FusedMuon.bind_views: views of a flat parameter")
        places = []
        for param, offset, numel, shape in specs:
            if offset < 0 or offset + numel > p.numel() or torch.Size(shape).numel() != numel:
                raise ValueError(f"FusedMuon.bind_views: {numel} elements at {offset} as {tuple(shape)} are no view of {p.numel()} elements")
            places.append((offset, numel, tuple(shape), len(shape) >= 2 and bool(self._is_matrix(param))))
        self._views[p] = places

    def _places(self, p: torch.Tensor) -> list:
        """(offset, number of elements, shape, whether it is a matrix) of the parameters in p."""
        if p in self._views:
            return self._views[p]
        return [(0, p.numel(), tuple(p.shape), p.dim() >= 2 and bool(self._is_matrix(p)))]

    def _adamw_elements(self, p: torch.Tensor) -> int:
        return sum(-(-n // 4) * 4 for _, n, _, matrix in self._places(p) if not matrix)

    def _init_state(self, p: torch.Tensor) -> dict:
        st = self.state[p]
        if not st:
            flat = p.detach().reshape(-1)
            st["step"] = 0
            st["master"] = flat if p.dtype == torch.float32 else flat.float()
            st["momentum"] = torch.zeros_like(st["master"])              # of what is no matrix: AdamW's first moment
            st["exp_avg_sq"] = torch.zeros(self._adamw_elements(p), dtype=torch.float32, device=p.device)
        return st

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            for p in group["params"]:
                if p.grad is None:
                    continue
                grad = p.grad.detach()
                if p in self._views:
                    flat = grad.reshape(-1)
                    owned = flat.dtype == torch.float32 and flat.is_contiguous()
                    self._update(p, group, flat if owned else flat.float().contiguous(), [None] * len(self._views[p]), self.zero_grad_in_step and owned)
                else:
                    self._update(p, group, None, [grad], False)
                    if self.zero_grad_in_step:
                        grad.zero_()
        return loss

    @torch.no_grad()
    def step_packed(self, p: torch.Tensor, grads, offsets, numels, flat_grad: torch.Tensor | None = None) -> None:
        """One step of the bucket `p` whose last gradients have not been packed: see FusedAdamW.step_packed."""
        group = next(g for g in self.param_groups if any(q is p for q in g["params"]))
        places = [(o, n) for o, n, *_ in self._places(p)]
        if p not in self._views or [tuple(x) for x in zip(offsets, numels)] != places:
            raise RuntimeError("FusedMuon.step_packed: gradients of the views that bind_views has been told of, in their order")
        self._update(p, group, flat_grad, list(grads), self.zero_grad_in_step and flat_grad is not None)

    def _update(self, p: torch.Tensor, group: dict, flat, grads, clear: bool) -> None:
        """grads: of each of _places, None: nothing beside `flat`"""
        if not p.is_contiguous():
            raise RuntimeError("FusedMuon needs contiguous parameters (flatten them into a bucket)")
        self._check_grads(p, flat, grads)
        st = self._init_state(p)
        st["step"] += 1
        shadow = None if p.dtype == torch.float32 else p.detach().reshape(-1)
        cut = lambda t, o, n: None if t is None else t[o:o + n]  # noqa: E731
        todo, second = [], 0
        for (o, n, shape, matrix), grad in zip(self._places(p), grads):
            if n == 0:
                continue
            buffers = [cut(t, o, n) for t in (st["master"], st["momentum"], flat, shadow)]
            if matrix:
                todo.append([None if t is None else t.view(shape) for t in buffers] + [grad])
            else:
                self._adamw(*buffers, grad, st["exp_avg_sq"][second:second + n], st["step"], group, clear)
                second += -(-n // 4) * 4
        if todo:
            masters, momenta, flats, shadows, grads = (list(t) for t in zip(*todo))
            ops.muon_fused(masters, momenta, grads, flat_grads=flats, shadows=shadows, lr=group["lr"], momentum=group["momentum"],
                           weight_decay=group["weight_decay"], nesterov=group["nesterov"], steps=group["ns_steps"],
                           coefficients=group["ns_coefficients"], eps=group["eps"], adjust_lr=group["adjust_lr"], zero_grad=clear,
                           half_products=self.half_products)

    def _check_grads(self, p: torch.Tensor, flat, grads) -> None:
        """Before anything is changed: a step refused for its tensors leaves weights and state as they were."""
        places = self._places(p)
        if p.dtype not in (torch.float32, torch.bfloat16):
            raise ValueError(f"FusedMuon: parameters are float32 or bfloat16, not {p.dtype}")
        if len(grads) != len(places):
            raise ValueError(f"FusedMuon: {len(grads)} gradients of {len(places)} parameters")
        types = set()
        for (_, n, _, matrix), grad in zip(places, grads):
            if grad is None:
                continue
            if grad.numel() != n or grad.device != p.device or grad.dtype not in (torch.float32, torch.bfloat16):
                raise ValueError(f"FusedMuon: a gradient of {grad.numel()} {grad.dtype} elements on {grad.device} for a parameter of {n} on {p.device}")
            if matrix and n:
                types.add(grad.dtype)
        if len(types) > 1:
            raise ValueError("FusedMuon: the matrices' gradients of one step share a dtype")
        if flat is not None and (flat.dtype != torch.float32 or flat.numel() != p.numel() or flat.device != p.device or not flat.is_contiguous()):
            raise ValueError(f"FusedMuon: the flat gradient is a contiguous float32 tensor of {p.numel()} elements on {p.device}")

    def _adamw(self, master, exp_avg, flat, shadow, grad, exp_avg_sq, step: int, group: dict, clear: bool) -> None:
        b1, b2 = group["adamw_betas"]
        given = (master, exp_avg, flat, shadow)
        # (16-byte boundaries: a bucket that was flattened without alignment goes through copies)
        used = [t if t is None or t.data_ptr() % 16 == 0 else t.clone() for t in given]
        ops.adamw_fused_packed(used[0], used[1], exp_avg_sq, used[2], [None if grad is None else grad.reshape(-1)], [0], [master.numel()], step=step,
                               lr=group["lr"] * group["adamw_lr_ratio"], beta1=b1, beta2=b2, eps=group["adamw_eps"], weight_decay=group["adamw_weight_decay"],
                               shadow=used[3], zero_grad=clear and flat is not None)
        for to, t in zip(given, used):
            if to is not t:
                to.copy_(t)

    def _restore(self, saved) -> None:
        self._restore_tensors(saved, dict(momentum=torch.float32, exp_avg_sq=torch.float32))

    def _checked(self, state_dict) -> list:
        found = self._found(state_dict)
        for p, st in found:
            n = p.numel()
            sizes = dict(master=n, momentum=n, exp_avg_sq=self._adamw_elements(p))
            if "step" not in st or any(k not in st or st[k].numel() != size for k, size in sizes.items()):
                raise ValueError(f"FusedMuon: the saved state is not one of a parameter of {n} elements with {sizes['exp_avg_sq']} in no matrix")
        return found
