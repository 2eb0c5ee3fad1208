"""AdamW over many tensors in one launch, with float32 or 8-bit states.

``adamw_step`` is the step on lists of tensors; ``AdamW`` keeps the states, as the
reference's ``FlatAdamW`` does for its flat buffers (``ravel_lm/runtime.py:44``), with its
clipping by the global norm (``runtime.py:9``).  Per element, in float32:

    g' = g min(1, max_norm / (|g| + 1e-6))            (|g| over every tensor)
    m = b1 m + (1 - b1) g',  v = b2 v + (1 - b2) g'^2
    p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)

(a positive eps below 2^-126 counts as 2^-126).  A 16-bit parameter is the rounding of a
float32 master that takes the steps.  8-bit states share a power of two per block of 256
elements, sign + 4 + 3 bits for m and 5 + 3 for v, and are rounded stochastically (the
random bits are a hash of step, tensor and element: a run repeats bit for bit).  ``AdamW``
keeps every positive v positive, so that a block may hold elements of very different
gradients.  A block that meets a NaN or an infinity stands for NaN as a whole from then on.

The step count lives on the device and the learning rate may too, so that a step
captured in a CUDA graph counts on in every replay.
"""
from __future__ import annotations

from typing import Optional, Sequence, Union

import torch

from . import _lib

Tensor = torch.Tensor
_BLOCK = 256   # elements that share an exponent
_EMPTY = -126  # the exponent of a block of zeros


def global_norm(tensors: Sequence[Tensor]) -> Tensor:
    """The 2-norm over every element of ``tensors`` (float32, bfloat16 or float16): float64, 0-dim, on their device."""
    return _lib.host().global_norm(list(tensors))


def adamw_step(params: Sequence[Tensor], grads: Sequence[Tensor], exp_avgs: Sequence[Tensor],
               exp_avg_sqs: Sequence[Tensor], step: Tensor, *, lr: Union[float, Tensor],
               betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 0.01,
               masters: Optional[Sequence[Tensor]] = None, exp_avg_exponents: Optional[Sequence[Tensor]] = None,
               exp_avg_sq_exponents: Optional[Sequence[Tensor]] = None, max_norm: Optional[float] = None,
               norm: Optional[Tensor] = None, positive_exp_avg_sq: bool = False) -> Optional[Tensor]:
    """One AdamW step in place on every tensor of the lists; all of one dtype, contiguous, on one device, none twice.

    Args:
        params:      float32, bfloat16 or float16; 16-bit ones need ``masters``, float32 of the same sizes.
        grads:       of the parameters' shapes and dtype.
        exp_avgs, exp_avg_sqs: float32, or uint8 codes with ``exp_avg_exponents`` and
                     ``exp_avg_sq_exponents`` (int8, one per block of 256 elements of a tensor).
        step:        one int64 on the device, the steps taken so far; counts up by one.
        lr:          a number, or one float32 on the device.
        max_norm:    gradients are scaled down to this norm over all of them, or by ``norm``
                     (``global_norm``'s) where other tensors share in it.
        positive_exp_avg_sq: 8-bit states: a positive second moment has code 1 at least (``AdamW``'s way).  Without it
                     one below 2^-33 of its block's largest may be rounded to 0 while the first
                     moment is not: in blocks whose gradients differ by factors past 1e4 steps of hundreds of lr.
    Returns:
        the norm (float32, 0-dim) with ``max_norm``, else None.
    """
    b1, b2 = betas
    on_device = isinstance(lr, Tensor)
    lists = [None if v is None else list(v) for v in (masters, exp_avg_exponents, exp_avg_sq_exponents)]
    return _lib.host().adamw_step(list(params), list(grads), list(exp_avgs), list(exp_avg_sqs), step, *lists,
                                  0.0 if on_device else float(lr), lr if on_device else None, float(b1), float(b2),
                                  float(eps), float(weight_decay), max_norm, norm, bool(positive_exp_avg_sq))


def state_values(codes: Tensor, exponents: Tensor, *, signed: bool, dtype: torch.dtype = torch.float32) -> Tensor:
    """What 8-bit state codes stand for: ``signed`` for exp_avg, not for exp_avg_sq; float32 or bfloat16 (the codes
    have 4 significant bits, so that bfloat16 holds them exactly, except below its normal range)."""
    if dtype not in (torch.float32, torch.bfloat16):
        raise TypeError(f"state_values gives float32 or bfloat16, not {dtype}")
    return _lib.host().state_values(codes, exponents, bool(signed), dtype == torch.bfloat16)


class AdamW(torch.optim.Optimizer):
    """AdamW with the states above, for CUDA parameters of float32, bfloat16 or float16.

    Args:
        state_bits: 32 or 8.
        max_norm:   clip gradients by their norm over every group; the last norm is ``grad_norm``.

    A parameter counts the steps in which it had a gradient.  Masters are made from 16-bit parameters at their
    first step: parameters overwritten later need ``reset_masters()``.  ``lr`` may be a float32 CUDA tensor.
    A step may be captured in a CUDA graph after an eager one with gradients for the same parameters.
    """

    def __init__(self, params, lr: Union[float, Tensor] = 1e-3, betas: tuple[float, float] = (0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 0.01, *, state_bits: int = 32,
                 max_norm: Optional[float] = None):
        if not isinstance(lr, Tensor) and not lr >= 0.0:
            raise ValueError(f"lr must not be negative, got {lr}")
        if not eps >= 0.0 or not weight_decay >= 0.0:
            raise ValueError("eps and weight_decay must not be negative")
        if not all(0.0 <= b < 1.0 for b in betas):
            raise ValueError(f"betas must lie in [0, 1), got {betas}")
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits}")
        if max_norm is not None and not max_norm > 0.0:
            raise ValueError(f"max_norm must be positive, got {max_norm}")
        self.state_bits, self.max_norm, self.grad_norm = state_bits, max_norm, None
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))

    def _new_state(self, p: Tensor, step: Tensor) -> dict:
        st = {"step": step}
        if self.state_bits == 32:
            st["exp_avg"] = torch.zeros_like(p, dtype=torch.float32)
            st["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.float32)
        else:
            blocks = (p.numel() + _BLOCK - 1) // _BLOCK
            for name in ("exp_avg", "exp_avg_sq"):
                st[name] = torch.zeros_like(p, dtype=torch.uint8)
                st[name + "_exponents"] = torch.full((blocks,), _EMPTY, dtype=torch.int8, device=p.device)
        if p.dtype != torch.float32:
            st["master"] = p.detach().float()
        return st

    def _state_names(self, p: Tensor) -> set[str]:
        """The names of ``_new_state(p, step)``."""
        names = {"step", "exp_avg", "exp_avg_sq"}
        if self.state_bits == 8:
            names |= {"exp_avg_exponents", "exp_avg_sq_exponents"}
        return names if p.dtype == torch.float32 else names | {"master"}

    @torch.no_grad()
    def reset_masters(self) -> None:
        """Take the float32 masters from the parameters as they are now."""
        for p, st in self.state.items():
            if "master" in st:
                st["master"].copy_(p)

    def _buckets(self, group: dict) -> list[list[Tensor]]:
        """The group's parameters with gradients, by the step tensor they share: those of one dtype and device that have
        counted the same steps.  Where one of them has no gradient now, the others go on with a copy.  Neither new
        states nor copies are made inside a capture: every replay would make them again."""
        idle = {id(self.state[p]["step"]) for p in group["params"] if p.grad is None and self.state.get(p)}
        fresh: dict = {}
        moved: dict = {}
        buckets: dict = {}
        for p in group["params"]:
            if p.grad is None:
                continue
            st = self.state.get(p)
            if (not st or id(st["step"]) in idle) and torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("AdamW: take a step with gradients for the same parameters before a capture; a "
                                   + ("new state" if not st else "step count copied for some of them")
                                   + " would start again in every replay")
            if not st:
                kind = (p.dtype, p.device)
                if kind not in fresh:
                    fresh[kind] = torch.zeros(1, dtype=torch.int64, device=p.device)
                st = self.state[p] = self._new_state(p, fresh[kind])
            elif id(st["step"]) in idle:
                old = st["step"]
                if id(old) not in moved:
                    moved[id(old)] = old.clone()
                st["step"] = moved[id(old)]
            buckets.setdefault(id(st["step"]), []).append(p)
        return list(buckets.values())

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        buckets = [(group, ps) for group in self.param_groups for ps in self._buckets(group)]
        norm = None
        if self.max_norm is not None:
            grads = [p.grad for g in self.param_groups for p in g["params"] if p.grad is not None]
            norm = global_norm(grads) if grads else None
            self.grad_norm = norm
        for group, ps in buckets:
            sts = [self.state[p] for p in ps]

            def each(name):
                return [st[name] for st in sts] if name in sts[0] else None
            adamw_step(ps, [p.grad for p in ps], each("exp_avg"), each("exp_avg_sq"), sts[0]["step"],
                       lr=group["lr"], betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"],
                       masters=each("master"), exp_avg_exponents=each("exp_avg_exponents"),
                       exp_avg_sq_exponents=each("exp_avg_sq_exponents"), max_norm=self.max_norm, norm=norm,
                       positive_exp_avg_sq=self.state_bits == 8)
        return loss

    def load_state_dict(self, state_dict: dict) -> None:
        """As ``torch.optim.Optimizer``'s, with the states in their own types (not cast to their parameters').  States of
        another ``state_bits`` or another optimizer are refused before anything is loaded."""
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        owned = [(p, k) for k, g in enumerate(self.param_groups) for p in g["params"]]
        for i, (p, _) in zip(ids, owned):
            src = state_dict["state"].get(i)
            if not src:
                continue
            if "exp_avg" in src and (src["exp_avg"].dtype == torch.uint8) != (self.state_bits == 8):
                raise ValueError(f"the loaded states do not have state_bits={self.state_bits}")
            if (not self._state_names(p) <= set(src) or ("master" in src) != (p.dtype != torch.float32)
                    or getattr(src["step"], "dtype", None) != torch.int64):
                raise ValueError(f"the loaded states are not this optimizer's for a parameter of {p.dtype}")
        super().load_state_dict(state_dict)
        shared: dict = {}
        for i, (p, g) in zip(ids, owned):
            src = state_dict["state"].get(i)
            if not src:
                continue
            st = {k: v.detach().to(p.device, copy=True) for k, v in src.items()}
            st["step"] = shared.setdefault((g, p.dtype, p.device, int(st["step"])), st["step"])
            self.state[p] = st

    def __getstate__(self) -> dict:
        return {**super().__getstate__(), "state_bits": self.state_bits, "max_norm": self.max_norm,
                "grad_norm": self.grad_norm}


__all__ = ["AdamW", "adamw_step", "global_norm", "state_values"]
