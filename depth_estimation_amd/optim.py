"""The optimiser for weight matrices: momentum, then an update whose singular values are all near one.

A weight matrix (a linear layer; a convolution as (out, in*kh*kw)) is stepped along its momentum with the singular values
taken out by Newton-Schulz products (HIP kernels, ds_orthogonalize); biases and other vectors stay with torch.optim.Adam, as
the reference steps everything (train.py:140).  Not in the reference.
"""
from __future__ import annotations

import torch

from . import ops

COEFFICIENTS = (3.4445, -4.7750, 2.0315)   # steep at zero: five steps bring singular values from 0.01 up into 0.7 .. 1.2


def orthogonalize(update: torch.Tensor, steps: int = 5, coefficients=COEFFICIENTS, eps: float = 1e-7) -> torch.Tensor:
    """update (...,m,n) float32, float16 or bfloat16 on the GPU -> same shape and dtype: X = G / (|G|_F + eps), then `steps`
    (0..32) times X = (a I + b A + c A A) X with A = X X^T on the smaller side.  No gradient flows.  Products on 22-bit
    operands with float32 sums, one rounding at the end; up to six steps of bfloat16 matrices with sides of 512 and more take
    11-bit operands where that costs less than the rounding of the result does (1.2e-3 of its norm at most, against 1.7e-3;
    coefficients whose polynomial is steeper than the default's keep 22 bits).  Coefficients that would take singular values of
    [0,1] beyond 2^24 before the last step are refused (the default keeps them below 1.3).  Parts of X below 2^-38 are not
    kept: with a norm of G far below eps the result loses digits."""
    return ops.orthogonalize(update, steps, coefficients, eps)


class Muon(torch.optim.Optimizer):
    """Momentum with orthogonalised steps for parameters of two or more dimensions (flattened to (size(0), rest)):

        buf = momentum buf + grad;  u = grad + momentum buf (nesterov) or buf
        p = p (1 - lr weight_decay) - lr sqrt(max(1, m/n)) orthogonalize(u)

    Matrices of one shape and dtype are orthogonalised as one batch."""

    def __init__(self, params, lr: float = 0.02, momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0,
                 steps: int = 5, coefficients=COEFFICIENTS, eps: float = 1e-7):
        if lr < 0 or not 0 <= momentum < 1 or weight_decay < 0:
            raise ValueError(f"bad lr, momentum or weight_decay: {lr}, {momentum}, {weight_decay}")
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps,
                                      coefficients=tuple(coefficients), eps=eps))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        for p in self.param_groups[-1]["params"]:
            if p.dim() < 2:
                self.param_groups.pop()
                raise ValueError(f"Muon steps matrices; a parameter of shape {tuple(p.shape)} belongs to another optimiser")

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            same = {}
            for p in group["params"]:
                if p.grad is None or p.numel() == 0:
                    continue
                state = self.state[p]
                if "momentum_buffer" not in state:
                    state["momentum_buffer"] = torch.zeros_like(p.grad)
                buf = state["momentum_buffer"]
                buf.mul_(group["momentum"]).add_(p.grad)
                u = p.grad.add(buf, alpha=group["momentum"]) if group["nesterov"] else buf
                u = u.flatten(1)
                same.setdefault((tuple(u.shape), u.dtype, u.device), []).append((p, u))
            for ((m, n), _, _), members in same.items():
                us = torch.stack([u for _, u in members])
                scale = group["lr"] * max(1.0, m / n) ** 0.5
                for (p, _), o in zip(members, orthogonalize(us, group["steps"], group["coefficients"], group["eps"])):
                    if group["weight_decay"]:
                        p.mul_(1 - group["lr"] * group["weight_decay"])
                    p.add_(o.view(p.shape), alpha=-scale)
        return loss
