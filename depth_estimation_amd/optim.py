"""The optimiser for weight matrices: momentum, then an update whose singular values are all near one.

A weight matrix (a linear layer; a convolution as (out, in*kh*kw)) is stepped along its momentum with the singular values
taken out by Newton-Schulz products (HIP kernels, ds_orthogonalize); biases and other vectors stay with torch.optim.Adam, as
the reference steps everything (train.py:140).  Not in the reference.  The method and the coefficients are published: Muon, K.
Jordan and others, 2024.
"""
from __future__ import annotations

import torch

from . import _lib as L
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

    Matrices of one shape and dtype are orthogonalised as one batch.  Parameters that no call would take (fewer than two
    dimensions, other types, a flattened side beyond 65536 or a smaller one beyond 32768: a head of 100000 classes) are refused
    when they are added; a step that cannot be made raises before it has changed anything."""

    def __init__(self, params, lr: float = 0.02, momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0,
                 steps: int = 5, coefficients=COEFFICIENTS, eps: float = 1e-7):
        if lr < 0 or not 0 <= momentum < 1 or weight_decay < 0:
            raise ValueError(f"bad lr, momentum or weight_decay: {lr}, {momentum}, {weight_decay}")
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps,
                                      coefficients=tuple(coefficients), eps=eps))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            try:
                ops.orthogonalize_options(group["steps"], group["coefficients"], group["eps"])
            except RuntimeError as e:
                raise ValueError(str(e)) from None
            for p in group["params"]:
                self._fits(p)
        except ValueError:
            self.param_groups.pop()
            raise

    @staticmethod
    def _fits(p):
        if p.dim() < 2:
            raise ValueError(f"Muon steps matrices; a parameter of shape {tuple(p.shape)} belongs to another optimiser")
        if p.dtype not in L.DTYPES:
            raise ValueError(f"Muon steps float32, float16 and bfloat16; got {p.dtype}")
        m, n = p.size(0), p.numel() // max(p.size(0), 1)
        if max(m, n) > 1 << 16 or min(m, n) > 1 << 15:
            raise ValueError(f"Muon steps matrices up to 65536 x 32768; a parameter of shape {tuple(p.shape)} ({m} x {n}) belongs "
                             "to another optimiser")

    def _check(self):
        """Whatever would make a call of orthogonalize fail, before a buffer or a parameter has changed."""
        for group in self.param_groups:
            steps, co, eps = ops.orthogonalize_options(group["steps"], group["coefficients"], group["eps"])
            shapes = {}
            for p in group["params"]:
                if p.grad is None or p.numel() == 0:
                    continue
                if p.grad.layout != torch.strided:
                    raise RuntimeError(f"Muon: dense gradients only, got {p.grad.layout}")
                L.dev_float(p.grad, "gradient")
                L.same_device(p.grad, p)
                key = p.grad.dtype, p.size(0), p.numel() // p.size(0)
                shapes[key] = shapes.get(key, 0) + 1
            for (dtype, m, n), b in shapes.items():
                ops.orthogonalize_check(dtype, b, m, n, steps, co, eps)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        self._check()
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
