"""Orthogonalised updates of weight matrices.

``orthogonalise(update)`` brings the singular values of a matrix near 1 by Newton-Schulz products, as the Muon optimiser
does; ``orthogonal_step`` is the whole update of a list of weights, momentum included, and ``OrthogonalSGD`` the optimiser
around it.  The products run on the tensor cores, with operands held to 22 bits and 2^-37 of the matrix' norm, which leaves the
result within 1e-6 or so of itself, about as near as fp32 products.  An update with rows or columns so far below its others that
they would lose more than 2e-4 of themselves (a stretch with four or more that are not 0, and none of 2^-24 of the norm) goes by fp32 products without
tensor cores, at a tenth of the speed, and keeps all their digits.  The reference has no training loop of its own
(benchmark/parallel/benchmark_gcn_cpu.py:92-103 stops at the gradients).
"""
from __future__ import annotations

import math
from array import array

import torch

from . import _lib
from .dense import _call

QUINTIC = (3.4445, -4.7750, 2.0315)
MAX_STEPS = 64                          # include/cbm_b200.h, CBM_B200_MAX_STEPS
MAX_SIDE, MAX_STACK = 1 << 16, 1 << 15  # on the GPU


def _on_host(u, steps, eps):
    """By torch's elementary operations, for CPU tensors."""
    a, b, c = QUINTIC
    turned = u.size(-2) > u.size(-1)
    x = u.transpose(-1, -2) if turned else u
    x = x * (1.0 / (x.double().square().sum(dim=(-1, -2), keepdim=True).sqrt() + eps)).float()
    for _ in range(steps):
        gram = x @ x.transpose(-1, -2)
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.transpose(-1, -2).contiguous() if turned else x


def _check_steps(steps, eps):
    if not 1 <= steps <= MAX_STEPS:
        raise ValueError(f"steps must be between 1 and {MAX_STEPS}")
    if not eps >= 0.0:
        raise ValueError("eps must not be negative")


def _too_large(rows, cols):
    return f"{rows} x {cols}, sides of at most {MAX_SIDE} on the GPU" if max(rows, cols) > MAX_SIDE else None


def orthogonalise(update: torch.Tensor, steps: int = 5, eps: float = 1e-7) -> torch.Tensor:
    """``update`` [m, n] or [B, m, n] (fp32; each matrix for itself) divided by its norm plus ``eps`` and led towards the
    nearest matrix with orthonormal rows or columns by ``steps`` quintic Newton-Schulz products: five take singular values from
    a few thousandths of the norm up to between 0.68 and 1.21.  A matrix of zeros stays one.  Not differentiable.
    On the GPU sides of up to 65 536 and stacks of up to 32 768."""
    if update.dim() not in (2, 3):
        raise RuntimeError(f"orthogonalise: [m, n] or [B, m, n] expected, not {tuple(update.shape)}")
    if update.dtype != torch.float32:
        raise RuntimeError(f"orthogonalise: fp32 expected, not {update.dtype}")
    _check_steps(steps, eps)
    u = update.detach()
    if u.numel() == 0:
        return torch.empty_like(u)
    if not u.is_cuda:
        return _on_host(u, steps, eps)
    if _too_large(u.size(-2), u.size(-1)) or (u.dim() == 3 and u.size(0) > MAX_STACK):  # (asked here: the library's sizes have 32 bits)
        raise RuntimeError(f"orthogonalise: {tuple(u.shape)}, sides of at most {MAX_SIDE} and stacks of at most {MAX_STACK} on the GPU")
    if u.stride(-1) != 1 or u.stride(-2) < u.size(-1):
        u = u.contiguous()
    batch, rows, cols = (1, *u.shape) if u.dim() == 2 else u.shape
    out = torch.empty(u.shape, dtype=u.dtype, device=u.device)
    space = _lib.lib().cbm_b200_orthogonalise_workspace(batch, rows, cols)
    ws = torch.empty(space, dtype=torch.uint8, device=u.device)
    _call("cbm_b200_orthogonalise", u.get_device(), u.data_ptr(), max(u.stride(-2), cols), u.stride(0) if u.dim() == 3 else 0, out.data_ptr(), cols,
          rows * cols, batch, rows, cols, steps, eps, ws.data_ptr(), space)
    return out


def orthogonal_step(weights, grads, momenta, lr: float, momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0,
                    steps: int = 5, eps: float = 1e-7) -> None:
    """One update of every weight [m, n] of a list (fp32, unit column stride), in place, with its gradient and momentum::

        m <- momentum m + g;  u = g + momentum m (nesterov) or m
        w <- (1 - lr weight_decay) w - lr sqrt(max(1, rows / cols)) orthogonalise(u, steps, eps)

    All tensors of a call lie on one device; weights and momenta must not overlap one another or the gradients.  On the GPU
    sides of up to 65 536."""
    weights, grads, momenta = list(weights), list(grads), list(momenta)
    if not len(weights) == len(grads) == len(momenta):
        raise RuntimeError(f"orthogonal step: {len(weights)} weights, {len(grads)} gradients, {len(momenta)} momenta")
    _check_steps(steps, eps)
    if not weights:
        return
    dev = weights[0].device
    words, held = array("q"), []
    for w, g, m in zip(weights, grads, momenta):
        for t in (w, g, m):
            if t.dim() != 2 or t.shape != w.shape:
                raise RuntimeError(f"orthogonal step: shape mismatch, {tuple(w.shape)}, {tuple(g.shape)} and {tuple(m.shape)}")
            if t.dtype != torch.float32 or t.is_sparse:
                raise RuntimeError("orthogonal step: dense fp32 tensors expected")
            if t.device != dev:
                raise RuntimeError(f"orthogonal step: operands on {dev} and {t.device}")
    written = [t.data_ptr() for t in weights + momenta if t.numel() and t.device.type != "meta"]
    if len(set(written)) < len(written):
        raise RuntimeError("orthogonal step: a weight or a momentum is there twice")
    if not set(written).isdisjoint(g.data_ptr() for g in grads if g.numel() and g.device.type != "meta"):
        raise RuntimeError("orthogonal step: a gradient is a weight or a momentum, too")
    with torch.no_grad():
        if dev.type != "cuda":
            for w, g, m in zip(weights, grads, momenta):
                m.mul_(momentum).add_(g)
                o = _on_host(g + momentum * m if nesterov else m, steps, eps) if w.numel() else w
                w.mul_(1.0 - lr * weight_decay).add_(o, alpha=-lr * math.sqrt(max(1.0, w.size(0) / max(1, w.size(1)))))
            return
        for w, g, m in zip(weights, grads, momenta):
            if g.stride(1) != 1 or g.stride(0) < g.size(1):
                g = g.contiguous()
                held.append(g)
            for t in (w, m):
                if t.numel() and ((t.size(1) > 1 and t.stride(1) != 1) or (t.size(0) > 1 and t.stride(0) < t.size(1))):
                    raise RuntimeError("orthogonal step: weights and momenta of unit column stride expected")
            rows, cols = w.shape
            if _too_large(rows, cols):
                raise RuntimeError(f"orthogonal step: {_too_large(rows, cols)}")
            words.extend((w.data_ptr(), g.data_ptr(), m.data_ptr(), *(max(t.stride(0), cols) for t in (w, g, m)), rows | cols << 32))
        of = words.buffer_info()[0]
        space = _lib.lib().cbm_b200_orthogonal_step_workspace(of, len(weights))
        ws = torch.empty(space, dtype=torch.uint8, device=dev)
        _call("cbm_b200_orthogonal_step", weights[0].get_device(), of, len(weights), lr, momentum, int(nesterov), weight_decay, steps, eps,
              ws.data_ptr(), space)
    torch.autograd.graph.increment_version(weights + momenta)  # written without torch's knowledge


class OrthogonalSGD(torch.optim.Optimizer):
    """``orthogonal_step`` on the weights of dense maps.  Takes matrices alone, on the GPU with sides of up to 65 536: biases, norms and
    the embeddings of a large graph's nodes go to another optimiser."""

    def __init__(self, params, lr: float = 0.02, momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0, steps: int = 5,
                 eps: float = 1e-7):
        if not (lr >= 0.0 and 0.0 <= momentum < 1.0 and weight_decay >= 0.0):
            raise ValueError("lr and weight_decay must not be negative, momentum lies in [0, 1)")
        _check_steps(steps, eps)
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps, eps=eps))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        for p in self.param_groups[-1]["params"]:
            if p.dim() != 2 or p.dtype != torch.float32:
                raise ValueError(f"OrthogonalSGD updates fp32 matrices, not {p.dtype} of {tuple(p.shape)}")
            if p.is_cuda and _too_large(*p.shape):
                raise ValueError(f"OrthogonalSGD: {_too_large(*p.shape)}")

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            by_device = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                state = self.state[p]
                if "momentum" not in state:
                    state["momentum"] = torch.zeros(p.shape, dtype=p.dtype, device=p.device)
                by_device.setdefault(p.device, []).append((p, p.grad, state["momentum"]))
            for found in by_device.values():
                orthogonal_step(*zip(*found), lr=group["lr"], momentum=group["momentum"], nesterov=group["nesterov"],
                                weight_decay=group["weight_decay"], steps=group["steps"], eps=group["eps"])
        return loss
