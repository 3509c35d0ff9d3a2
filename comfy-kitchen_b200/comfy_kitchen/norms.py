"""Root-mean-square norm with the residual's addition, and the global norm of a model's gradients.

* :func:`rms_norm`: over the last dimension, with a weight (as it stands, or as the distance from ``weight_offset``) and, if a residual is given, of
  the sum, which is returned beside the result: ``y, h = rms_norm(x, weight, residual)`` is one pass where a layer would add, write,
  read and normalize.  Differentiable in x, residual and weight.
* :func:`rms_norm_mxfp8`: the same with the result in MXFP8, as the next layer's :func:`comfy_kitchen.scaled_mm_mxfp8` or
  :func:`comfy_kitchen.grouped_mm_mxfp8` takes it; what ``quantize_mxfp8`` gives for :func:`rms_norm`'s rows, up to the last bit of a row's norm (narrow rows
  and ones off 32-byte boundaries have their squares added in another order).  For inference: codes carry no gradient.
* :class:`RMSNorm`: a module around them.
* :func:`grad_norm`, :func:`clip_grad_norm_`: the 2-norm over all gradients, and their scaling where it is above a bound, in two launches for up
  to 1024 tensors and without a read on the host.

The arithmetic is fp32 with one rounding; the sum of x and residual is rounded to their type first, and the norm is of what stands there.
Gradients of gradients and forward-mode derivatives are refused.
"""
from __future__ import annotations

import math
from collections.abc import Iterable

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from .ops import host_operator, host_step
from .training import _call, _eager, _no_tangents, _run, replaced

__all__ = ["rms_norm", "rms_norm_forward", "rms_norm_backward", "rms_norm_mxfp8", "RMSNorm", "grad_norm", "clip_grad_norm_"]


# ---- the operators -----------------------------------------------------------------------------
def rms_norm_forward(x: torch.Tensor, weight: torch.Tensor | None = None, residual: torch.Tensor | None = None, eps: float = 1e-6,
                     weight_offset: float = 0.0) -> tuple[torch.Tensor, torch.Tensor | None, torch.Tensor]:
    """``(y, h, rstd)`` of :func:`rms_norm`: the result, the sum (None without a residual) and the fp32 inverse root of each row, which carries
    no gradient."""
    y, h, rstd = _call("rms_norm_forward", {"x": x, "weight": weight, "residual": residual, "eps": float(eps), "weight_offset": float(weight_offset)})
    return y, None if residual is None else h, rstd


def rms_norm_backward(dy: torch.Tensor, h: torch.Tensor, rstd: torch.Tensor, weight: torch.Tensor | None = None, dh: torch.Tensor | None = None,
                      weight_offset: float = 0.0) -> tuple[torch.Tensor, torch.Tensor | None]:
    """``(dx, dweight)`` of :func:`rms_norm`, ``h`` what was normalized and ``dh`` the gradient that reaches it by other ways; dx is
    x's and the residual's gradient alike, dweight None without a weight."""
    dx, dweight = _call("rms_norm_backward", {"dy": dy, "h": h, "rstd": rstd, "weight": weight, "dh": dh, "weight_offset": float(weight_offset),
                                              "weight_grad": weight is not None})
    return dx, None if weight is None else dweight


def rms_norm_mxfp8(x: torch.Tensor, weight: torch.Tensor | None = None, residual: torch.Tensor | None = None, eps: float = 1e-6,
                   weight_offset: float = 0.0) -> tuple[torch.Tensor, ...]:
    """``quantize_mxfp8`` of :func:`rms_norm`'s rows from one pass: ``(codes, block_scales)``, or with a residual ``(codes, block_scales, h)``.

    Codes are ``[rows, cols]`` whatever x's rank; cols is a multiple of 32."""
    eps, weight_offset = float(eps), float(weight_offset)
    host = host_operator("rms_norm_mxfp8")
    if host is not None:
        out = host(x, weight, residual, eps, weight_offset)
        if out is not None:
            return out
    if x.dim() == 0 or x.shape[-1] % 32 != 0:
        raise ValueError(f"an MXFP8 result needs rows of a multiple of 32, got {tuple(x.shape)}")
    codes, scales, h = _call("rms_norm_mxfp8", {"x": x, "weight": weight, "residual": residual, "eps": eps, "weight_offset": weight_offset})
    return (codes, scales) if residual is None else (codes, scales, h)


# ---- autograd ----------------------------------------------------------------------------------
class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps, weight_offset):
        y, h, rstd = _run("rms_norm_forward", {"x": x, "weight": weight, "residual": residual, "eps": eps, "weight_offset": weight_offset})
        ctx.save_for_backward(x if h is None else h, rstd, weight)
        ctx.weight_offset = weight_offset
        ctx.set_materialize_grads(False)
        return y if h is None else (y, h)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh=None):
        h, rstd, weight = ctx.saved_tensors
        need = ctx.needs_input_grad
        if dy is None:
            return dh if need[0] else None, None, dh if need[2] else None, None, None
        dx, dweight = _run("rms_norm_backward", {"dy": dy, "h": h, "rstd": rstd, "weight": weight, "dh": dh, "weight_offset": ctx.weight_offset,
                                                 "weight_grad": need[1]})
        return dx if need[0] else None, dweight if need[1] else None, dx if need[2] else None, None, None


_TRAINING, _INFERENCE = ("rms_norm_forward", "rms_norm_backward"), ("rms_norm_forward",)


def rms_norm(x: torch.Tensor, weight: torch.Tensor | None = None, residual: torch.Tensor | None = None, eps: float = 1e-6,
             weight_offset: float = 0.0):
    """RMS norm over the last dimension: ``h / sqrt(mean(h * h) + eps) * (weight_offset + weight)`` with ``h = x + residual``, or x itself.

    Returns y, or ``(y, h)`` with a residual.  ``weight`` (None: no factor) is ``[cols]`` of x's dtype or float32, ``residual`` of x's shape and
    dtype; x and residual may be slices of larger tensors."""
    eps, weight_offset = float(eps), float(weight_offset)
    graph = torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or (residual is not None and residual.requires_grad))
    operators = _TRAINING if graph else _INFERENCE
    host = host_step("rms_norm", operators)
    if host is not None:
        out = host(x, weight, residual, eps, weight_offset)
        if out is not None:
            return out
    if _eager((x, weight, residual)) and not any(replaced(name) for name in operators):
        if graph:
            return _RmsNorm.apply(x, weight, residual, eps, weight_offset)
        y, h = _run("rms_norm_inference", {"x": x, "weight": weight, "residual": residual, "eps": eps, "weight_offset": weight_offset})
    else:
        _no_tangents("rms_norm", x, weight, residual)
        y, h, _ = torch.ops.comfy_kitchen.rms_norm_forward(x, weight, residual, eps, weight_offset)
    return y if residual is None else (y, h)


class RMSNorm(nn.Module):
    """RMS norm over the last dimension with a learned weight; ``forward(x, residual)`` returns ``(y, x + residual)``.

    The parameter is named as ``nn.RMSNorm`` names it; ``eps`` is 1e-6 unless given, where torch's module takes the input type's epsilon."""

    def __init__(self, features: int, eps: float = 1e-6, device=None, dtype=None) -> None:
        super().__init__()
        self.features, self.eps = features, eps
        self.weight = nn.Parameter(torch.ones(features, device=device, dtype=dtype))

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None):
        return rms_norm(x, self.weight, residual, self.eps)

    def extra_repr(self) -> str:
        return f"{self.features}, eps={self.eps}"


# ---- gradients ---------------------------------------------------------------------------------
def _list_call(name: str, grads: list[torch.Tensor], *args):
    if _eager(grads) and not replaced(name):
        out = _run(name, {"grads": grads, **({"max_norm": args[0]} if args else {})})
        if args:
            torch.autograd.graph.increment_version(grads)
        return out
    return getattr(torch.ops.comfy_kitchen, name)(grads, *args)


def grad_norm(tensors: Iterable[torch.Tensor]) -> torch.Tensor:
    """The 2-norm of all elements of the tensors (bf16, fp16 or fp32, on one GPU): a 0-d float32 tensor on that GPU, for no tensors a zero on the CPU."""
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    if not tensors:
        return torch.zeros((), dtype=torch.float32)
    dense = [t.detach() if t.is_contiguous() else t.detach().contiguous() for t in tensors]
    return _list_call("grad_norm", dense)


def clip_grad_norm_(parameters: Iterable[torch.Tensor] | torch.Tensor, max_norm: float, error_if_nonfinite: bool = False) -> torch.Tensor:
    """``torch.nn.utils.clip_grad_norm_`` for the 2-norm: every gradient times ``min(1, max_norm / (norm + 1e-6))``, in place; returns the norm,
    0-d float32 (where no parameter has a gradient a zero on the first one's device).

    Gradients are bf16, fp16 or fp32, mixed at will, on one GPU, and do not overlap (a parameter that is given twice counts once).  Nothing is read
    on the host, so a step can be captured, except with ``error_if_nonfinite``, which raises before a gradient is changed."""
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must not be negative, got {max_norm}")
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    if not error_if_nonfinite:
        host = host_step("clip_grad_norm", ("clip_grads",))
        if host is not None:
            norm = host(parameters, max_norm)
            if norm is not None:
                return norm
    grads = list({id(p): p.grad for p in parameters if p.grad is not None}.values())
    if not grads:
        return torch.zeros((), dtype=torch.float32, device=parameters[0].device if parameters else None)
    if error_if_nonfinite:
        norm = grad_norm(grads)
        if not math.isfinite(norm.item()):
            raise RuntimeError(f"The total norm of the gradients is {norm.item()}, so it cannot be clipped")
    if all(g.is_contiguous() and not g.is_neg() for g in grads):
        return _list_call("clip_grads", grads, max_norm)
    dense = [g.resolve_neg().contiguous() for g in grads]
    norm = _list_call("clip_grads", dense, max_norm)
    with torch.no_grad():
        for g, d in zip(grads, dense):
            if d is not g:
                g.copy_(d)
    return norm
