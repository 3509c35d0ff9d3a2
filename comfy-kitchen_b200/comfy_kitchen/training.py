"""Training operators: layer norm, GELU and linear layers whose saved activations are MXFP8 copies.

A layer of a transformer keeps its input for its backward pass, two or four bytes an element.  The functions here keep the
MXFP8 form that the quantized linears use (E4M3 codes, one E8M0 scale for 32 of a row: 1.03 bytes), write it in
the same pass that computes the result, and read it in the backward pass without a dense copy in between.  Results of the forward pass are
those of the dense input.  Gradients are taken at the values that stand in the copy: those of GELU and of a linear layer's weight are the
exact derivatives there; the norm's are its formula with the copy's values in the input's place beside the statistics of the dense input,
so not exactly the derivative of anything (these values' own mean and variance are others).

* :func:`layer_norm`: over the last dimension, with a learned weight and bias or with one row of them for each sample
  (``weight_offset=1`` and the scale and shift of a modulated norm).  Differentiable with and without a copy of its input.
* :func:`gelu_checkpointed`: tanh-form GELU.
* :func:`linear_checkpointed`: a linear layer with a dense weight, whose gradient comes from the copy of its input, or with
  a frozen MXFP8 weight, through which the input's gradient is taken.
* :class:`CheckpointedLayerNorm`, :class:`CheckpointedGELU`, :class:`CheckpointedLinear`, :class:`CheckpointedMLP`: modules around them.

The functions that these are built from (``layer_norm_forward`` ... ``linear_input_grad_mxfp8``) are operators of the package like
the quantizers; statistics and copies that they return carry no gradient, and gradients of gradients are not available.
"""
from __future__ import annotations

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from .ops import _MAY_BE_PENDING, _PLAIN_TYPES, DTYPE_TO_CODE, _impl, dispatcher_adds_nothing, host_operator, host_step, replaced
from .tensor import QuantizedTensor, TensorCoreMXFP8Layout
from .tensor.blockwise import crop, strict_status_check

BLOCK = 32  # elements of one scale


def _run(name: str, kwargs: dict):
    """An operator straight from the registry; under CK_STRICT=1 a wait in its kernels that gave up raises here."""
    out = _impl(name, kwargs)
    strict_status_check(name)
    return out


def _call(name: str, kwargs: dict):
    """An operator without a gradient: straight to the registry where the dispatcher would add nothing."""
    tensors = [v for v in kwargs.values() if isinstance(v, torch.Tensor)]
    if not replaced(name) and dispatcher_adds_nothing(tensors):
        return _run(name, kwargs)
    return getattr(torch.ops.comfy_kitchen, name)(*[DTYPE_TO_CODE[v] if isinstance(v, torch.dtype) else v for v in kwargs.values()])


# ---- the operators -----------------------------------------------------------------------------
def layer_norm_forward(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, eps: float = 1e-5,
                       weight_offset: float = 0.0) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(y, mean, rstd)`` of :func:`layer_norm`: the result and the fp32 statistics of each row, which carry no gradient."""
    return _call("layer_norm_forward", {"x": x, "weight": weight, "bias": bias, "eps": float(eps), "weight_offset": float(weight_offset)})


def layer_norm_forward_mxfp8(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, eps: float = 1e-5,
                             weight_offset: float = 0.0) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(y, mean, rstd, codes, block_scales)``: :func:`layer_norm_forward` and ``quantize_mxfp8`` of x's rows from one pass."""
    return _call("layer_norm_forward_mxfp8", {"x": x, "weight": weight, "bias": bias, "eps": float(eps), "weight_offset": float(weight_offset)})


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor, weight: torch.Tensor | None = None,
                        weight_offset: float = 0.0, groups: int = 1,
                        param_dtype: torch.dtype | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(dx, dweight, dbias)``; the last two ``[groups, cols]`` in ``param_dtype`` (the weight's, or dy's without one)."""
    param_dtype = param_dtype or (dy.dtype if weight is None else weight.dtype)
    return _call("layer_norm_backward", {"dy": dy, "x": x, "mean": mean, "rstd": rstd, "weight": weight, "weight_offset": float(weight_offset),
                                         "groups": groups, "param_dtype": param_dtype})


def layer_norm_backward_mxfp8(dy: torch.Tensor, codes: torch.Tensor, block_scales: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
                              weight: torch.Tensor | None = None, weight_offset: float = 0.0, groups: int = 1,
                              param_dtype: torch.dtype | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """:func:`layer_norm_backward` from the MXFP8 copy of x."""
    param_dtype = param_dtype or (dy.dtype if weight is None else weight.dtype)
    return _call("layer_norm_backward_mxfp8", {"dy": dy, "codes": codes, "block_scales": block_scales, "mean": mean, "rstd": rstd, "weight": weight,
                                               "weight_offset": float(weight_offset), "groups": groups, "param_dtype": param_dtype})


def gelu_mxfp8_forward(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(gelu_tanh(x), *quantize_mxfp8(x))`` of a 2-D tensor from one pass."""
    return _call("gelu_mxfp8_forward", {"x": x})


def gelu_mxfp8_backward(dy: torch.Tensor, codes: torch.Tensor, block_scales: torch.Tensor) -> torch.Tensor:
    """``dy`` times the derivative of the tanh-form GELU at the values that stand in the MXFP8 copy."""
    return _call("gelu_mxfp8_backward", {"dy": dy, "codes": codes, "block_scales": block_scales})


def linear_weight_grad_mxfp8(dy: torch.Tensor, x_codes: torch.Tensor, x_block_scales: torch.Tensor, out_dtype: torch.dtype | None = None,
                             bias_grad: bool = False) -> tuple[torch.Tensor, torch.Tensor | None]:
    """``(dy.T @ x, dy.sum(0) or None)`` with ``dy`` [M, N] and x [M, K] held in MXFP8, in ``out_dtype`` (dy's by default).

    fp32 accumulation of exact products, one rounding; N a multiple of 8, K of 32."""
    host = host_operator("linear_weight_grad_mxfp8")
    if host is not None:
        out = host(dy, x_codes, x_block_scales, out_dtype, bias_grad)
        if out is not None:
            return out
    dweight, dbias = _call("linear_weight_grad_mxfp8", {"dy": dy, "x_codes": x_codes, "x_block_scales": x_block_scales,
                                                        "out_dtype": out_dtype or dy.dtype, "bias_grad": bool(bias_grad)})
    return dweight, dbias if bias_grad else None


def linear_input_grad_mxfp8(dy: torch.Tensor, w_codes: torch.Tensor, w_block_scales: torch.Tensor,
                            out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``dy @ w`` with ``dy`` [M, N] and a linear layer's weight w [N, K] held in MXFP8, in ``out_dtype`` (dy's by default).

    fp32 accumulation of exact products, one rounding; N a multiple of 8, K of 32."""
    host = host_operator("linear_input_grad_mxfp8")
    if host is not None:
        out = host(dy, w_codes, w_block_scales, out_dtype)
        if out is not None:
            return out
    return _call("linear_input_grad_mxfp8", {"dy": dy, "w_codes": w_codes, "w_block_scales": w_block_scales, "out_dtype": out_dtype or dy.dtype})


# ---- autograd ----------------------------------------------------------------------------------
def _eager(tensors) -> bool:
    """True when the dispatcher would add nothing but the autograd graph: plain CUDA tensors, nobody who watches or rewrites
    operator calls (as :func:`comfy_kitchen.ops.dispatcher_adds_nothing`, with gradients)."""
    if torch.compiler.is_compiling() or torch.autograd._profiler_enabled() or torch._C._get_tracing_state() is not None or \
            torch._C._len_torch_dispatch_stack() or torch._C._len_torch_function_stack() or \
            torch._C._functorch.peek_interpreter_stack() is not None or torch.autograd.forward_ad._current_level >= 0:
        return False
    for t in tensors:
        if t is not None and (type(t) not in _PLAIN_TYPES or not t.is_cuda or (t.dtype in _MAY_BE_PENDING and (t.is_neg() or t._is_zerotensor()))):
            return False
    return True


def _groups(*params) -> int:
    return next((p.shape[0] for p in params if p is not None and p.dim() > 1), 1)


def _param_grads(ctx, dweight, dbias):
    shape = ctx.param_shape
    return (dweight.view(shape) if ctx.needs_input_grad[1] else None), (dbias.view(shape) if ctx.needs_input_grad[2] else None)


_NORM_OPERATORS = {False: ("layer_norm_forward", "layer_norm_backward"), True: ("layer_norm_forward_mxfp8", "layer_norm_backward_mxfp8")}
_NORM_INFERENCE = ("layer_norm_forward",)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, weight_offset, checkpoint):
        kwargs = {"x": x, "weight": weight, "bias": bias, "eps": eps, "weight_offset": weight_offset}
        if checkpoint:
            y, mean, rstd, codes, scales = _run("layer_norm_forward_mxfp8", kwargs)
            ctx.save_for_backward(codes, scales, mean, rstd, weight)
        else:
            y, mean, rstd = _run("layer_norm_forward", kwargs)
            ctx.save_for_backward(x, mean, rstd, weight)
        some = weight if weight is not None else bias
        ctx.param_shape, ctx.param_dtype = (some.shape, some.dtype) if some is not None else (None, x.dtype)
        ctx.weight_offset, ctx.groups = weight_offset, _groups(weight, bias)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        *held, mean, rstd, weight = ctx.saved_tensors
        kwargs = {"dy": dy, "mean": mean, "rstd": rstd, "weight": weight, "weight_offset": ctx.weight_offset, "groups": ctx.groups,
                  "param_dtype": ctx.param_dtype, "weight_grad": ctx.needs_input_grad[1], "bias_grad": ctx.needs_input_grad[2]}
        if len(held) == 2:
            dx, dweight, dbias = _run("layer_norm_backward_mxfp8", {**kwargs, "codes": held[0], "block_scales": held[1]})
        else:
            dx, dweight, dbias = _run("layer_norm_backward", {**kwargs, "x": held[0]})
        return (dx if ctx.needs_input_grad[0] else None, *_param_grads(ctx, dweight, dbias), None, None, None)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, eps: float = 1e-5,
               weight_offset: float = 0.0, checkpoint: bool = False) -> torch.Tensor:
    """Layer norm over x's last dimension: ``(x - mean) / sqrt(var + eps) * (weight_offset + weight) + bias``.

    ``weight`` and ``bias`` (each may be None; both of the same shape and dtype, x's or float32) are ``[cols]``, or
    ``[groups, cols]`` where groups is x's first dimension: ``layer_norm(x, scale, shift, weight_offset=1.0)`` is the modulated norm of a
    diffusion transformer, with ``scale`` and ``shift`` for each sample.  x may be a slice of a larger tensor.  The arithmetic is
    fp32 with one rounding.  With ``checkpoint`` the backward pass works from an MXFP8 copy of x (the last dimension a
    multiple of 32) instead of x itself."""
    eps, weight_offset = float(eps), float(weight_offset)
    graph = torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or (bias is not None and bias.requires_grad))
    operators = _NORM_OPERATORS[bool(checkpoint)] if graph else _NORM_INFERENCE  # a copy that nothing reads is not made
    host = host_step("layer_norm", operators)
    if host is not None:
        y = host(x, weight, bias, eps, weight_offset, checkpoint)
        if y is not None:
            return y
    if checkpoint and x.shape[-1] % BLOCK != 0:
        raise ValueError(f"an MXFP8 checkpoint needs rows of a multiple of {BLOCK}, got {x.shape[-1]}")
    if _eager((x, weight, bias)) and not any(replaced(name) for name in operators):
        if graph:
            return _LayerNorm.apply(x, weight, bias, eps, weight_offset, checkpoint)
        return _run("layer_norm_inference", {"x": x, "weight": weight, "bias": bias, "eps": eps, "weight_offset": weight_offset})
    op = torch.ops.comfy_kitchen.layer_norm_forward_mxfp8 if checkpoint and graph else torch.ops.comfy_kitchen.layer_norm_forward
    return op(x, weight, bias, eps, weight_offset)[0]


_GELU_OPERATORS = ("gelu_mxfp8_forward", "gelu_mxfp8_backward")


class _Gelu(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x):
        y, codes, scales = _run("gelu_mxfp8_forward", {"x": x})
        ctx.save_for_backward(codes, scales)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        codes, scales = ctx.saved_tensors
        return _run("gelu_mxfp8_backward", {"dy": dy, "codes": codes, "block_scales": scales})


def gelu_checkpointed(x: torch.Tensor) -> torch.Tensor:
    """Tanh-form GELU whose backward pass works from an MXFP8 copy of x (the last dimension a multiple of 32)."""
    graph = torch.is_grad_enabled() and x.requires_grad
    operators = _GELU_OPERATORS if graph else _GELU_OPERATORS[:1]
    host = host_step("gelu_checkpointed", operators)
    if host is not None:
        y = host(x)
        if y is not None:
            return y
    if x.dim() == 0 or x.shape[-1] % BLOCK != 0:
        raise ValueError(f"an MXFP8 checkpoint needs rows of a multiple of {BLOCK}, got {tuple(x.shape)}")
    shape = x.shape
    x2 = x if len(shape) == 2 else x.reshape(-1, shape[-1])
    if _eager((x2,)) and not any(replaced(name) for name in operators):
        y = _Gelu.apply(x2) if graph else _run("gelu_inference", {"x": x2})
    else:
        y = torch.ops.comfy_kitchen.gelu_mxfp8_forward(x2)[0]
    return y if len(shape) == 2 else y.view(shape)


class _Linear(torch.autograd.Function):
    """A dense weight: x is kept as its MXFP8 copy."""

    @staticmethod
    def forward(ctx, x, weight, bias):
        codes = scales = None
        if ctx.needs_input_grad[1]:
            codes, scales = _call("quantize_mxfp8", {"x": x.contiguous(), "pad_32x": False})
        ctx.save_for_backward(codes, scales, weight if ctx.needs_input_grad[0] else None)
        ctx.weight_dtype = weight.dtype
        return F.linear(x, weight, bias)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        codes, scales, weight = ctx.saved_tensors
        dx = dy @ weight if ctx.needs_input_grad[0] else None
        dweight = dbias = None
        if ctx.needs_input_grad[1]:
            dweight, dbias = linear_weight_grad_mxfp8(dy, codes, scales, ctx.weight_dtype, ctx.needs_input_grad[2])
        elif ctx.needs_input_grad[2]:
            dbias = dy.sum(0)
        return dx, dweight, dbias


class _FrozenLinear(torch.autograd.Function):
    """An MXFP8 weight: nothing of x is kept."""

    @staticmethod
    def forward(ctx, x, weight, bias):
        ctx.save_for_backward(weight._qdata, weight._params.scale)
        ctx.shape = weight._params.orig_shape
        padded = weight._qdata.shape[0] - ctx.shape[0]  # rows up to the scale block's size
        if bias is not None and padded:
            bias = F.pad(bias, (0, padded))
        with torch.no_grad():
            y = TensorCoreMXFP8Layout.scaled_mm(QuantizedTensor.from_float(x.contiguous(), "TensorCoreMXFP8Layout"), weight, bias, x.dtype)
        strict_status_check("linear_checkpointed")
        return crop(y, x.shape[0], ctx.shape[0])

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        dx = None
        if ctx.needs_input_grad[0]:
            codes, scales = ctx.saved_tensors
            rows, cols = ctx.shape
            padded = dy if codes.shape[0] == rows else F.pad(dy, (0, codes.shape[0] - rows))
            dx = linear_input_grad_mxfp8(padded, codes, scales)
            dx = dx if codes.shape[1] == cols else dx[:, :cols]
        return dx, None, dy.sum(0) if ctx.needs_input_grad[2] else None


def linear_checkpointed(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None) -> torch.Tensor:
    """``F.linear(x, weight, bias)`` for training.

    A dense ``weight`` [N, K] (of x's dtype, or of any under autocast; N a multiple of 8, K of 32): the result is the dense product, and the weight's
    and the bias's gradients come from an MXFP8 copy of x, which is all that is kept of it.  A ``QuantizedTensor`` in the MXFP8
    layout: x is quantized and multiplied as in ``MXFP8Linear``, the weight stays frozen, and the input's gradient is taken
    through it (the quantization of x passes its gradient on unchanged)."""
    shape = x.shape
    frozen = isinstance(weight, QuantizedTensor)
    if frozen and (weight.layout_cls is not TensorCoreMXFP8Layout or weight._params.transposed):
        raise ValueError("linear_checkpointed takes a dense weight or one in the MXFP8 layout")
    n, k = weight._params.orig_shape if frozen else weight.shape
    if x.dim() == 0 or shape[-1] != k:
        raise ValueError(f"the weight is [{n}, {k}], the input {tuple(shape)}")
    if not frozen:
        if k % BLOCK != 0 or n % 8 != 0:
            raise ValueError(f"an MXFP8 checkpoint needs input features of a multiple of {BLOCK} and output features of 8, got [{n}, {k}]")
        if x.is_cuda and torch.is_autocast_enabled("cuda"):
            dtype = torch.get_autocast_dtype("cuda")
            x, weight, bias = x.to(dtype), weight.to(dtype), bias if bias is None else bias.to(dtype)
        if weight.dtype != x.dtype:
            raise ValueError(f"the weight is {weight.dtype}, the input {x.dtype}")
    if x.numel() == 0:  # nothing to keep
        return F.linear(x, weight.dequantize().to(x.dtype) if frozen else weight, bias)
    if not torch.is_grad_enabled() and not frozen:
        return F.linear(x, weight, bias)
    x2 = x if x.dim() == 2 else x.reshape(-1, k)
    y = (_FrozenLinear if frozen else _Linear).apply(x2, weight, bias)
    return y if x.dim() == 2 else y.view(*shape[:-1], n)


# ---- modules -----------------------------------------------------------------------------------
class CheckpointedLayerNorm(nn.LayerNorm):
    """``nn.LayerNorm`` over the last dimension that keeps its input in MXFP8 for the backward pass."""

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if len(self.normalized_shape) != 1:
            raise ValueError("CheckpointedLayerNorm is over the last dimension")
        if x.shape[-1:] != torch.Size(self.normalized_shape):
            raise ValueError(f"the norm is over rows of {self.normalized_shape[0]}, the input {tuple(x.shape)}")
        return layer_norm(x, self.weight, self.bias, self.eps, checkpoint=True)


class CheckpointedGELU(nn.Module):
    """Tanh-form GELU that keeps its input in MXFP8 for the backward pass."""

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return gelu_checkpointed(x)


class CheckpointedLinear(nn.Linear):
    """``nn.Linear`` that keeps its input in MXFP8 for the weight's gradient."""

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return linear_checkpointed(x, self.weight, self.bias)


class CheckpointedMLP(nn.Module):
    """``x + fc2(gelu(fc1(norm(x))))``, the MLP half of a transformer block, every activation that it keeps in MXFP8."""

    def __init__(self, features: int, hidden: int, eps: float = 1e-5, device=None, dtype=None) -> None:
        super().__init__()
        self.norm = CheckpointedLayerNorm(features, eps=eps, device=device, dtype=dtype)
        self.fc1 = CheckpointedLinear(features, hidden, device=device, dtype=dtype)
        self.act = CheckpointedGELU()
        self.fc2 = CheckpointedLinear(hidden, features, device=device, dtype=dtype)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return x + self.fc2(self.act(self.fc1(self.norm(x))))
