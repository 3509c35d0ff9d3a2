"""Products of rows that are grouped by expert with the experts' MXFP8 weights (a mixture-of-experts layer's linear layers).

Rows come in the experts' order: expert e has the rows ``[offsets[e - 1], offsets[e])``, the first one from 0 on, with ``offsets`` an int32
tensor ``[experts]`` on the device that nothing reads on the host, so a call can be captured in a CUDA graph and replayed with other ends.
Ends that do not decrease and lie within the rows are the caller's to give; others give unspecified rows, no access outside the
tensors and no more work than there are rows.  An expert may have no rows; rows behind the last expert's are zeros in the result.

* :func:`grouped_mm_mxfp8`: both operands held in MXFP8, as :func:`comfy_kitchen.scaled_mm_mxfp8` takes them for one weight.
* :func:`grouped_linear_mxfp8`: dense rows, quantized on the way; differentiable in the rows (the weights stay frozen, and the quantization
  of the rows passes its gradient on unchanged, as in :func:`comfy_kitchen.linear_checkpointed`).
* :func:`grouped_input_grad_mxfp8`: that gradient.
* :class:`MXFP8Experts`: a module around them.

Weights are ``[experts, N, K]`` E4M3 codes and ``[experts, roundup(N, 128), roundup(K / 32, 4)]`` E8M0 scales, each expert's as
:func:`comfy_kitchen.quantize_mxfp8` gives them (:func:`quantize_experts_mxfp8`); K is a multiple of 32, N of 8.
"""
from __future__ import annotations

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from .float_utils import roundup
from .ops import DTYPE_TO_CODE, host_operator
from .training import _call, _eager, _no_tangents, _run, replaced

__all__ = ["grouped_mm_mxfp8", "grouped_linear_mxfp8", "grouped_input_grad_mxfp8", "quantize_experts_mxfp8", "MXFP8Experts"]


def grouped_mm_mxfp8(a: torch.Tensor, b: torch.Tensor, block_scale_a: torch.Tensor, block_scale_b: torch.Tensor, offsets: torch.Tensor,
                     bias: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``a[i] @ b[e].T + bias[e]`` for the rows i of expert e: ``[M, N]`` in ``out_dtype`` (bf16 by default), ``bias`` ``[experts, N]``."""
    out_dtype = out_dtype or torch.bfloat16
    host = host_operator("grouped_mm_mxfp8")
    if host is not None:
        out = host(a, b, block_scale_a, block_scale_b, offsets, bias, out_dtype)
        if out is not None:
            return out
    return _call("grouped_mm_mxfp8", {"a": a, "b": b, "block_scale_a": block_scale_a, "block_scale_b": block_scale_b, "offsets": offsets, "bias": bias,
                                      "out_dtype": out_dtype})


def grouped_input_grad_mxfp8(dy: torch.Tensor, w_codes: torch.Tensor, w_block_scales: torch.Tensor, offsets: torch.Tensor,
                             out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``dy[i] @ w[e]`` for the rows i of expert e: ``[M, K]`` in ``out_dtype`` (dy's by default).

    fp32 accumulation of exact products, one rounding."""
    out_dtype = out_dtype or dy.dtype
    host = host_operator("grouped_input_grad_mxfp8")
    if host is not None:
        out = host(dy, w_codes, w_block_scales, offsets, out_dtype)
        if out is not None:
            return out
    return _call("grouped_input_grad_mxfp8", {"dy": dy, "w_codes": w_codes, "w_block_scales": w_block_scales, "offsets": offsets, "out_dtype": out_dtype})


class _GroupedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_codes, w_block_scales, offsets, bias):
        ctx.save_for_backward(w_codes, w_block_scales, offsets)
        return _run("grouped_linear_mxfp8", {"x": x, "w_codes": w_codes, "w_block_scales": w_block_scales, "offsets": offsets, "bias": bias})

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        w_codes, w_block_scales, offsets = ctx.saved_tensors
        return grouped_input_grad_mxfp8(dy, w_codes, w_block_scales, offsets), None, None, None, None


def grouped_linear_mxfp8(x: torch.Tensor, w_codes: torch.Tensor, w_block_scales: torch.Tensor, offsets: torch.Tensor,
                         bias: torch.Tensor | None = None) -> torch.Tensor:
    """``x[i] @ w[e].T + bias[e]`` for the rows i of expert e, x ``[M, K]`` quantized to MXFP8 on the way: ``[M, N]`` in x's dtype.

    The result has x's gradient; the bias is frozen like the weight."""
    graph = torch.is_grad_enabled() and x.requires_grad
    if torch.is_grad_enabled() and bias is not None and bias.requires_grad:
        raise ValueError("grouped_linear_mxfp8 has no gradient of the bias: detach it")
    if not graph:
        host = host_operator("grouped_linear_mxfp8")
        if host is not None:
            out = host(x, w_codes, w_block_scales, offsets, bias)
            if out is not None:
                return out
    elif _eager((x, w_codes, w_block_scales, offsets, bias)) and not replaced("grouped_linear_mxfp8") and not replaced("grouped_input_grad_mxfp8"):
        return _GroupedLinear.apply(x, w_codes, w_block_scales, offsets, bias)
    _no_tangents("grouped_linear_mxfp8", x, bias)
    return _call("grouped_linear_mxfp8", {"x": x, "w_codes": w_codes, "w_block_scales": w_block_scales, "offsets": offsets, "bias": bias})


def quantize_experts_mxfp8(weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(codes, block_scales)`` of dense weights ``[experts, N, K]``, each expert's as ``quantize_mxfp8`` gives them."""
    if weight.dim() != 3 or weight.shape[2] % 32 != 0 or weight.shape[1] % 8 != 0:
        raise ValueError(f"experts' weights are [experts, N, K] with N a multiple of 8 and K of 32, got {tuple(weight.shape)}")
    from . import quantize_mxfp8

    experts, n, k = weight.shape
    if n % 128 == 0:  # one expert's scale tiles end where the next one's begin
        codes, scales = quantize_mxfp8(weight.reshape(experts * n, k))
        return codes.view(experts, n, k), scales.view(experts, n, -1)
    codes = torch.empty((experts, n, k), dtype=torch.float8_e4m3fn, device=weight.device)
    scales = torch.empty((experts, roundup(n, 128), roundup(k // 32, 4)), dtype=torch.float8_e8m0fnu, device=weight.device)
    for e in range(experts):
        c, s = quantize_mxfp8(weight[e].contiguous())
        codes[e].copy_(c)
        scales[e].view(torch.uint8).copy_(s.view(torch.uint8))
    return codes, scales


class MXFP8Experts(nn.Module):
    """The experts' linear layers of one projection with frozen MXFP8 weights: ``forward(x, offsets)`` on rows in the experts' order.

    Keys of its state dict, as those of ``MXFP8Linear`` with the experts in front: ``weight`` and ``weight_scale`` (codes and scales, kept as
    bytes), ``bias``."""

    def __init__(self, experts: int, in_features: int, out_features: int, bias: bool = False, device=None, dtype=None) -> None:
        super().__init__()
        if in_features % 32 != 0 or out_features % 8 != 0:
            raise ValueError(f"MXFP8 experts need input features of a multiple of 32 and output features of 8, got {in_features} and {out_features}")
        self.experts, self.in_features, self.out_features = experts, in_features, out_features
        u8 = {"dtype": torch.uint8, "device": device}
        self.register_buffer("weight", torch.zeros((experts, out_features, in_features), **u8))
        self.register_buffer("weight_scale", torch.zeros((experts, roundup(out_features, 128), roundup(in_features // 32, 4)), **u8))
        self.register_buffer("bias", torch.zeros((experts, out_features), device=device, dtype=dtype) if bias else None)

    @classmethod
    def from_float(cls, weight: torch.Tensor, bias: torch.Tensor | None = None) -> "MXFP8Experts":
        """From dense weights ``[experts, N, K]`` on the GPU."""
        codes, scales = quantize_experts_mxfp8(weight)
        experts, n, k = weight.shape
        m = cls(experts, k, n, bias is not None, device="meta")
        m.weight, m.weight_scale = codes.view(torch.uint8), scales.view(torch.uint8)
        m.bias = None if bias is None else bias.detach().clone()
        return m

    def forward(self, x: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
        return grouped_linear_mxfp8(x, self.weight.view(torch.float8_e4m3fn), self.weight_scale.view(torch.float8_e8m0fnu), offsets, self.bias)

    def extra_repr(self) -> str:
        return f"experts={self.experts}, in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"
