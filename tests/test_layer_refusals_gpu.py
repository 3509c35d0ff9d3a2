"""What RMS norm, the experts' products and clipping refuse on the GPU, and in which words; nothing is changed by a refused call."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ck(cuda_device):
    import comfy_kitchen

    assert comfy_kitchen.list_backends()["cuda"]["available"]
    return comfy_kitchen


def _zeros(*shape, dtype=torch.float32, **kw):
    return torch.zeros(*shape, dtype=dtype, device="cuda", **kw)


def test_experts(ck):
    codes, scales = ck.quantize_experts_mxfp8(torch.ones(2, 64, 32, device="cuda"))
    ends, x = torch.tensor([1, 2], dtype=torch.int32, device="cuda"), torch.ones(2, 32, device="cuda")
    xc, xs = ck.quantize_mxfp8(x)
    cases = [
        (ck.NoCapableBackendError, "offsets: dtype", lambda: ck.grouped_linear_mxfp8(x, codes, scales, ends.long())),
        (ck.NoCapableBackendError, "offsets: device", lambda: ck.grouped_linear_mxfp8(x, codes, scales, ends.cpu())),
        (ck.NoCapableBackendError, "x: dtype", lambda: ck.grouped_linear_mxfp8(x.double(), codes, scales, ends)),
        (ck.NoCapableBackendError, "dy: dtype", lambda: ck.grouped_input_grad_mxfp8(_zeros(2, 64, dtype=torch.float64), codes, scales, ends, torch.float32)),
        (ck.NoCapableBackendError, "x: shape", lambda: ck.grouped_linear_mxfp8(x.view(1, 2, 32), codes, scales, ends)),
        (AssertionError, "one int32 end for each expert", lambda: ck.grouped_linear_mxfp8(x, codes, scales, ends[:1])),
        (AssertionError, "contiguous", lambda: ck.grouped_linear_mxfp8(x, codes, scales, ends.repeat(2)[::2])),
        (AssertionError, "contiguous", lambda: ck.grouped_linear_mxfp8(x, codes.transpose(1, 2).contiguous().transpose(1, 2), scales, ends)),
        (AssertionError, "dimensions do not match", lambda: ck.grouped_linear_mxfp8(x[:, :16], codes, scales, ends)),
        (AssertionError, "dimensions do not match", lambda: ck.grouped_input_grad_mxfp8(x, codes, scales, ends)),
        (AssertionError, "Invalid scale shape", lambda: ck.grouped_linear_mxfp8(x, codes, scales[:1], ends)),
        (AssertionError, "Invalid A scale shape", lambda: ck.grouped_mm_mxfp8(xc, codes, xs[:64], scales, ends)),
        (AssertionError, "bias must be", lambda: ck.grouped_linear_mxfp8(x, codes, scales, ends, _zeros(2, 63))),
        (ValueError, "no gradient of the bias", lambda: ck.grouped_linear_mxfp8(x, codes, scales, ends, _zeros(2, 64, requires_grad=True))),
        (ValueError, "N a multiple of 8", lambda: ck.quantize_experts_mxfp8(_zeros(2, 60, 32))),
        (ValueError, "multiple of 32", lambda: ck.experts.MXFP8Experts(2, 48, 64)),
    ]
    for kind, said, call in cases:
        with pytest.raises(kind, match=said):
            call()
    assert torch.equal(ck.grouped_linear_mxfp8(x, codes, scales, ends), torch.full((2, 64), 32.0, device="cuda"))


def test_norm(ck):
    x = torch.ones(4, 64, device="cuda")
    cases = [
        (AssertionError, "of the input's dtype or float32", lambda: ck.rms_norm(x, _zeros(64, dtype=torch.float16))),
        (AssertionError, r"must be \[64\]", lambda: ck.rms_norm(x, _zeros(63))),
        (AssertionError, "same shape and dtype", lambda: ck.rms_norm(x, None, x[:1])),
        (AssertionError, "same shape and dtype", lambda: ck.rms_norm(x, None, x.half())),
        (AssertionError, "one element at least", lambda: ck.rms_norm(_zeros(3, 0))),
        (AssertionError, "one fp32 value for each row", lambda: ck.rms_norm_backward(x, x, _zeros(3))),
        (ck.NoCapableBackendError, "x: shape", lambda: ck.rms_norm(_zeros(()))),
        (ck.NoCapableBackendError, "x: dtype", lambda: ck.rms_norm(x.double())),
        (ck.NoCapableBackendError, "weight: device", lambda: ck.rms_norm(x, torch.zeros(64))),
        (ValueError, "multiple of 32", lambda: ck.rms_norm_mxfp8(x[:, :40])),
    ]
    for kind, said, call in cases:
        with pytest.raises(kind, match=said):
            call()
    assert torch.equal(ck.rms_norm(x, eps=0.0), x)


def test_clipping(ck):
    def params(*grads):
        out = []
        for g in grads:
            p = torch.nn.Parameter(torch.empty_like(g))
            p.grad = g
            out.append(p)
        return out

    flat = torch.ones(100, device="cuda")
    cases = [
        (RuntimeError, "overlap", lambda: ck.clip_grad_norm_(params(flat[:60], flat[50:]), 1.0)),
        (ValueError, "max_norm", lambda: ck.clip_grad_norm_(params(flat), -1.0)),
        (ValueError, "max_norm", lambda: ck.clip_grad_norm_(params(flat), float("nan"))),
        (AssertionError, "float64", lambda: ck.clip_grad_norm_(params(flat.double()), 1.0)),
        (AssertionError, "complex64", lambda: ck.grad_norm([flat, flat.to(torch.complex64)])),
        (AssertionError, "one device", lambda: ck.clip_grad_norm_(params(flat, flat.cpu()), 1.0)),
        (AssertionError, "on the GPU", lambda: ck.clip_grad_norm_(params(flat.cpu()), 1.0)),
    ]
    for kind, said, call in cases:
        with pytest.raises(kind, match=said):
            call()
    assert torch.equal(flat, torch.ones_like(flat))
    assert ck.clip_grad_norm_(params(flat[:50], flat[50:]), 5.0).item() == 10.0 and torch.equal(flat, torch.full_like(flat, 5.0) / (10.0 + 1e-6))
