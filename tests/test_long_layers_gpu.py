"""RMS norm, experts' products and clipping on tensors with more elements than 32 bits count, on the GPU: their last rows against calls on those rows alone."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ck(cuda_device):
    import comfy_kitchen

    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB")
    yield comfy_kitchen
    torch.cuda.empty_cache()


def _filled(rows, cols, dtype, seed):
    """[rows, cols] of which the last 300 rows are drawn, the others one value"""
    t = torch.full((rows, cols), 0.5, device="cuda", dtype=dtype)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    t[-300:] = torch.randn(300, cols, generator=gen, device="cuda").to(dtype)
    return t


def test_rms_norm(ck):
    rows, cols = 2**32 // 4096 + 1100, 4096
    x, w = _filled(rows, cols, torch.bfloat16, 1), torch.linspace(0.5, 2, cols, device="cuda").to(torch.bfloat16)
    last = x[-300:].clone()
    y, h, rstd = ck.rms_norm_forward(x, w)
    assert torch.equal(y[-300:], ck.rms_norm(last, w)) and h is None
    codes, scales = ck.rms_norm_mxfp8(x, w)
    one, _ = ck.rms_norm_mxfp8(last, w)
    assert torch.equal(codes[-300:].view(torch.uint8), one.view(torch.uint8))
    del codes, scales
    dx, _ = ck.rms_norm_backward(y, x, rstd, w)
    alone, _ = ck.rms_norm_backward(y[-300:].clone(), last, rstd[-300:].clone(), w)
    assert torch.equal(dx[-300:], alone)


def test_many_rows_through_experts(ck):
    rows, n, k = 2**32 // 8192 + 1100, 8192, 64
    gen = torch.Generator(device="cuda").manual_seed(2)
    codes, scales = ck.quantize_experts_mxfp8(torch.randn(2, n, k, generator=gen, device="cuda"))
    ends, few = torch.tensor([rows - 300, rows], dtype=torch.int32, device="cuda"), torch.tensor([0, 300], dtype=torch.int32, device="cuda")
    x = _filled(rows, k, torch.bfloat16, 3)
    y = ck.grouped_linear_mxfp8(x, codes, scales, ends)
    assert torch.equal(y[-300:], ck.grouped_linear_mxfp8(x[-300:].clone(), codes, scales, few))
    assert torch.equal(y[0], y[rows - 301])
    dx = ck.grouped_input_grad_mxfp8(y, codes, scales, ends)
    alone = ck.grouped_input_grad_mxfp8(y[-300:].clone(), codes, scales, few)
    assert (dx[-300:].double() - alone.double()).norm() <= 2**-8 * alone.double().norm()  # another kernel, another order of additions: the last rounding
    assert torch.equal(dx[0], dx[rows - 301])


def test_large_weights(ck):
    """Codes of all experts past 2^32 bytes."""
    experts, n, k = 66, 8192, 8192
    gen = torch.Generator(device="cuda").manual_seed(4)
    codes = torch.full((experts, n, k), 0x28, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    scales = torch.full((experts, n, k // 32), 120, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)
    c, s = ck.quantize_mxfp8(torch.randn(n, k, generator=gen, device="cuda") * 0.02)
    codes[-1].copy_(c)
    scales[-1].view(torch.uint8).copy_(s.view(torch.uint8))
    for rows in (5, 700):
        x = torch.randn(rows, k, generator=gen, device="cuda").to(torch.bfloat16)
        ends = torch.zeros(experts, dtype=torch.int32, device="cuda")
        ends[-1] = rows
        one = torch.tensor([rows], dtype=torch.int32, device="cuda")
        y = ck.grouped_linear_mxfp8(x, codes, scales, ends)
        alone = ck.grouped_linear_mxfp8(x, c[None], s[None], one)
        assert (y.double() - alone.double()).norm() <= 2**-8 * alone.double().norm()
        dx, dx_alone = ck.grouped_input_grad_mxfp8(y, codes, scales, ends), ck.grouped_input_grad_mxfp8(y, c[None], s[None], one)
        assert (dx.double() - dx_alone.double()).norm() <= 2**-8 * dx_alone.double().norm()


def test_clip(ck):
    p = torch.nn.Parameter(torch.empty(2**32 + 4097, dtype=torch.bfloat16, device="cuda"))
    p.grad = torch.zeros_like(p)
    p.grad[-5:] = 3.0
    p.grad[0] = 4.0
    norm = ck.clip_grad_norm_([p], 1.0)
    want = 61**0.5
    assert abs(norm.item() - want) <= 1e-6 * want
    factor = torch.tensor(1.0, device="cuda") / (norm + 1e-6)
    assert (p.grad[-5:] == (3.0 * factor).to(torch.bfloat16)).all() and p.grad[0] == (4.0 * factor).to(torch.bfloat16) and (p.grad[1:1000] == 0).all()
