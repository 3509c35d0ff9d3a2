"""The few-row gradients where their MMAs keep shared memory busy: a place of the codes' ring is given back while reads of it may still be held up, and
what the next copy writes there must not reach them.  The result is the same in every pass, bit for bit."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
PARTS = {torch.float32: 3, torch.float16: 2, torch.bfloat16: 1}


def _made(shape, dtype, seed, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


@pytest.mark.parametrize("grouped", [True, False])
@pytest.mark.parametrize("dtype,rows,n,k", [
    (torch.bfloat16, 200, 4864, 8192), (torch.bfloat16, 224, 1544, 8192), (torch.bfloat16, 200, 4864, 128), (torch.float16, 200, 4864, 8192), (torch.float16, 96, 4864, 8192),
    (torch.float32, 200, 4864, 4096), (torch.float32, 40, 4864, 8192)])
def test_every_pass_alike(cuda_device, dtype, rows, n, k, grouped):
    import comfy_kitchen as ck

    dy = _made((rows, n), dtype, 4)
    codes, scales = ck.quantize_experts_mxfp8(_made((1, n, k), torch.bfloat16, 5, 0.05))
    ends = torch.tensor([rows], dtype=torch.int32, device="cuda")

    def grad():
        if grouped:
            return ck.grouped_input_grad_mxfp8(dy, codes, scales, ends, out_dtype=torch.float32)
        return ck.linear_input_grad_mxfp8(dy, codes[0], scales[0], out_dtype=torch.float32)

    first = grad()
    w = ck.dequantize_mxfp8(codes[0], scales[0], torch.float32).double()
    # exact products, fp32 additions of 16 at once at most (for each bf16 part of dY), each off by 2^-22 of the running sum of magnitudes
    limit = ((n / 16 * PARTS[dtype] + 4) * 2.0**-22 + 2.0**-24) * (dy.double().abs() @ w.abs())
    assert ((first.double() - dy.double() @ w).abs() <= limit).all()
    differ = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(200):
        differ += (grad() != first).any()
    assert differ.item() == 0, f"{differ.item()} of 200 passes"
