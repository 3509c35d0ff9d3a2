"""Calls that begin with a tensor map, made on a thread that has not used the GPU before (as gradients are, on the autograd engine's)."""
from __future__ import annotations

import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", ["linear", "grouped", "scaled_mm"])
def test_first_call(cuda_device, which):
    import comfy_kitchen as ck

    w, dy, x = torch.randn(64, 96, device="cuda"), torch.randn(8, 64, device="cuda").bfloat16(), torch.randn(8, 96, device="cuda")
    codes, scales = ck.quantize_mxfp8(w)
    x_codes, x_scales = ck.quantize_mxfp8(x)
    ends = torch.tensor([8], dtype=torch.int32, device="cuda")
    calls = {"linear": lambda: ck.linear_input_grad_mxfp8(dy, codes, scales),
             "grouped": lambda: ck.grouped_input_grad_mxfp8(dy, codes[None], scales[None], ends),
             "scaled_mm": lambda: ck.scaled_mm_mxfp8(x_codes, codes, x_scales, scales)}
    want, got, errors = calls[which](), [], []
    torch.cuda.synchronize()

    def run():
        try:
            got.append(calls[which]())
        except Exception as e:  # noqa: BLE001 - told to the test's thread
            errors.append(e)

    thread = threading.Thread(target=run)
    thread.start()
    thread.join(60)
    torch.cuda.synchronize()
    assert not errors and torch.equal(got[0], want)
