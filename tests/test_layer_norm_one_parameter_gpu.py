"""One tensor as the layer norm's weight and bias."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("checkpoint", [False, True])
@pytest.mark.parametrize("shape,param", [((6, 64), (64,)), ((2, 3, 96), (96,)), ((3, 5, 64), (3, 64))])
def test_weight_and_bias_alike(cuda_device, shape, param, checkpoint):
    """Against a copy in the bias's place, which takes the same kernels: equal but for the two gradients' sum, one fp32 rounding."""
    import comfy_kitchen as ck

    gen = torch.Generator(device="cuda").manual_seed(1)
    x, w, dy = (torch.randn(s, generator=gen, device="cuda") for s in (shape, param, shape))
    with torch.no_grad():
        assert torch.equal(ck.layer_norm(x, w, w), ck.layer_norm(x, w, w.clone()))
    x1, w1, x2, w2, b2 = (t.clone().requires_grad_() for t in (x, w, x, w, w))
    y1, y2 = ck.layer_norm(x1, w1, w1, checkpoint=checkpoint), ck.layer_norm(x2, w2, b2, checkpoint=checkpoint)
    assert torch.equal(y1, y2)
    dx1, dw1 = torch.autograd.grad(y1, (x1, w1), dy)
    dx2, dw2, db2 = torch.autograd.grad(y2, (x2, w2, b2), dy)
    assert torch.equal(dx1, dx2) and torch.equal(dw1, dw2 + db2)
    normalized = torch.nn.functional.layer_norm(x.double(), shape[-1:])
    rows = w.double() if len(param) == 1 else w.double().unsqueeze(1)
    # fp32 statistics of rows of a hundred, a few operations: some units of 2^-24 of the magnitudes
    assert ((y1.double() - (normalized * rows + rows)).abs() <= 64 * 2.0**-24 * (normalized.abs() + 1) * (rows.abs() + 1)).all()
