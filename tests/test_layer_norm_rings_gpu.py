"""Layer norm over many rows, which come through rings in shared memory: against the definition in 64 bits, with the bounds of test_layer_norm_gpu.py."""
from __future__ import annotations

import pytest
import torch
from test_layer_norm_gpu import DTYPES, _made, _run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ck(cuda_device):
    import comfy_kitchen

    assert comfy_kitchen.list_backends()["cuda"]["available"]
    return comfy_kitchen


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols,pitch", [(9000, 1001, 1001), (9001, 770, 773), (6000, 1601, 1607), (4000, 3070, 3071)])
def test_a_stage_whose_rows_lie_otherwise_in_their_16_bytes(ck, dtype, rows, cols, pitch):
    """Many rows one after another in each stage, every one with another offset: what one row brings by plain stores the next one's bulk copy
    brings, and the other way round.  First and last elements stand out, so that a stale one would show."""
    def made(seed):
        t = _made((rows, pitch), dtype, seed)[:, :cols]
        t[:, :8] *= 30 * (1 - 2 * (torch.arange(rows, device="cuda") % 2)).to(dtype).unsqueeze(1)
        t[:, -8:] *= 20
        return t

    x, dy = made(1), made(2)
    w, b = _made((cols,), dtype, 3, 0.2, 1.0), _made((cols,), dtype, 4, 0.2)
    _run(ck, x, w, b, dy=dy)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    first, second = ([y, *torch.autograd.grad(y, leaves, dy)] for y in (ck.layer_norm(*leaves), ck.layer_norm(*leaves)))
    assert all(torch.equal(p, q) for p, q in zip(first, second))
