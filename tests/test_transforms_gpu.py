"""The differentiable functions under torch.func and forward-mode differentiation: a transform gives what the plain calls give, or is refused."""
from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def functions(cuda_device):
    import comfy_kitchen as ck

    assert ck.list_backends()["cuda"]["available"]
    gen = torch.Generator(device="cuda").manual_seed(1)
    w = torch.randn(64, generator=gen, device="cuda")
    codes, scales = ck.quantize_experts_mxfp8(torch.randn(2, 32, 64, generator=gen, device="cuda"))
    ends = torch.tensor([2, 6], dtype=torch.int32, device="cuda")
    return {
        "rms_norm": lambda x: ck.rms_norm(x, w),
        "rms_norm with a residual": lambda x: ck.rms_norm(w.expand(6, 64), w, x)[0],
        "layer_norm": lambda x: ck.layer_norm(x, w, w),
        "gelu": ck.training.gelu_checkpointed,
        "grouped_linear": lambda x: ck.grouped_linear_mxfp8(x, codes, scales, ends),
    }


NAMES = ["rms_norm", "rms_norm with a residual", "layer_norm", "gelu", "grouped_linear"]


def _x(*shape):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")


@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_refused(functions, name):
    f, x = functions[name], _x(6, 64)
    want = f(x)
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            f(forward_ad.make_dual(x, x))
        assert torch.equal(f(x), want)  # no tangent of its own
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(f, (x,), (x,))


@pytest.mark.parametrize("name", NAMES)
def test_mapped_over_a_batch(functions, name):
    f, x = functions[name], _x(3, 6, 64)
    y = torch.func.vmap(f)(x)
    assert torch.equal(y, torch.stack([f(v) for v in x]))
