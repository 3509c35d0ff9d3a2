"""Hooks on the tensors that the native autograd nodes save: identity, offloading, non-reentrant checkpointing (which ends its recomputation by an
exception out of a hook), and hooks that raise."""
from __future__ import annotations

import pytest
import torch
from torch.utils.checkpoint import checkpoint

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ck(cuda_device):
    import comfy_kitchen

    assert comfy_kitchen.list_backends()["cuda"]["available"]
    return comfy_kitchen


def _x():
    gen = torch.Generator(device="cuda").manual_seed(1)
    return torch.randn(6, 64, generator=gen, device="cuda").requires_grad_()


def _functions(ck):
    w = torch.linspace(0.5, 1.5, 64, device="cuda")
    codes, scales = ck.quantize_experts_mxfp8(torch.eye(64, device="cuda").repeat(2, 1, 1))
    ends = torch.tensor([2, 6], dtype=torch.int32, device="cuda")
    return {
        "rms_norm": lambda x: ck.rms_norm(x, w),
        "rms_norm with a residual": lambda x: sum(ck.rms_norm(x, w, x.detach() * 2)),
        "layer_norm": lambda x: ck.layer_norm(x, w, w),
        "layer_norm with a copy": lambda x: ck.layer_norm(x, w, w, checkpoint=True),
        "gelu": ck.training.gelu_checkpointed,
        "grouped_linear": lambda x: ck.grouped_linear_mxfp8(x, codes, scales, ends),
        "all": lambda x: ck.training.gelu_checkpointed(ck.grouped_linear_mxfp8(ck.rms_norm(ck.layer_norm(x, w, w), w), codes, scales, ends)),
    }


NAMES = ["rms_norm", "rms_norm with a residual", "layer_norm", "layer_norm with a copy", "gelu", "grouped_linear", "all"]


def _grad(y, x):
    return torch.autograd.grad((y * torch.linspace(-1, 1, 64, device="cuda")).sum(), x)[0]


def _checkpointed(f, reentrant):
    x = _x()
    (checkpoint(f, x, use_reentrant=reentrant) * torch.linspace(-1, 1, 64, device="cuda")).sum().backward()
    return x.grad


@pytest.mark.parametrize("name", NAMES)
def test_the_same_gradient(ck, name):
    f, x = _functions(ck)[name], _x()
    want = _grad(f(x), x)
    for reentrant in (False, True):
        assert torch.equal(_checkpointed(f, reentrant), want)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t):
        y = f(x)
    assert torch.equal(_grad(y, x), want)
    with torch.autograd.graph.save_on_cpu():
        y = f(x)
    assert torch.equal(_grad(y, x), want)


@pytest.mark.parametrize("name", NAMES)
def test_a_hook_that_raises(ck, name):
    f, x = _functions(ck)[name], _x()
    want = _grad(f(x), x)

    def refuse(_):
        raise LookupError("not kept")

    with torch.autograd.graph.saved_tensors_hooks(refuse, lambda t: t), pytest.raises(LookupError, match="not kept"):
        f(x)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, refuse):
        y = f(x)
        with pytest.raises(LookupError, match="not kept"):
            _grad(y, x)
    assert torch.equal(_grad(f(x), x), want)
