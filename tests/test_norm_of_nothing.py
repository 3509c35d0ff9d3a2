"""The gradients' norm where there are no gradients: a float32 zero where the parameters are, whatever torch's defaults say."""
from __future__ import annotations

import pytest
import torch

import comfy_kitchen as ck


@pytest.fixture(params=[torch.float32, torch.float64])
def default_dtype(request):
    before = torch.get_default_dtype()
    torch.set_default_dtype(request.param)
    yield
    torch.set_default_dtype(before)


def _check(norm, device):
    assert norm.shape == () and norm.dtype == torch.float32 and norm.device.type == device and norm.item() == 0.0


def test_on_the_cpu(default_dtype):
    _check(ck.grad_norm([]), "cpu")
    _check(ck.clip_grad_norm_([], 1.0), "cpu")
    _check(ck.clip_grad_norm_(torch.nn.Linear(3, 3).parameters(), 1.0), "cpu")
    assert ck.clip_grad_norm_(torch.nn.Linear(3, 3, device="meta").parameters(), 1.0, error_if_nonfinite=True).is_meta


@pytest.mark.gpu
def test_on_the_gpu(cuda_device, default_dtype):
    p = torch.nn.Parameter(torch.zeros(3, device=cuda_device))
    _check(ck.clip_grad_norm_([p], 1.0), "cuda")
    _check(ck.clip_grad_norm_(p, 1.0, error_if_nonfinite=True), "cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = ck.clip_grad_norm_([p], 1.0)
    graph.replay()
    _check(norm, "cuda")
    del graph
