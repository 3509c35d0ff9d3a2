"""GELU with an MXFP8 copy of its input, on the GPU, against the definition in 64 bits.

Bounds.  u = 2^-24.  The exponent 2 z is off by 8 u |2 z|, its exponential by 8 u more, and the gate by no more than that relative to
itself; the slope's second factor |u 2 z'| by 8 u.  One rounding to the result's type.
"""
from __future__ import annotations

import math

import pytest
import torch
from gpu_util import bits

pytestmark = pytest.mark.gpu
U = 2.0**-24
ROUND = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
TINY = {torch.float32: 1e-27, torch.float16: 2.0**-24, torch.bfloat16: 1e-27}  # where the gate vanishes the kernel stops at 1e-28
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
ROOT = math.sqrt(2 / math.pi)


@pytest.fixture(scope="module")
def ck(cuda_device):
    import comfy_kitchen

    assert comfy_kitchen.list_backends()["cuda"]["available"]
    return comfy_kitchen


def _made(shape, dtype, seed, scale=2.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _definition(x, kept, dy):
    x, v, dy = x.double(), kept.double(), dy.double()
    z = lambda t: 2 * ROOT * (t + 0.044715 * t**3)  # noqa: E731
    y = x * torch.sigmoid(z(x))
    s, slope = torch.sigmoid(z(v)), 2 * ROOT * (1 + 3 * 0.044715 * v * v)
    second = v * slope * s * torch.sigmoid(-z(v))
    off = U * (16 + 16 * z(v).abs())
    return (y, y.abs() * U * (16 + 16 * z(x).abs())), (dy * (s + second), dy.abs() * (s * off + 3 * second.abs() * off))


def _check(got, want, name):
    value, bound = want
    limit = bound + ROUND[got.dtype] * (value.abs() + bound) + TINY[got.dtype]
    off = (got.double() - value).abs()
    assert got.shape == value.shape and torch.isfinite(got).all() and (off <= limit).all(), f"{name}: {(off / limit).max().item():.3g}"


def _run(ck, x, dy=None):
    leaf = x.detach().requires_grad_()
    y = ck.gelu_checkpointed(leaf)
    dy = _made(x.shape, x.dtype, 77, 1.0) if dy is None else dy
    (dx,) = torch.autograd.grad(y, leaf, dy)
    kept = ck.dequantize_mxfp8(*ck.quantize_mxfp8(x.detach().reshape(-1, x.shape[-1]).contiguous()), torch.float32).view(x.shape)
    want_y, want_dx = _definition(x.detach(), kept, dy)
    _check(y.detach(), want_y, "y")
    _check(dx, want_dx, "dx")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 32), (3, 96), (129, 160), (77, 4096), (1003, 2080), (5, 12288), (32,), (2, 3, 5, 64)])
def test_against_the_definition(ck, dtype, shape):
    _run(ck, _made(shape, dtype, 1))


@pytest.mark.parametrize("dtype", DTYPES)
def test_wide_range(ck, dtype):
    """Rows of one magnitude each, from where the cube vanishes to where the gate is 0 or 1."""
    x = _made((24, 64), dtype, 2, 1.0) * torch.logspace(-6, 4, 24, device="cuda").unsqueeze(1).to(dtype)
    _run(ck, x)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [32, 160, 4096])
def test_copy_is_the_quantizers(ck, dtype, cols):
    x = _made((133, cols), dtype, 3)
    x[0], x[1, :32] = 0, 0
    x[4, 5], x[5, 6] = float("inf"), float("nan")
    codes, scales = ck.quantize_mxfp8(x)
    _, got_codes, got_scales = ck.gelu_mxfp8_forward(x)
    assert (bits(got_codes) == bits(codes)).all() and (bits(got_scales) == bits(scales)).all()


def test_infinity_and_nan(ck):
    x = _made((4, 32), torch.float32, 4)
    x[0, 0], x[1, 1] = float("inf"), float("nan")
    leaf = x.requires_grad_()
    y = ck.gelu_checkpointed(leaf)
    (dx,) = torch.autograd.grad(y, leaf, torch.ones_like(y))
    assert y[0, 0] == float("inf") and torch.isnan(y[1, 1]) and torch.isfinite(y[2:]).all() and torch.isfinite(y[0, 1:]).all()
    assert dx[0, 0] == 1 and torch.isnan(dx[1, 1]) and torch.isfinite(dx[2:]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_alignment(ck, dtype):
    base = _made((20, 3, 97), dtype, 5)
    for x in (base[:, 1, 1:97], base[::2, :, :64], base.flatten()[1:1 + 32 * 60].view(60, 32), base[..., :96].transpose(0, 1)):
        _run(ck, x)
        _run(ck, x, torch.ones((), dtype=dtype, device="cuda").expand(x.shape))
        _run(ck, x, _made((*x.shape[:-1], 2 * x.shape[-1]), dtype, 6)[..., 1::2])


def test_empty(ck):
    x = torch.empty(0, 64, device="cuda", requires_grad=True)
    y = ck.gelu_checkpointed(x)
    (dx,) = torch.autograd.grad(y, x, torch.empty_like(y))
    assert y.shape == dx.shape == (0, 64)


def test_gradient_against_differences(ck):
    """Where the input is its own copy (one magnitude a block): step 2^-8, third derivative below 2, rounding of y 2^-22 / 2^-8."""
    x = torch.full((1, 32), 0.75, device="cuda")
    leaf = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(ck.gelu_checkpointed(leaf), leaf, torch.ones_like(x))
    step = 2.0**-8
    around = (ck.gelu_checkpointed(x + step) - ck.gelu_checkpointed(x - step)) / (2 * step)
    assert (around - dx).abs().max().item() <= 2e-4


def test_through_the_dispatcher_and_in_a_graph(ck):
    x = _made((40, 64), torch.bfloat16, 7).requires_grad_()
    dy = _made(x.shape, x.dtype, 8)
    (eager,) = torch.autograd.grad(ck.gelu_checkpointed(x), x, dy)
    (op,) = torch.autograd.grad(torch.ops.comfy_kitchen.gelu_mxfp8_forward(x)[0], x, dy)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, codes, scales = ck.gelu_mxfp8_forward(x.detach())
        dx = ck.gelu_mxfp8_backward(dy, codes, scales)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(eager, op) and torch.equal(eager, dx)


def test_refusals(ck):
    with pytest.raises(ValueError, match="multiple of 32"):
        ck.gelu_checkpointed(torch.zeros(4, 40, device="cuda"))
    with pytest.raises(ck.NoCapableBackendError):
        ck.gelu_checkpointed(torch.zeros(4, 64, device="cuda", dtype=torch.float64))
    with pytest.raises(ck.NoCapableBackendError):
        ck.gelu_checkpointed(torch.zeros(4, 64))
    x = torch.zeros(4, 64, device="cuda")
    _, codes, scales = ck.gelu_mxfp8_forward(x)
    with pytest.raises(AssertionError):
        ck.gelu_mxfp8_backward(x[:3], codes, scales)
    with pytest.raises(AssertionError):
        ck.gelu_mxfp8_backward(x, codes, scales[:64])
