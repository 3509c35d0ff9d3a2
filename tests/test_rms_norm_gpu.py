"""RMS norm, its MXFP8 form and its gradients on the GPU, against the formulas in 64 bits.

Bounds.  u = 2^-24.  A row's sum of squares adds at most 32 terms in a thread (cols / 1024 in rows that no block holds), five levels of a warp and 32
warps: with the division, eps and the root's own two, rstd is off by (38 + 2 + cols / 2048) u at most.  y is three products behind it, one
of a factor that is itself a rounded sum; dx has rstd in three places, a sum over the row of as many terms and a few
products.  dweight adds the rows' terms in some order: less than one rounding for each.  Then one rounding to the result's type.
"""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0**-24
ROUND = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
TINY = {torch.float32: 2.0**-126, torch.float16: 2.0**-24, torch.bfloat16: 2.0**-126}
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def ck(cuda_device):
    import comfy_kitchen

    assert comfy_kitchen.list_backends()["cuda"]["available"]
    return comfy_kitchen


def _made(shape, dtype, seed, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _near(got, value, limit, name):
    limit = limit + ROUND[got.dtype] * (value.abs() + limit) + TINY[got.dtype]
    off = (got.double() - value).abs()
    assert got.shape == value.shape and torch.isfinite(got).all(), name
    assert (off <= limit).all(), f"{name}: {(off / limit).max().item():.3g} times the bound"


def _check(ck, x, weight, residual, offset, seed, eps=1e-6):
    """Forward and backward of one call."""
    rows, cols = x.numel() // x.shape[-1], x.shape[-1]
    e_r = (40 + cols / 2048) * U
    leaves = [t.detach().requires_grad_() for t in (x, weight, residual) if t is not None]
    call = iter(leaves)
    xl, wl, rl = next(call), next(call) if weight is not None else None, next(call) if residual is not None else None
    out = ck.rms_norm(xl, wl, rl, eps=eps, weight_offset=offset)
    y, h = out if residual is not None else (out, None)
    if residual is not None:
        assert torch.equal(h, (x.float() + residual.float()).to(x.dtype))
    v = (h if residual is not None else x).detach().double()
    rstd = (v.square().mean(-1, keepdim=True) + eps).rsqrt()
    f = torch.ones(cols, dtype=torch.float64, device="cuda") if weight is None else weight.double() + offset
    loose = f.abs() + (0 if weight is None else abs(offset) + weight.double().abs())
    _near(y, v * rstd * f, (v * rstd).abs() * loose * (e_r + 4 * U), "y")
    with torch.no_grad():
        again = ck.rms_norm(x, weight, residual, eps=eps, weight_offset=offset)
        assert torch.equal(again[0] if residual is not None else again, y)
        yf, hf, rf = ck.rms_norm_forward(x, weight, residual, eps=eps, weight_offset=offset)
        assert torch.equal(yf, y) and (hf is None) == (residual is None)
        assert ((rf.double() - rstd.reshape(-1)).abs() <= e_r * rstd.reshape(-1)).all()
    dy = _made(x.shape, x.dtype, seed + 50)
    dh = _made(x.shape, x.dtype, seed + 51) if residual is not None else None
    grads = iter(torch.autograd.grad(out, leaves, dy if residual is None else (dy, dh)))
    dx, dw, dr = next(grads), next(grads) if weight is not None else None, next(grads) if residual is not None else None
    d, un = dy.double(), v * rstd
    g = d * f
    size = (d.abs() * loose)
    along, size_along = (g * un).mean(-1, keepdim=True), (size * un.abs()).mean(-1, keepdim=True)
    value, magnitude = rstd * (g - un * along), rstd * (size + un.abs() * size_along)
    limit = (200 + cols / 256) * U * magnitude
    if dh is not None:
        value, limit = value + dh.double(), limit + 4 * U * dh.double().abs()
        assert torch.equal(dx, dr)
    _near(dx, value, limit, "dx")
    if weight is not None:
        assert dw.dtype == weight.dtype and dw.shape == weight.shape
        terms = (d * un).reshape(rows, cols)
        _near(dw, terms.sum(0), (rows + 240) * U * terms.abs().sum(0), "dw")
        if dw.dtype == torch.float32 and terms.sum(0).norm() > 0:
            assert (dw.double() - terms.sum(0)).norm() <= 2e-6 * terms.norm()


SIZES = [(1, 1), (1, 32), (3, 7), (2, 4096), (129, 128), (5, 769), (300, 1777), (70, 1024), (1000, 96), (33, 2050), (17, 8200), (4, 16384), (3, 16390),
         (2, 40000), (5000, 64), (2048, 520), (1, 100001)]


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", SIZES)
def test_norm(ck, dtype, rows, cols, residual):
    x = _made((rows, cols), dtype, 1)
    _check(ck, x, _made((cols,), dtype, 2), _made((rows, cols), dtype, 3, 2.0) if residual else None, 0.0, 4)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("weight_dtype,offset", [(None, 0.0), (torch.float32, 0.0), (torch.float32, 1.0), ("same", 1.0)])
@pytest.mark.parametrize("cols", [33, 256, 4096])
def test_weights(ck, dtype, weight_dtype, offset, cols):
    weight = None if weight_dtype is None else _made((cols,), dtype if weight_dtype == "same" else weight_dtype, 5, 0.2)
    _check(ck, _made((65, cols), dtype, 6), weight, _made((65, cols), dtype, 7), offset, 8)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_rows(ck, dtype):
    """Heads in the middle of a projection's result, a slice of tokens, rows that start anywhere, a dimension of size one."""
    for x in (_made((10, 3, 4, 128), dtype, 9)[:, 1], _made((3, 9, 64), dtype, 10)[:, 2:7], _made((20, 100), dtype, 11)[:, 3:90], _made((5, 1, 48), dtype, 12),
              _made((40, 256), dtype, 13)[::2], _made((7,), dtype, 14), _made((48, 6), dtype, 15).t(), _made((2, 3, 4, 5, 16), dtype, 16).transpose(1, 3)):
        _check(ck, x, _made((x.shape[-1],), dtype, 17), None, 0.0, 18)
        _check(ck, x, _made((x.shape[-1],), dtype, 17), _made(x.shape, dtype, 19), 0.0, 18)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 64), (130, 96), (128, 128), (1, 4096), (257, 1056), (7, 16384), (2, 65600)])
def test_mxfp8(ck, dtype, rows, cols):
    x, weight, residual = _made((rows, cols), dtype, 20), _made((cols,), dtype, 21), _made((rows, cols), dtype, 22, 3.0)
    x[rows // 2, :32] = 0
    want, want_scales = ck.quantize_mxfp8(ck.rms_norm(x, weight))
    codes, scales = ck.rms_norm_mxfp8(x, weight)
    assert torch.equal(codes.view(torch.uint8), want.view(torch.uint8)) and torch.equal(scales.view(torch.uint8), want_scales.view(torch.uint8))
    y, h = ck.rms_norm(x, weight, residual, weight_offset=1.0)
    want, want_scales = ck.quantize_mxfp8(y)
    codes, scales, got_h = ck.rms_norm_mxfp8(x, weight, residual, weight_offset=1.0)
    assert torch.equal(codes.view(torch.uint8), want.view(torch.uint8)) and torch.equal(scales.view(torch.uint8), want_scales.view(torch.uint8))
    assert torch.equal(got_h, h)


def test_mxfp8_of_a_slice(ck):
    x = _made((6, 5, 200), torch.bfloat16, 23)[:, 1:4, 8:72]
    weight = _made((70,), torch.bfloat16, 24)[3:67]
    codes, scales = ck.rms_norm_mxfp8(x, weight)
    want, want_scales = ck.quantize_mxfp8(ck.rms_norm(x, weight).reshape(18, 64))
    assert torch.equal(codes.view(torch.uint8), want.view(torch.uint8)) and torch.equal(scales.view(torch.uint8), want_scales.view(torch.uint8))


def test_gradient_against_differences(ck):
    """Central differences of the kernel's own fp32 forward pass along random directions."""
    x, w, r = _made((6, 40), torch.float32, 25), _made((40,), torch.float32, 26), _made((6, 40), torch.float32, 27)
    dy, dh = _made((6, 40), torch.float32, 28), _made((6, 40), torch.float32, 29)
    leaves = [t.requires_grad_() for t in (x, w, r)]
    grads = torch.autograd.grad(ck.rms_norm(*leaves), leaves, (dy, dh))
    step = 2.0**-7
    for i, g in enumerate(grads):
        direction = _made(g.shape, torch.float32, 30 + i)
        value = []
        for sign in (1, -1):
            moved = [t.detach() + (sign * step * direction if j == i else 0) for j, t in enumerate(leaves)]
            y, h = ck.rms_norm(*moved)
            value.append((y.double() * dy).sum() + (h.double() * dh).sum())
        slope, want = (value[0] - value[1]) / (2 * step), (g.double() * direction).sum()
        scale = (dy.abs().sum() + dh.abs().sum()).item()
        # third derivatives of order 10 times step^2 / 6, and roundings of 2^-22 of the terms over the step
        assert abs(slope - want) <= scale * (10 * step**2 / 6 + 2.0**-22 / step), (i, slope, want)


def test_partial_gradients(ck):
    x, w, r = _made((9, 64), torch.bfloat16, 31), _made((64,), torch.bfloat16, 32), _made((9, 64), torch.bfloat16, 33)
    dy, dh = _made((9, 64), torch.bfloat16, 34), _made((9, 64), torch.bfloat16, 35)
    leaves = [t.clone().requires_grad_() for t in (x, w, r)]
    y, h = ck.rms_norm(*leaves)
    full = torch.autograd.grad((y, h), leaves, (dy, dh), retain_graph=True)
    only_h = torch.autograd.grad(h, (leaves[0], leaves[2]), dh, retain_graph=True)
    assert torch.equal(only_h[0], dh) and torch.equal(only_h[1], dh)
    only_y = torch.autograd.grad(y, leaves, dy)
    with_zero = torch.autograd.grad(ck.rms_norm(*leaves), leaves, (dy, torch.zeros_like(dh)))
    assert all(torch.equal(a, b) for a, b in zip(only_y, with_zero)) and torch.equal(only_y[1], full[1])
    xl = x.clone().requires_grad_()
    y, h = ck.rms_norm(xl, w, r)
    (dx,) = torch.autograd.grad((y, h), xl, (dy, dh))
    assert torch.equal(dx, full[0])
    wl = w.clone().requires_grad_()
    (dw,) = torch.autograd.grad(ck.rms_norm(x, wl, r)[0], wl, dy)
    assert torch.equal(dw, full[1])


def test_the_dispatchers_route(ck):
    from torch.utils._python_dispatch import TorchDispatchMode

    class Watch(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.seen = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.seen.append(str(func))
            return func(*args, **(kwargs or {}))

    leaves = [_made(s, torch.float16, 36 + i).requires_grad_() for i, s in enumerate([(8, 96), (96,), (8, 96)])]
    d = (_made((8, 96), torch.float16, 39), _made((8, 96), torch.float16, 40))
    want = torch.autograd.grad(ck.rms_norm(*leaves), leaves, d)
    alone = torch.autograd.grad(ck.rms_norm(*leaves[:2]), leaves[:2], d[0])
    with Watch() as watch:
        got = torch.autograd.grad(ck.rms_norm(*leaves), leaves, d)
        got_alone = torch.autograd.grad(ck.rms_norm(*leaves[:2]), leaves[:2], d[0])
        codes = ck.rms_norm_mxfp8(*[t.detach() for t in leaves])
    assert any("rms_norm_forward" in s for s in watch.seen) and any("rms_norm_backward" in s for s in watch.seen)
    assert all(torch.equal(a, b) for a, b in zip(got + got_alone, want + alone))
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(codes, ck.rms_norm_mxfp8(*[t.detach() for t in leaves])))


def test_infinities_and_nan_stay_in_their_rows(ck):
    x = _made((5, 256), torch.bfloat16, 41)
    want = ck.rms_norm(x)
    x[1, 3], x[3, 200] = float("nan"), float("inf")
    got = ck.rms_norm(x)
    keep = [0, 2, 4]
    assert torch.equal(got[keep], want[keep]) and got[1].isnan().all()
    assert got[3, 200].isnan() and (got[3, :200] == 0).all()


def test_zero_rows_and_empty_tensors(ck):
    assert (ck.rms_norm(torch.zeros(4, 64, device="cuda", dtype=torch.bfloat16)) == 0).all()
    w = torch.ones(64, device="cuda", requires_grad=True)
    x = torch.zeros(0, 64, device="cuda", requires_grad=True)
    y = ck.rms_norm(x, w)
    assert y.shape == (0, 64)
    dx, dw = torch.autograd.grad(y, (x, w), torch.zeros(0, 64, device="cuda"))
    assert dx.shape == (0, 64) and (dw == 0).all()
    codes, scales = ck.rms_norm_mxfp8(torch.zeros(0, 64, device="cuda"))
    assert codes.shape == (0, 64) and scales.shape == (0, 4)


def test_captured_and_on_another_stream(ck):
    leaves = [_made(s, torch.bfloat16, 42 + i).requires_grad_() for i, s in enumerate([(300, 512), (512,), (300, 512)])]
    d = (_made((300, 512), torch.bfloat16, 45), _made((300, 512), torch.bfloat16, 46))
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        torch.autograd.grad(ck.rms_norm(*leaves), leaves, d)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ck.rms_norm(*leaves)
        grads = torch.autograd.grad(out, leaves, d)
    with torch.no_grad():
        leaves[0].copy_(_made((300, 512), torch.bfloat16, 47))
    graph.replay()
    want = ck.rms_norm(*leaves)
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    assert all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(want, leaves, d)))
    del graph, out, grads


def test_repeated_calls_give_the_same_bits(ck):
    leaves = [_made(s, torch.bfloat16, 48 + i).requires_grad_() for i, s in enumerate([(5000, 264), (264,)])]
    d = _made((5000, 264), torch.bfloat16, 50)
    first = torch.autograd.grad(ck.rms_norm(*leaves), leaves, d)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(ck.rms_norm(*leaves), leaves, d)))


def test_norm_feeds_the_linear_layers(ck):
    """A layer as it is used: norm into codes, a plain product and the experts' on the same operand."""
    x, w, r = _made((130, 128), torch.bfloat16, 51), _made((128,), torch.bfloat16, 52), _made((130, 128), torch.bfloat16, 53)
    codes, scales, h = ck.rms_norm_mxfp8(x, w, r)
    weights, weight_scales = ck.quantize_experts_mxfp8(_made((2, 64, 128), torch.bfloat16, 54, 0.1))
    ends = torch.tensor([70, 130], dtype=torch.int32).cuda()
    got = ck.grouped_mm_mxfp8(codes, weights, scales, weight_scales, ends)
    y = ck.rms_norm(x, w, r)[0]
    assert torch.equal(got, ck.grouped_linear_mxfp8(y, weights, weight_scales, ends))


def test_refusals(ck):
    x, w = torch.zeros(4, 64, device="cuda"), torch.ones(64, device="cuda")
    for bad in (lambda: ck.rms_norm(x, w[:32]), lambda: ck.rms_norm(x, w.half()), lambda: ck.rms_norm(x, w, x[:2]), lambda: ck.rms_norm(x, w, x.half()),
                lambda: ck.rms_norm(x.cpu()), lambda: ck.rms_norm(x.double()), lambda: ck.rms_norm(x, w.cpu()), lambda: ck.rms_norm(x, w, x.cpu()),
                lambda: ck.rms_norm(x[:, :0]), lambda: ck.rms_norm(torch.zeros((), device="cuda")), lambda: ck.rms_norm_mxfp8(x[:, :40]),
                lambda: ck.rms_norm_backward(x, x, torch.zeros(3, device="cuda")), lambda: ck.rms_norm_backward(x, x.half(), torch.zeros(4, device="cuda")),
                lambda: ck.rms_norm(x, w.view(1, 64))):
        with pytest.raises(Exception):
            bad()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols,start", [(30000, 32, 0), (20000, 64, 0), (9000, 128, 0), (2000, 1856, 3), (300, 6336, 8)])
def test_mxfp8_of_many_rows(ck, dtype, rows, cols, start):
    """Rows whose squares are added in another order than rms_norm's, so that a last bit may differ: values within the roundings to their type and to codes,
    scales the smallest powers of two that hold a block (or twice that where its largest value stands on the border)."""
    x = _made((rows, cols + start), dtype, 91)[:, start:]
    w = _made((cols,), torch.float32, 92)
    codes, scales = ck.rms_norm_mxfp8(x, w)
    value = x.double() * (x.double().square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w.double()
    off_by = (40 + cols / 2048 + 4) * U + ROUND[dtype]  # the norm and the products in fp32, the rounding to x's type
    blocks = value.abs().view(rows, -1, 32).amax(-1)
    held = ck.dequantize_mxfp8(codes, scales, torch.float32).double()
    r, c = torch.arange(rows, device="cuda").unsqueeze(1), torch.arange(cols // 32, device="cuda").unsqueeze(0)
    at = ((r // 128) * (scales.shape[1] // 4) + c // 4) * 512 + (r % 32) * 16 + (r // 32 % 4) * 4 + c % 4
    step = 2.0 ** (scales.view(torch.uint8).reshape(-1)[at].double() - 127)
    assert (step * 448 >= blocks * (1 - 2 * off_by)).all() and (step * 224 <= blocks * (1 + 2 * off_by)).all()
    # E4M3: half a step is 2^-4 of the value, or 2^-10 of the scale below 2^-6 of it
    limit = off_by * value.abs() + 2.0**-4 * value.abs() * (1 + off_by) + 2.0**-10 * step.repeat_interleave(32, 1)
    assert ((held - value).abs() <= limit).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_mxfp8_of_infinities_and_nan(ck, dtype):
    """As the quantizer has them, and only in their own rows."""
    x, w = _made((40, 256), dtype, 95), _made((256,), dtype, 96)
    clean = ck.rms_norm_mxfp8(x, w)
    x[3, 40], x[7, 200], x[20, 0] = float("inf"), float("nan"), float("-inf")
    w2 = w.clone()
    w2[100] = float("nan")
    for weight in (w, w2):
        codes, scales = ck.rms_norm_mxfp8(x, weight)
        want, want_scales = ck.quantize_mxfp8(ck.rms_norm(x, weight))
        assert torch.equal(codes.view(torch.uint8), want.view(torch.uint8)) and torch.equal(scales.view(torch.uint8), want_scales.view(torch.uint8))
    rest = [i for i in range(40) if i not in (3, 7, 20)]
    codes, scales = ck.rms_norm_mxfp8(x, w)
    assert torch.equal(codes.view(torch.uint8)[rest], clean[0].view(torch.uint8)[rest])
    linear = ck.dequantize_mxfp8(codes, scales, torch.float32)
    assert torch.equal(linear[rest], ck.dequantize_mxfp8(*clean, torch.float32)[rest])
