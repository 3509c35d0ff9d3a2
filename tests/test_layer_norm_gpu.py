"""Layer norm on the GPU against its definition in 64 bits: results, gradients, the MXFP8 copy, strides, groups, odd sizes.

Bounds.  u = 2^-24.  A row's sums add at most 64 terms in a thread one after another and 2^5 * 32 partial sums in trees and short loops:
an error of at most 128 u times the sum of magnitudes, so the mean is off by 128 u mean|x| and 1/std by 128 u of itself at most.
Column sums add at most all rows of a group one after another.  Results are rounded to their type once.
"""
from __future__ import annotations

import pytest
import torch
from gpu_util import bits

pytestmark = pytest.mark.gpu
U = 2.0**-24
ROUND = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
TINY = {torch.float32: 2.0**-149, torch.float16: 2.0**-24, torch.bfloat16: 2.0**-133}
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def ck(cuda_device):
    import comfy_kitchen

    assert comfy_kitchen.list_backends()["cuda"]["available"]
    return comfy_kitchen


def _made(shape, dtype, seed, scale=1.0, shift=0.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=gen, device="cuda") * scale + shift).to(dtype)


def _definition(x, weight, bias, eps, offset, dy=None, kept=None):
    """{name: (value, bound of the fp32 arithmetic)} in 64 bits; `kept`: the values that the backward pass reads in x's place."""
    x = x.double()
    cols = x.shape[-1]
    mean, var = x.mean(-1, keepdim=True), x.var(-1, correction=0, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    shape = (-1, *[1] * (x.dim() - 2), cols) if x.dim() > 1 else (cols,)
    f = torch.ones((), dtype=torch.float64, device=x.device) if weight is None else (offset + weight.double()).reshape(shape if weight.dim() > 1 else (cols,))
    b = torch.zeros((), dtype=torch.float64, device=x.device) if bias is None else bias.double().reshape(shape if bias.dim() > 1 else (cols,))
    f, b = f.expand(x.shape), b.expand(x.shape)
    off_h = lambda v: 128 * U * ((v - mean).abs() * rstd + x.abs().mean(-1, keepdim=True) * rstd) + 4 * U * v.abs() * rstd  # noqa: E731
    h = (x - mean) * rstd
    got = {"y": (h * f + b, off_h(x) * f.abs() + 4 * U * (h * f).abs() + 4 * U * b.abs())}
    if dy is None:
        return got
    v = x if kept is None else kept.double()
    h, dh = (v - mean) * rstd, off_h(v)
    dy = dy.double()
    g = dy * f
    c2 = (g * h).mean(-1, keepdim=True)
    off_c1 = 128 * U * g.abs().mean(-1, keepdim=True)
    off_c2 = (g.abs() * (dh + 128 * U * h.abs())).mean(-1, keepdim=True)
    dx = rstd * (g - g.mean(-1, keepdim=True) - h * c2)
    got["dx"] = (dx, rstd * (8 * U * (g.abs() + (h * c2).abs()) + off_c1 + h.abs() * off_c2 + dh * c2.abs()) + 256 * U * dx.abs())
    some = weight if weight is not None else bias
    if some is not None:
        dims = tuple(range(1, x.dim() - 1)) if some.dim() > 1 else tuple(range(x.dim() - 1))
        add = lambda t: t.sum(dims).reshape(some.shape) if dims else t.reshape(some.shape)  # noqa: E731
        terms = x.numel() // some.numel() + 64
        got["dw"] = (add(dy * h), add(dy.abs() * dh) + terms * U * add((dy * h).abs()))
        got["db"] = (add(dy), terms * U * add(dy.abs()))
    return got


def _check(got, want, name):
    value, bound = want
    assert got.shape == value.shape, name
    limit = bound + ROUND[got.dtype] * (value.abs() + bound) + TINY[got.dtype]
    off = (got.double() - value).abs()
    assert torch.isfinite(got).all(), name
    assert (off <= limit).all(), f"{name}: {(off / limit).max().item():.3g} times the bound"


def _run(ck, x, weight, bias, offset=0.0, checkpoint=False, eps=1e-5, dy=None):
    x, weight, bias = (None if t is None else t.detach().requires_grad_() for t in (x, weight, bias))
    y = ck.layer_norm(x, weight, bias, eps, offset, checkpoint)
    dy = _made(y.shape, y.dtype, 99) if dy is None else dy
    leaves = [t for t in (x, weight, bias) if t is not None]
    grads = torch.autograd.grad(y, leaves, dy)
    kept = None
    if checkpoint:
        flat = x.detach().reshape(-1, x.shape[-1]).contiguous()
        kept = ck.dequantize_mxfp8(*ck.quantize_mxfp8(flat), torch.float32).view(x.shape)
    want = _definition(x.detach(), None if weight is None else weight.detach(), None if bias is None else bias.detach(), eps, offset, dy, kept)
    _check(y.detach(), want["y"], "y")
    _check(grads[0], want["dx"], "dx")
    if weight is not None:
        assert grads[1].dtype == weight.dtype
        _check(grads[1], want["dw"], "dw")
    if bias is not None:
        _check(grads[-1], want["db"], "db")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 3072), (3, 7), (5, 33), (2, 256), (129, 512), (77, 769), (300, 1152), (1003, 1000), (64, 3072),
                                       (9, 5120), (33, 8192), (17, 12288), (5, 16384), (3, 9001), (2, 70000)])
def test_affine(ck, dtype, rows, cols):
    x = _made((rows, cols), dtype, 1, 2.0, 0.3)
    _run(ck, x, _made((cols,), dtype, 2, 0.2, 1.0), _made((cols,), dtype, 3, 0.2))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(2000, 1), (2000, 7), (1500, 33), (700, 129), (700, 130), (600, 257), (600, 1001), (500, 3070), (400, 5001), (350, 9754),
                                       (310, 12287), (300, 12290), (300, 16383)])
def test_many_rows_off_vectors(ck, dtype, rows, cols):
    """Rows that do not lie on 16-byte boundaries, in every place of 16 bytes, from one to many of them a team."""
    x = _made((rows, cols), dtype, 50, 2.0, 0.3)
    _run(ck, x, _made((cols,), dtype, 51, 0.2, 1.0), _made((cols,), dtype, 52, 0.2))
    if cols > 8:
        wide = _made((rows, cols + 3), dtype, 53)
        _run(ck, wide[:, 1:cols + 1], _made((cols,), torch.float32, 54, 0.2, 1.0), None, dy=_made((rows, cols + 5), dtype, 55)[:, 2:cols + 2])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 32), (5, 96), (129, 512), (1003, 1024), (64, 3072), (300, 4096), (17, 12288), (4, 16384), (2, 32768)])
def test_from_the_mxfp8_copy(ck, dtype, rows, cols):
    x = _made((rows, cols), dtype, 4, 2.0, 0.3)
    _run(ck, x, _made((cols,), dtype, 5, 0.2, 1.0), _made((cols,), dtype, 6, 0.2), checkpoint=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [32, 160, 3072, 12288])
def test_copy_is_the_quantizers(ck, dtype, cols):
    """Codes and scales are the quantizer's bit for bit: zeros, huge and tiny blocks, infinities and NaN among them, padding too."""
    x = _made((133, cols), dtype, 7)
    x[0] = 0
    x[1, :32] = 0
    x[2] *= 1e4
    x[3] *= 1e-6
    x[4, 5] = float("inf")
    x[5, 6] = float("nan")
    codes, scales = ck.quantize_mxfp8(x)
    _, _, _, got_codes, got_scales = ck.layer_norm_forward_mxfp8(x)
    assert (bits(got_codes) == bits(codes)).all() and (bits(got_scales) == bits(scales)).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("checkpoint", [False, True])
def test_full_precision_parameters(ck, dtype, checkpoint):
    x = _made((150, 1536), dtype, 8)
    _run(ck, x, _made((1536,), torch.float32, 9, 0.2, 1.0), _made((1536,), torch.float32, 10), checkpoint=checkpoint)


@pytest.mark.parametrize("weight,bias", [(True, False), (False, True), (False, False)])
@pytest.mark.parametrize("checkpoint", [False, True])
def test_without_parameters(ck, weight, bias, checkpoint):
    x = _made((70, 640), torch.bfloat16, 11)
    _run(ck, x, _made((640,), x.dtype, 12) if weight else None, _made((640,), x.dtype, 13) if bias else None, 0.5, checkpoint)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("checkpoint", [False, True])
@pytest.mark.parametrize("groups,tokens,cols", [(1, 200, 256), (3, 1, 96), (8, 37, 1024), (200, 3, 64), (2, 700, 3072)])
def test_modulation(ck, dtype, checkpoint, groups, tokens, cols):
    """A scale and a shift for each sample: chunks of one projection's result."""
    x = _made((groups, tokens, cols), dtype, 14)
    mod = _made((groups, 6 * cols), dtype, 15, 0.3).chunk(6, dim=-1)
    _run(ck, x, mod[1], mod[0], 1.0, checkpoint)
    _run(ck, x, mod[1].unsqueeze(1), mod[0].unsqueeze(1), 1.0, checkpoint)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("checkpoint", [False, True])
def test_strided_rows(ck, dtype, checkpoint):
    """Slices, transposed dimensions, a misaligned start, a stride of zero, gradients that are expanded or strided."""
    w, b = _made((96,), dtype, 16), _made((96,), dtype, 17)
    base = _made((4, 50, 3 * 96), dtype, 18)
    for x in (base[:, 3:40, :96], base[1:3, ::2, 96:192], base[0, :, 192:], base.transpose(0, 1)[5:, :, 96:192], base[:, :, 1:97],
              base[:, :1, :96].expand(4, 6, 96), base[..., ::3]):
        _run(ck, x, w, b, checkpoint=checkpoint)
        _run(ck, x, w, b, checkpoint=checkpoint, dy=_made((1, 96), dtype, 19).expand(x.shape))
        _run(ck, x, w, b, checkpoint=checkpoint, dy=torch.ones((), dtype=dtype, device="cuda").expand(x.shape))
        _run(ck, x, w, b, checkpoint=checkpoint, dy=_made((*x.shape[:-1], 2 * 96), dtype, 20)[..., 96:])


@pytest.mark.parametrize("shape", [(64,), (2, 3, 4, 64), (0, 64), (3, 0, 64)])
@pytest.mark.parametrize("checkpoint", [False, True])
def test_ranks_and_empty(ck, shape, checkpoint):
    x = _made(shape, torch.bfloat16, 21).requires_grad_()
    w, b = _made((64,), x.dtype, 22).requires_grad_(), _made((64,), x.dtype, 23).requires_grad_()
    if x.numel():
        return _run(ck, x.detach(), w.detach(), b.detach(), checkpoint=checkpoint)
    y = ck.layer_norm(x, w, b, checkpoint=checkpoint)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
    assert y.shape == dx.shape == x.shape and (dw == 0).all() and (db == 0).all()


def test_a_large_mean_and_a_constant_row(ck):
    x = _made((40, 3072), torch.float32, 24, 0.01, 100.0)
    x[3] = 7.0
    _run(ck, x, _made((3072,), torch.float32, 25), _made((3072,), torch.float32, 26))


@pytest.mark.parametrize("checkpoint", [False, True])
def test_nan_and_infinity_stay_in_their_rows(ck, checkpoint):
    x = _made((20, 256), torch.bfloat16, 27)
    clean = x.clone()
    x[4, 9], x[11, 0] = float("nan"), float("inf")
    y = ck.layer_norm(x, checkpoint=checkpoint)
    rows = torch.tensor([r for r in range(20) if r not in (4, 11)], device="cuda")
    assert torch.isnan(y[4]).all() and torch.isnan(y[11]).all()
    assert torch.equal(y[rows], ck.layer_norm(clean)[rows])


def test_some_gradients_only(ck):
    x, w, b = _made((33, 128), torch.bfloat16, 28), _made((128,), torch.bfloat16, 29), _made((128,), torch.bfloat16, 30)
    dy = _made(x.shape, x.dtype, 31)

    def grads(which):
        leaves = [t.detach().requires_grad_(i in which) for i, t in enumerate((x, w, b))]
        return dict(zip(which, torch.autograd.grad(ck.layer_norm(*leaves), [leaves[i] for i in which], dy)))

    whole = grads((0, 1, 2))
    for which in ((0,), (1,), (2,), (0, 1), (1, 2)):
        for i, g in grads(which).items():
            assert torch.equal(g, whole[i])


def test_same_bits_again_and_in_a_graph(ck):
    """Sums are added in a fixed order, also on another stream than the default one and in a captured call."""
    x, w, b = _made((2000, 1024), torch.bfloat16, 32), _made((1024,), torch.float32, 33), _made((1024,), torch.float32, 34)
    dy = _made(x.shape, x.dtype, 35)

    def step():
        y, mean, rstd = ck.layer_norm_forward(x, w, b)
        return (y, *ck.layer_norm_backward(dy, x, mean, rstd, w))

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        third = step()
    graph.replay()
    torch.cuda.synchronize()
    for a, b_, c in zip(first, second, third):
        assert torch.equal(a, b_) and torch.equal(a, c)


def test_gradient_against_differences(ck):
    """Central differences of the forward pass in fp32, step 2^-6: truncation 2^-12/6 of a third derivative of order 10, rounding of y
    128 u / 2^-6 of a sum of 96 terms."""
    x, w, b = _made((3, 96), torch.float32, 36), _made((96,), torch.float32, 37), _made((96,), torch.float32, 38)
    dy = _made(x.shape, x.dtype, 39)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(ck.layer_norm(*leaves), leaves, dy)
    step = 2.0**-6
    for i, at in ((0, (1, 5)), (0, (2, 95)), (1, (7,)), (2, (50,))):
        sides = []
        for sign in (1, -1):
            moved = [t.detach().clone() for t in (x, w, b)]
            moved[i][at] += sign * step
            sides.append((ck.layer_norm(*moved).double() * dy.double()).sum().item())
        assert abs((sides[0] - sides[1]) / (2 * step) - grads[i][at].item()) <= 5e-3


@pytest.mark.parametrize("checkpoint", [False, True])
def test_through_the_dispatcher(ck, checkpoint):
    """Traced calls take the operators' own gradients: the same bits as the eager call's."""
    x, w, b = (t.requires_grad_() for t in (_made((4, 9, 64), torch.bfloat16, 40), _made((4, 64), torch.bfloat16, 41), _made((4, 64), torch.bfloat16, 42)))
    dy = _made(x.shape, x.dtype, 43)
    eager = torch.autograd.grad(ck.layer_norm(x, w, b, weight_offset=1.0, checkpoint=checkpoint), (x, w, b), dy)
    op = torch.ops.comfy_kitchen.layer_norm_forward_mxfp8 if checkpoint else torch.ops.comfy_kitchen.layer_norm_forward
    out = op(x, w, b, 1e-5, 1.0)
    for a, g in zip(eager, torch.autograd.grad(out[0], (x, w, b), dy)):
        assert torch.equal(a, g)
    with torch.profiler.profile(activities=[torch.profiler.ProfilerActivity.CPU]):
        watched = torch.autograd.grad(ck.layer_norm(x, w, b, weight_offset=1.0, checkpoint=checkpoint), (x, w, b), dy)
    assert all(torch.equal(a, g) for a, g in zip(eager, watched))


def test_refusals(ck):
    x = _made((4, 64), torch.bfloat16, 44)
    w = _made((64,), torch.bfloat16, 45)
    with pytest.raises(ValueError, match="multiple of 32"):
        ck.layer_norm(x[:, :40], checkpoint=True)
    with pytest.raises(ck.NoCapableBackendError):
        ck.layer_norm(x.double())
    with pytest.raises(ck.NoCapableBackendError):
        ck.layer_norm(x.cpu())
    for bad_w, bad_b in ((w[:32], None), (w, w[:32]), (w, w.float()), (w.expand(3, 64), None), (w.half(), None), (w.cpu(), None)):
        with pytest.raises((AssertionError, RuntimeError, ck.NoCapableBackendError)):
            ck.layer_norm(x, bad_w, bad_b)
    _, mean, rstd = ck.layer_norm_forward(x, w)
    with pytest.raises(AssertionError):
        ck.layer_norm_backward(x, x[:, :32], mean, rstd, w)
    with pytest.raises(AssertionError):
        ck.layer_norm_backward(x, x, mean[:2], rstd, w)
    with pytest.raises(RuntimeError):  # no gradients of gradients
        leaf = x.detach().requires_grad_()
        (g,) = torch.autograd.grad(ck.layer_norm(leaf), leaf, x, create_graph=True)
        g.sum().backward()


@pytest.mark.parametrize("cols", [2_097_120, 2_097_128, 2_200_000])
def test_gradients_of_very_wide_rows(ck, monkeypatch, cols):
    """More strips of 32 columns than a grid's second dimension counts.  A thread of 512 adds its columns one after another: the bounds grow as those do."""
    monkeypatch.setitem(globals(), "U", U * (cols / 512 + 64) / 128)
    x = _made((2, cols), torch.bfloat16, 46)
    _run(ck, x, _made((cols,), torch.bfloat16, 47, 0.2, 1.0), _made((cols,), torch.bfloat16, 48))
