"""Gradients of a linear layer from MXFP8 matrices, on the GPU, against the definition in 64 bits.

Bounds.  Operands are exact (an E4M3 number times a power of two in bf16, dY as one to three bf16 numbers), the accumulation is fp32: one
addition for 16 contraction steps and bf16 part of dY, each at most 2^-22 of the running sum of magnitudes, and 64 additions of splits.
One rounding to the result's type.
"""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
ROUND = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
TINY = {torch.float32: 2.0**-126, torch.float16: 2.0**-24, torch.bfloat16: 2.0**-126}
PARTS = {torch.float32: 3, torch.float16: 2, torch.bfloat16: 1}
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def ck(cuda_device):
    import comfy_kitchen

    assert comfy_kitchen.list_backends()["cuda"]["available"]
    return comfy_kitchen


def _made(shape, dtype, seed, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _held(ck, rows, cols, seed, scale=1.0):
    codes, scales = ck.quantize_mxfp8(_made((rows, cols), torch.float32, seed, scale))
    return codes, scales, ck.dequantize_mxfp8(codes, scales, torch.float32).double()


def _check(got, left, right, parts, name):
    """got against left @ right"""
    value, magnitude = left @ right, left.abs() @ right.abs()
    limit = (left.shape[1] / 16 * parts + 64) * 2.0**-22 * magnitude
    limit = limit + ROUND[got.dtype] * (value.abs() + limit) + TINY[got.dtype]
    off = (got.double() - value).abs()
    assert got.shape == value.shape and torch.isfinite(got).all(), name
    assert (off <= limit).all(), f"{name}: {(off / limit).max().item():.3g} times the bound"
    if got.dtype == torch.float32 and value.norm() > 0:
        assert off.norm() <= 1e-5 * value.norm(), f"{name}: {(off.norm() / value.norm()).item():.3g}"


def _weight(ck, m, n, k, dtype, out, bias=True):
    dy = _made((m, n), dtype, 1)
    codes, scales, x = _held(ck, m, k, 2)
    dw, db = ck.linear_weight_grad_mxfp8(dy, codes, scales, out_dtype=out, bias_grad=bias)
    assert dw.dtype == (out or dtype)
    _check(dw, dy.double().t(), x, PARTS[dtype], "dw")
    if bias:
        _check(db.unsqueeze(0), torch.ones(1, m, dtype=torch.float64, device="cuda"), dy.double(), 16, "db")
    else:
        assert db is None


def _input(ck, m, n, k, dtype, out=None):
    dy = _made((m, n), dtype, 3)
    codes, scales, w = _held(ck, n, k, 4, 0.02)
    dx = ck.linear_input_grad_mxfp8(dy, codes, scales, out_dtype=out)
    assert dx.dtype == (out or dtype)
    _check(dx, dy.double(), w, PARTS[dtype], "dx")


SIZES = [(1, 8, 32), (3, 16, 64), (64, 256, 256), (65, 264, 288), (127, 1000, 96), (300, 520, 544), (1000, 768, 1056), (2049, 384, 320), (4096, 256, 256)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_weight(ck, dtype, m, n, k):
    _weight(ck, m, n, k, dtype, None)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", SIZES + [(2, 3000, 512), (8, 4096, 1024), (16, 1024, 2048), (40, 2048, 32), (128, 2048, 2048), (16, 12288, 128),
                                           (72, 12288, 256), (128, 12288, 384), (200, 12288, 128), (208, 6000, 256), (209, 6000, 256)])
def test_input(ck, dtype, m, n, k):
    _input(ck, m, n, k, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("out", DTYPES)
def test_result_types(ck, dtype, out):
    _weight(ck, 200, 264, 288, dtype, out)
    _input(ck, 200, 264, 288, dtype, out)
    _input(ck, 5, 264, 288, dtype, out)
    _weight(ck, 200, 264, 288, dtype, out, bias=False)


def test_the_mlp_of_the_stack(ck):
    _weight(ck, 4608, 3072, 1024, torch.bfloat16, torch.float32)
    _input(ck, 4608, 3072, 1024, torch.bfloat16)


@pytest.mark.parametrize("dtype", DTYPES)
def test_zero_blocks_and_large_scales(ck, dtype):
    """Blocks of zeros (scale byte 0), blocks of far apart magnitudes."""
    x = _made((130, 96), torch.float32, 5)
    x[7], x[9, 32:64] = 0, 0
    x[11] *= 2.0**20
    x[12] *= 2.0**-30
    codes, scales = ck.quantize_mxfp8(x)
    held = ck.dequantize_mxfp8(codes, scales, torch.float32).double()
    dy = _made((130, 40), dtype, 6, 2.0**-12)
    dw, _ = ck.linear_weight_grad_mxfp8(dy, codes, scales, out_dtype=torch.float32)
    _check(dw, dy.double().t(), held, PARTS[dtype], "dw")
    g = _made((70, 130 // 8 * 8), dtype, 7, 2.0**-12)
    codes, scales = codes[:128].contiguous(), scales[:128].contiguous()
    _check(ck.linear_input_grad_mxfp8(g, codes, scales, out_dtype=torch.float32), g.double(), held[:128], PARTS[dtype], "dx")


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_every_bit_of_dy_counts(ck, dtype):
    """One row of dY against a matrix of ones on the diagonal: the result is dY to the last bit."""
    eye = torch.zeros(64, 64, device="cuda")
    eye.fill_diagonal_(1.0)
    codes, scales = ck.quantize_mxfp8(eye)
    dy = _made((16, 64), dtype, 8, 3.0)
    dy[0, :4] = torch.tensor([torch.finfo(dtype).max, -torch.finfo(dtype).max, torch.finfo(dtype).tiny, -0.0], dtype=dtype)
    assert torch.equal(ck.linear_input_grad_mxfp8(dy, codes, scales, out_dtype=torch.float32), dy.float())
    many = dy.repeat(20, 1)
    assert torch.equal(ck.linear_input_grad_mxfp8(many, codes, scales, out_dtype=torch.float32), many.float())


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinity_and_nan_stay_in_their_rows(ck, dtype):
    codes, scales, _ = _held(ck, 64, 64, 9)
    dy = _made((40, 64), dtype, 10)
    clean = ck.linear_input_grad_mxfp8(dy, codes, scales)
    dy[3, 5], dy[20, 6] = float("inf"), float("nan")
    dx = ck.linear_input_grad_mxfp8(dy, codes, scales)
    rows = torch.tensor([r for r in range(40) if r not in (3, 20)], device="cuda")
    assert torch.equal(dx[rows], clean[rows]) and torch.isnan(dx[20]).all() and not torch.isfinite(dx[3]).any()


def test_no_tokens(ck):
    codes, scales = torch.empty(0, 64, dtype=torch.float8_e4m3fn, device="cuda"), torch.empty(0, 4, dtype=torch.float8_e8m0fnu, device="cuda")
    dw, db = ck.linear_weight_grad_mxfp8(torch.empty(0, 16, device="cuda"), codes, scales, bias_grad=True)
    assert dw.shape == (16, 64) and db.shape == (16,) and not dw.any() and not db.any()
    w, s, _ = _held(ck, 16, 64, 11)
    assert ck.linear_input_grad_mxfp8(torch.empty(0, 16, device="cuda"), w, s).shape == (0, 64)


def test_strided_gradients_and_the_same_bits(ck):
    codes, scales, _ = _held(ck, 200, 128, 12)
    wide = _made((200, 3 * 64), torch.bfloat16, 13)
    dy = wide[:, 64:128]
    first = ck.linear_weight_grad_mxfp8(dy, codes, scales, bias_grad=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = ck.linear_weight_grad_mxfp8(dy.contiguous(), codes, scales, bias_grad=True)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        third = ck.linear_weight_grad_mxfp8(dy, codes, scales, bias_grad=True)
    graph.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(first, second, third):
        assert torch.equal(a, b) and torch.equal(a, c)
    one = wide.flatten()[1:1 + 64 * 8].view(8, 64)  # not on a 16-byte boundary
    assert torch.equal(ck.linear_weight_grad_mxfp8(one, codes[:8].contiguous(), scales[:128].contiguous())[0],
                       ck.linear_weight_grad_mxfp8(one.clone(), codes[:8].contiguous(), scales[:128].contiguous())[0])


def test_operators(ck):
    codes, scales, _ = _held(ck, 48, 64, 14)
    dy = _made((48, 16), torch.bfloat16, 15)
    dw, none = torch.ops.comfy_kitchen.linear_weight_grad_mxfp8(dy, codes, scales, 0, False)
    assert none.numel() == 0 and torch.equal(dw, ck.linear_weight_grad_mxfp8(dy, codes, scales, torch.float32)[0])
    g = _made((5, 48), torch.bfloat16, 16)
    assert torch.equal(torch.ops.comfy_kitchen.linear_input_grad_mxfp8(g, codes, scales, 2), ck.linear_input_grad_mxfp8(g, codes, scales))


def test_refusals(ck):
    codes, scales, _ = _held(ck, 64, 64, 17)
    with pytest.raises(AssertionError, match="do not match"):
        ck.linear_weight_grad_mxfp8(_made((32, 16), torch.bfloat16, 18), codes, scales)
    with pytest.raises(AssertionError, match="do not match"):
        ck.linear_input_grad_mxfp8(_made((32, 16), torch.bfloat16, 18), codes, scales)
    with pytest.raises(AssertionError, match="multiple"):
        ck.linear_weight_grad_mxfp8(_made((64, 12), torch.bfloat16, 18), codes, scales)
    with pytest.raises(AssertionError, match="scale"):
        ck.linear_weight_grad_mxfp8(_made((64, 16), torch.bfloat16, 18), codes, scales[:64])
    with pytest.raises(ck.NoCapableBackendError):
        ck.linear_weight_grad_mxfp8(_made((64, 16), torch.float64, 18), codes, scales)
    with pytest.raises(ck.NoCapableBackendError):
        ck.linear_weight_grad_mxfp8(_made((64, 16), torch.bfloat16, 18), codes.view(torch.uint8), scales)
    with pytest.raises(ck.NoCapableBackendError):
        ck.linear_input_grad_mxfp8(_made((64, 64), torch.bfloat16, 18).cpu(), codes.cpu(), scales.cpu())


@pytest.mark.parametrize("m,n,k", [(9, 6208, 512), (64, 12288, 128), (300, 560, 512), (300, 4096, 512)])
def test_small_numbers_of_dy_are_added_before_large_ones(ck, m, n, k):
    """An fp32 dY enters as three bf16 numbers, 2^-8 and 2^-16 of the first.  An accumulator loses up to 2^-23 of what it has reached with each addition of
    16 steps: 2048 steps of first numbers at most lose 128 * 2^-23 * 0.5 in the mean, towards zero, so 7.6e-6 if all sums
    had one size; they grow as the root of the number of steps, which leaves two thirds, and half of the additions leave the sum smaller: 2.6e-6.  With the
    others added at the same magnitude, three times the additions, it would be 7.6e-6."""
    dy = _made((m, n), torch.float32, 19)
    codes, scales, w = _held(ck, n, k, 20)
    dx = ck.linear_input_grad_mxfp8(dy, codes, scales)
    want = dy.double() @ w
    assert (dx.double() - want).norm() <= 2.6e-6 * want.norm()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [8, 40, 72, 128, 200, 264])
def test_padding_of_the_scales_is_not_read(ck, dtype, n):
    """Scales come in tiles of 128 rows and four blocks; what stands in those past the matrix's rows and columns must not reach a result: 0xFF is
    infinite, and the codes of rows past the last one are zeros."""
    k = 160
    codes, scales, _ = _held(ck, n, k, 21)
    bad = scales.clone()
    tall, wide = scales.shape[0] // 128, scales.shape[1] // 4
    rows = torch.arange(tall * 128, device="cuda").view(tall, 1, 4, 32, 1).transpose(2, 3)  # tile row, tile column, row % 32, row // 32, block
    blocks = torch.arange(wide * 4, device="cuda").view(1, wide, 1, 1, 4)
    tiles = bad.view(torch.uint8).view(tall, wide, 32, 4, 4)
    tiles[((rows >= n) | (blocks >= k // 32)).expand(tiles.shape)] = 0xFF
    assert (bad.view(torch.uint8) == 0xFF).sum() == scales.numel() - n * (k // 32)
    for m in (1, 5, 33, 300):  # decoded inside the product, and before it
        dy = _made((m, n), dtype, 22)
        got, clean = (ck.linear_input_grad_mxfp8(dy, codes, s) for s in (bad, scales))
        assert torch.isfinite(clean).all() and torch.equal(got, clean), m
    x_dy = _made((n, 64), dtype, 23)
    got, clean = (ck.linear_weight_grad_mxfp8(x_dy, codes, s, bias_grad=True) for s in (bad, scales))
    assert torch.equal(got[0], clean[0]) and torch.equal(got[1], clean[1])
