"""Products of rows grouped by expert with MXFP8 weights, on the GPU, against the definition in 64 bits.

Bounds.  Operands are exact, the accumulation is fp32: one addition for 16 contraction steps at most (and, for the gradient, bf16 part of dY), each off by
at most 2^-22 of the running sum of magnitudes.  Then a bias, whose addition is off by 2^-24, and one rounding to the result's type.
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


def _weights(ck, experts, n, k, seed=5):
    codes, scales = ck.quantize_experts_mxfp8(_made((experts, n, k), torch.float32, seed, 0.05))
    values = torch.stack([ck.dequantize_mxfp8(codes[e], scales[e], torch.float32) for e in range(experts)])
    return codes, scales, values.double()


def _ends(sizes):
    return torch.tensor(sizes, dtype=torch.int32).cumsum(0).to(torch.int32).cuda()


def _check(got, rows, weights, sizes, parts, bias=None, name="y"):
    """got against rows[i] @ weights[e] for each expert's rows, zeros behind them"""
    first = 0
    deep = rows.shape[1]
    assert torch.isfinite(got).all(), name
    for e, count in enumerate(sizes):
        if count:
            left, right = rows[first:first + count], weights[e]
            value, magnitude = left @ right, left.abs() @ right.abs()
            limit = (deep / 16 * parts + 4) * 2.0**-22 * magnitude
            if bias is not None:
                value = value + bias[e].double()
                limit = limit + 2.0**-24 * (value.abs() + limit)
            limit = limit + ROUND[got.dtype] * (value.abs() + limit) + TINY[got.dtype]
            off = (got[first:first + count].double() - value).abs()
            assert (off <= limit).all(), f"{name}, expert {e}: {(off / limit).max().item():.3g} times the bound"
        first += count
    assert (got[first:] == 0).all(), f"{name}: rows behind the last expert"


# (experts' rows, rows behind them, N, K)
CASES = [
    ([1], 0, 8, 32),
    ([0], 3, 16, 64),
    ([0, 1, 0], 0, 72, 96),
    ([5, 0, 3, 0, 0, 130], 7, 200, 160),
    ([127, 129, 128, 1], 0, 264, 288),
    ([300, 0, 77], 140, 520, 544),
    ([33, 31, 9, 8, 7, 1, 255], 0, 1000, 1056),
    ([1] * 40, 2, 136, 128),
    ([700, 1, 0, 900, 257], 11, 1544, 320),
    ([256, 256], 0, 4864, 256),
    ([2100], 4, 2568, 416),
    ([0] * 1000 + [3] * 24, 0, 64, 64),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes,behind,n,k", CASES)
def test_linear(ck, dtype, sizes, behind, n, k):
    m = sum(sizes) + behind
    x = _made((m, k), dtype, 1)
    codes, scales, w = _weights(ck, len(sizes), n, k)
    y = ck.grouped_linear_mxfp8(x, codes, scales, _ends(sizes))
    assert y.dtype == dtype and y.shape == (m, n)
    xc, xs = ck.quantize_mxfp8(x)
    held = ck.dequantize_mxfp8(xc, xs, torch.float32).double()
    _check(y, held, w.transpose(1, 2), sizes, 1)


@pytest.mark.parametrize("out", DTYPES)
@pytest.mark.parametrize("sizes,behind,n,k", CASES)
def test_mm_with_bias(ck, out, sizes, behind, n, k):
    m = sum(sizes) + behind
    xc, xs = ck.quantize_mxfp8(_made((m, k), torch.bfloat16, 2))
    codes, scales, w = _weights(ck, len(sizes), n, k)
    bias = _made((len(sizes), n), out, 3)
    y = ck.grouped_mm_mxfp8(xc, codes, xs, scales, _ends(sizes), bias, out_dtype=out)
    _check(y, ck.dequantize_mxfp8(xc, xs, torch.float32).double(), w.transpose(1, 2), sizes, 1, bias)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes,behind,n,k", CASES)
def test_input_grad(ck, dtype, sizes, behind, n, k):
    m = sum(sizes) + behind
    dy = _made((m, n), dtype, 4)
    codes, scales, w = _weights(ck, len(sizes), n, k)
    dx = ck.grouped_input_grad_mxfp8(dy, codes, scales, _ends(sizes))
    assert dx.dtype == dtype and dx.shape == (m, k)
    _check(dx, dy.double(), w, sizes, PARTS[dtype], name="dx")


@pytest.mark.parametrize("n", [256, 200])
def test_one_expert_is_the_plain_product(ck, n):
    """The rows of one expert alone: the same numbers as scaled_mm_mxfp8 and linear_input_grad_mxfp8 give, to the order of their sums."""
    xc, xs = ck.quantize_mxfp8(_made((384, 256), torch.bfloat16, 6))
    codes, scales, _ = _weights(ck, 1, n, 256)
    got = ck.grouped_mm_mxfp8(xc, codes, xs, scales, _ends([384]), out_dtype=torch.float32)
    want = ck.scaled_mm_mxfp8(xc, codes[0], xs, scales[0], out_dtype=torch.float32)
    assert (got - want).abs().max() <= 1e-5 * want.abs().max()


def test_gradient_through_autograd(ck):
    sizes, n, k = [40, 0, 100], 264, 320
    codes, scales, w = _weights(ck, 3, n, k)
    x = _made((140, k), torch.bfloat16, 7).requires_grad_()
    dy = _made((140, n), torch.bfloat16, 8)
    y = ck.grouped_linear_mxfp8(x, codes, scales, _ends(sizes))
    (dx,) = torch.autograd.grad(y, x, dy)
    _check(dx, dy.double(), w, sizes, 1, name="dx")
    with torch.no_grad():
        assert torch.equal(y, ck.grouped_linear_mxfp8(x, codes, scales, _ends(sizes)))
    # and against differences of the product with the rows as the gradient takes them: linear in dy
    assert torch.equal(ck.grouped_input_grad_mxfp8(dy * 2, codes, scales, _ends(sizes)), dx * 2)


def test_the_dispatchers_route(ck):
    """Under a mode that watches operators the call goes through torch.ops, gradient included."""
    from torch.utils._python_dispatch import TorchDispatchMode

    class Watch(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.seen = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.seen.append(str(func))
            return func(*args, **(kwargs or {}))

    codes, scales, _ = _weights(ck, 2, 64, 96)
    ends = _ends([10, 20])
    x, dy = _made((30, 96), torch.float16, 9).requires_grad_(), _made((30, 64), torch.float16, 10)
    want = torch.autograd.grad(ck.grouped_linear_mxfp8(x, codes, scales, ends), x, dy)[0]
    with Watch() as watch:
        got = torch.autograd.grad(ck.grouped_linear_mxfp8(x, codes, scales, ends), x, dy)[0]
    assert any("grouped_linear_mxfp8" in s for s in watch.seen) and any("grouped_input_grad_mxfp8" in s for s in watch.seen)
    assert torch.equal(got, want)


def test_what_belongs_to_nobody_has_no_part(ck):
    """NaN in the weights of experts without rows, in rows behind the last expert, and in the scales' padding: no trace in the result."""
    sizes, n, k = [50, 0, 70, 0], 136, 96
    codes, scales, w = _weights(ck, 4, n, k)
    ends = _ends(sizes)
    x = _made((150, k), torch.bfloat16, 11)
    dy = _made((150, n), torch.bfloat16, 12)
    y, dx = ck.grouped_linear_mxfp8(x, codes, scales, ends), ck.grouped_input_grad_mxfp8(dy, codes, scales, ends)
    for e in (1, 3):
        codes[e].view(torch.uint8).fill_(0x7F)
        scales[e].view(torch.uint8).fill_(0xFF)
    tiles = scales.view(torch.uint8).view(4, 2, 1, 32, 4, 4)  # [expert, row block, column tile, row % 32, row / 32, column]
    tiles[:, :, :, :, :, 3] = 0xFF  # the fourth of three columns
    tiles[:, 1, :, 8:] = 0xFF       # rows from 136 on
    x[120:], dy[120:] = float("nan"), float("nan")
    assert torch.equal(y, ck.grouped_linear_mxfp8(x, codes, scales, ends))
    assert torch.equal(dx, ck.grouped_input_grad_mxfp8(dy, codes, scales, ends))
    xc, xs = ck.quantize_mxfp8(_made((150, k), torch.bfloat16, 11))
    assert torch.equal(y, ck.grouped_mm_mxfp8(xc, codes, xs, scales, ends))


def test_nan_and_infinities_stay_in_their_rows(ck):
    sizes, n, k = [50, 70], 136, 96
    codes, scales, _ = _weights(ck, 2, n, k)
    dy = _made((120, n), torch.float32, 12)
    want = ck.grouped_input_grad_mxfp8(dy, codes, scales, _ends(sizes))
    dy[49, 3], dy[50, 7], dy[119, 0] = float("nan"), float("inf"), float("nan")
    got = ck.grouped_input_grad_mxfp8(dy, codes, scales, _ends(sizes))
    other = [i for i in range(120) if i not in (49, 50, 119)]
    assert torch.equal(got[other], want[other])
    assert got[49].isnan().all() and got[119].isnan().all() and not got[50].isfinite().any()


def test_ends_that_make_no_sense_stay_inside(ck):
    """Ends that decrease, lie below zero or behind the rows: any rows, but the call ends and the groups that are right are right."""
    n, k = 72, 64
    codes, scales, w = _weights(ck, 4, n, k)
    x = _made((100, k), torch.bfloat16, 13)
    for ends in ([30, 10, 5, 100], [-5, 40, 2**31 - 1, 7], [200, 300, 400, 500], [-1, -1, -1, -1]):
        e = torch.tensor(ends, dtype=torch.int32).cuda()
        assert ck.grouped_linear_mxfp8(x, codes, scales, e).shape == (100, n)
        assert ck.grouped_input_grad_mxfp8(_made((100, n), torch.float32, 1), codes, scales, e).shape == (100, k)
    torch.cuda.synchronize()
    from comfy_kitchen.backends.cuda import check_device_status

    check_device_status()


def test_captured_and_replayed_with_other_ends(ck):
    n, k, experts = 520, 256, 5
    codes, scales, _ = _weights(ck, experts, n, k)
    x, dy = _made((600, k), torch.bfloat16, 14), _made((600, n), torch.bfloat16, 15)
    ends = _ends([100, 100, 100, 100, 100])
    ck.grouped_linear_mxfp8(x, codes, scales, ends), ck.grouped_input_grad_mxfp8(dy, codes, scales, ends)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, dx = ck.grouped_linear_mxfp8(x, codes, scales, ends), ck.grouped_input_grad_mxfp8(dy, codes, scales, ends)
    for sizes in ([100] * 5, [600, 0, 0, 0, 0], [0, 1, 2, 500, 90], [0, 0, 0, 0, 3]):
        ends.copy_(_ends(sizes))
        graph.replay()
        assert torch.equal(y, ck.grouped_linear_mxfp8(x, codes, scales, ends))
        assert torch.equal(dx, ck.grouped_input_grad_mxfp8(dy, codes, scales, ends))
    del graph


def test_two_streams_at_once(ck):
    sizes = [300, 200, 12]
    codes, scales, _ = _weights(ck, 3, 1032, 512)
    ends = _ends(sizes)
    xs = [_made((512, 512), torch.bfloat16, s) for s in (16, 17)]
    want = [ck.grouped_linear_mxfp8(x, codes, scales, ends) for x in xs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [None, None]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = ck.grouped_linear_mxfp8(xs[i], codes, scales, ends)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_strided_and_misaligned_rows(ck):
    sizes, n, k = [9, 21], 72, 96
    codes, scales, _ = _weights(ck, 2, n, k)
    ends = _ends(sizes)
    wide = _made((30, k + 8), torch.bfloat16, 18)
    x = wide[:, 3:3 + k]
    assert torch.equal(ck.grouped_linear_mxfp8(x, codes, scales, ends), ck.grouped_linear_mxfp8(x.contiguous(), codes, scales, ends))
    flat = _made((30 * n + 1,), torch.bfloat16, 19)
    dy = flat[1:].view(30, n)
    assert torch.equal(ck.grouped_input_grad_mxfp8(dy, codes, scales, ends), ck.grouped_input_grad_mxfp8(dy.clone(), codes, scales, ends))


def test_no_rows(ck):
    codes, scales, _ = _weights(ck, 2, 64, 32)
    ends = _ends([0, 0])
    assert ck.grouped_linear_mxfp8(torch.empty(0, 32, device="cuda"), codes, scales, ends).shape == (0, 64)
    assert ck.grouped_input_grad_mxfp8(torch.empty(0, 64, device="cuda"), codes, scales, ends).shape == (0, 32)


def test_module(ck):
    from comfy_kitchen.experts import MXFP8Experts

    w, b = _made((3, 136, 96), torch.bfloat16, 20, 0.1), _made((3, 136), torch.bfloat16, 21)
    layer = MXFP8Experts.from_float(w, b)
    x, ends = _made((40, 96), torch.bfloat16, 22), _ends([10, 0, 30])
    y = layer(x, ends)
    other = MXFP8Experts(3, 96, 136, bias=True, device="cuda", dtype=torch.bfloat16)
    other.load_state_dict(layer.state_dict())
    assert torch.equal(other(x, ends), y)
    xc, xs = ck.quantize_mxfp8(x)
    held = ck.dequantize_mxfp8(xc, xs, torch.float32).double()
    values = torch.stack([ck.dequantize_mxfp8(layer.weight[e].view(torch.float8_e4m3fn), layer.weight_scale[e].view(torch.float8_e8m0fnu), torch.float32)
                          for e in range(3)]).double()
    _check(y, held, values.transpose(1, 2), [10, 0, 30], 1, b)


def test_refusals(ck):
    codes, scales, _ = _weights(ck, 2, 64, 32)
    ends, x = _ends([1, 1]), torch.zeros(2, 32, device="cuda")
    with pytest.raises(Exception):
        ck.grouped_linear_mxfp8(x, codes, scales, ends.long())
    with pytest.raises(Exception):
        ck.grouped_linear_mxfp8(x, codes, scales, ends[:1])
    with pytest.raises(Exception):
        ck.grouped_linear_mxfp8(x[:, :16], codes, scales, ends)
    with pytest.raises(Exception):
        ck.grouped_linear_mxfp8(x, codes, scales[:1], ends)
    with pytest.raises(Exception):
        ck.grouped_linear_mxfp8(x, codes, scales, ends.cpu())
    with pytest.raises(Exception):
        ck.grouped_linear_mxfp8(x.double(), codes, scales, ends)
    with pytest.raises(Exception):
        ck.grouped_linear_mxfp8(x, codes.transpose(1, 2), scales, ends)
    with pytest.raises(Exception):
        ck.grouped_linear_mxfp8(x, codes, scales, ends, torch.zeros(2, 63, device="cuda"))
    with pytest.raises(ValueError):
        ck.grouped_linear_mxfp8(x, codes, scales, ends, torch.zeros(2, 64, device="cuda", requires_grad=True))
    with pytest.raises(Exception):
        ck.grouped_input_grad_mxfp8(x, codes, scales, ends)
    with pytest.raises(Exception):
        ck.grouped_mm_mxfp8(codes[0], codes, scales[:, :64], scales, ends)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("sizes,behind,n,k", [
    ([17] * 9, 0, 72, 160), ([1, 2, 3, 60, 5, 0, 0, 90], 5, 1160, 288), ([200] + [0] * 30 + [3], 1, 64, 96), ([100, 120, 140], 0, 200, 1056),
    ([40] * 24, 0, 328, 416), ([3] * 160, 0, 136, 64), ([130, 1], 0, 2056, 128), ([8], 0, 6208, 2624)])
def test_input_grad_of_few_rows(ck, dtype, out, sizes, behind, n, k):
    """Groups of up to about a hundred rows, among them some with several tiles' worth and some with none."""
    dy = _made((sum(sizes) + behind, n), dtype, 23)
    codes, scales, w = _weights(ck, len(sizes), n, k)
    dx = ck.grouped_input_grad_mxfp8(dy, codes, scales, _ends(sizes), out_dtype=out)
    assert dx.dtype == out
    _check(dx, dy.double(), w, sizes, PARTS[dtype], name="dx")
    for _ in range(3):
        assert torch.equal(dx, ck.grouped_input_grad_mxfp8(dy, codes, scales, _ends(sizes), out_dtype=out))


@pytest.mark.parametrize("dtype,rows,k", [(torch.bfloat16, 200, 256), (torch.float16, 96, 128), (torch.float16, 200, 256), (torch.float32, 200, 256)])
def test_input_grad_again_and_again(ck, dtype, rows, k):
    """A long contraction whose MMAs are behind the decoding: codes that were read late were those of a later step, in one pass of ten."""
    dy = _made((rows, 4864), dtype, 24)
    codes, scales, w = _weights(ck, 1, 4864, k)
    first = ck.grouped_input_grad_mxfp8(dy, codes, scales, _ends([rows]), out_dtype=torch.float32)
    _check(first, dy.double(), w, [rows], PARTS[dtype], name="dx")
    for _ in range(300):
        assert torch.equal(first, ck.grouped_input_grad_mxfp8(dy, codes, scales, _ends([rows]), out_dtype=torch.float32))
