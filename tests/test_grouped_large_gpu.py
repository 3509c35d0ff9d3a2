"""The experts' products and their input gradient where there are many rows: the kernels of CTA pairs.

Bounds as in test_grouped_gpu.py: operands are exact, the accumulation is fp32, one addition for 16 contraction steps at most (and bf16 part of dY), each off by at
most 2^-22 of the running sum of magnitudes; then a bias, off by 2^-24, and one rounding to the result's type.
"""
from __future__ import annotations

import ctypes

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
    return codes, scales, torch.stack([ck.dequantize_mxfp8(codes[e], scales[e], torch.float32) for e in range(experts)])


def _ends(sizes):
    return torch.tensor(sizes, dtype=torch.int32).cumsum(0).to(torch.int32).cuda()


def _check(got, rows, weights, sizes, parts, bias=None, name="y"):
    """got against rows[i] @ weights[e] for each expert's rows, zeros behind them"""
    first = 0
    deep = rows.shape[1]
    assert torch.isfinite(got).all(), name
    for e, count in enumerate(sizes):
        if count:
            left, right = rows[first:first + count].double(), weights[e].double()
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


def _pairs(m, n, k, experts):
    """The product's own rule for its pairs: groups of more than 128 rows on average, more than 32 stages of 128 of the contraction for each SM."""
    used = min(experts, m)
    rows = -(-m // used)
    tiles = used * -(-rows // 128) * -(-n // 128)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    return rows > 128 and tiles > sms and tiles * -(-k // 128) > 32 * sms


def _kernel_edges(run):
    """Types of the dependencies between the kernels of a captured call: 0 for plain stream order, 1 for a programmatic start."""
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        out = run()
    edges_of, raw = ctypes.CDLL("libcuda.so.1").cuGraphGetEdges_v2, ctypes.c_void_p(graph.raw_cuda_graph())
    count = ctypes.c_size_t(0)
    assert edges_of(raw, None, None, None, ctypes.byref(count)) == 0
    nodes, data = ctypes.c_void_p * count.value, (ctypes.c_uint8 * 8 * count.value)()  # of an edge: ports at both ends, type, reserved
    assert edges_of(raw, nodes(), nodes(), data, ctypes.byref(count)) == 0
    del out, graph
    return [edge[2] for edge in data]


def test_pairs_start_behind_the_kernel_in_front(ck):
    """A pair's waits for the kernel in front of it, for tensor memory and for its other CTA have no limit: it starts where there is nothing to wait for."""
    m, n, k, experts = 1536, 1544, 4128, 4
    assert _pairs(m, n, k, experts)
    codes, scales, _ = _weights(ck, experts, n, k)
    ends, x, dy = _ends([384] * 4), _made((m, k), torch.bfloat16, 1), _made((m, n), torch.bfloat16, 2)
    xc, xs = ck.quantize_mxfp8(x)
    assert _kernel_edges(lambda: ck.grouped_linear_mxfp8(x, codes, scales, ends)) == [0]
    assert _kernel_edges(lambda: ck.grouped_mm_mxfp8(xc, codes, xs, scales, ends)) == [0]
    assert _kernel_edges(lambda: ck.grouped_input_grad_mxfp8(dy, codes, scales, ends)) == [0]


UNEVEN = [37 * i % 290 for i in range(64)]
# (experts' rows, rows behind them, N, K)
CASES = [
    ([700, 1, 0, 900, 257], 11, 1544, 4128),
    ([300, 0, 77, 255, 256, 513, 31, 2], 140, 2056, 4128),
    ([2100], 4, 2568, 4160),
    (UNEVEN, 0, 264, 1600),
    ([513, 255, 0, 300, 511], 0, 1544, 4096),
    ([1, 0, 0, 1900], 0, 1544, 4128),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes,behind,n,k", CASES)
def test_products(ck, dtype, sizes, behind, n, k):
    m = sum(sizes) + behind
    assert _pairs(m, n, k, len(sizes))
    x = _made((m, k), dtype, 1)
    codes, scales, w = _weights(ck, len(sizes), n, k)
    bias = _made((len(sizes), n), dtype, 3)
    xc, xs = ck.quantize_mxfp8(x)
    held = ck.dequantize_mxfp8(xc, xs, torch.float32)
    y = ck.grouped_linear_mxfp8(x, codes, scales, _ends(sizes))
    assert y.dtype == dtype and y.shape == (m, n)
    _check(y, held, w.transpose(1, 2), sizes, 1)
    y = ck.grouped_mm_mxfp8(xc, codes, xs, scales, _ends(sizes), bias, out_dtype=dtype)
    _check(y, held, w.transpose(1, 2), sizes, 1, bias)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("sizes,behind,n,k", [c for c in CASES if sum(c[0]) + c[1] > 256 * len(c[0])])
def test_input_grad(ck, dtype, sizes, behind, n, k):
    dy = _made((sum(sizes) + behind, n), dtype, 4)
    codes, scales, w = _weights(ck, len(sizes), n, k)
    for out in {dtype, torch.float32}:
        dx = ck.grouped_input_grad_mxfp8(dy, codes, scales, _ends(sizes), out_dtype=out)
        _check(dx, dy, w, sizes, PARTS[dtype], name="dx")


@pytest.mark.parametrize("m,n", [(384, 256), (384, 200), (2560, 1544)])
def test_one_experts_gradient_is_the_plain_one(ck, m, n):
    """The same exact products, added in another order: twice the bound of one result."""
    dy = _made((m, n), torch.bfloat16, 6)
    codes, scales, w = _weights(ck, 1, n, 256)
    got = ck.grouped_input_grad_mxfp8(dy, codes, scales, _ends([m]), out_dtype=torch.float32)
    want = ck.linear_input_grad_mxfp8(dy, codes[0], scales[0], out_dtype=torch.float32)
    magnitude = dy.double().abs() @ w[0].double().abs()
    assert ((got.double() - want.double()).abs() <= 2 * ((n / 16 + 4) * 2.0**-22 + 2.0**-24) * magnitude).all()


SIZES, BEHIND, N, K = [700, 0, 500, 0], 300, 1544, 4128  # pairs in the product, the GEMM in the gradient


@pytest.fixture(scope="module")
def large(ck):
    m = sum(SIZES) + BEHIND
    assert _pairs(m, N, K, 4) and m > 4 * 256
    codes, scales, _ = _weights(ck, 4, N, K)
    return codes, scales, _made((m, K), torch.bfloat16, 11), _made((m, N), torch.bfloat16, 12)


def _both(ck, x, dy, codes, scales, ends):
    return ck.grouped_linear_mxfp8(x, codes, scales, ends), ck.grouped_input_grad_mxfp8(dy, codes, scales, ends)


def _poison():
    """Memory that the next calls' results and workspaces come from, full of NaN."""
    held = [torch.full((1 << 28,), 0xFF, dtype=torch.uint8, device="cuda") for _ in range(2)]
    del held


def test_what_belongs_to_nobody_has_no_part(ck, large):
    """NaN in the weights of experts without rows, in rows behind the last expert, in the scales' padding and in what a call works on: no trace in the result."""
    codes, scales, x, dy = (t.clone() for t in large)
    ends = _ends(SIZES)
    y, dx = _both(ck, x, dy, codes, scales, ends)
    for e in (1, 3):
        codes[e].view(torch.uint8).fill_(0x7F)
        scales[e].view(torch.uint8).fill_(0xFF)
    tiles = scales.view(torch.uint8).view(4, 13, 33, 32, 4, 4)  # [expert, row block, column tile, row % 32, row / 32, column]
    tiles[:, :, 32, :, :, 1:] = 0xFF  # columns from 129 on
    tiles[:, 12, :, 8:] = 0xFF        # rows from 1544 on
    tiles[:, 12, :, :, 1:] = 0xFF
    x[1200:], dy[1200:] = float("nan"), float("nan")
    _poison()
    again = _both(ck, x, dy, codes, scales, ends)
    assert torch.equal(y, again[0]) and torch.equal(dx, again[1])
    xc, xs = ck.quantize_mxfp8(large[2])
    _poison()
    assert torch.equal(y, ck.grouped_mm_mxfp8(xc, codes, xs, scales, ends))


def test_nan_and_infinities_stay_in_their_rows(ck, large):
    codes, scales, x, dy = (t.clone() for t in large)
    ends = _ends([700, 0, 500, 300])
    y, dx = _both(ck, x, dy, codes, scales, ends)
    rows = [699, 700, 1199, 1499]
    x[rows, 5], dy[rows, 7] = float("nan"), float("nan")
    dy[1200, 0] = float("inf")
    again = _both(ck, x, dy, codes, scales, ends)
    assert again[0][rows].isnan().all() and again[1][rows].isnan().all() and not again[1][1200].isfinite().any()
    others = torch.ones(1500, dtype=torch.bool, device="cuda")
    others[rows] = False
    assert torch.equal(y[others], again[0][others])
    others[1200] = False
    assert torch.equal(dx[others], again[1][others])


def test_captured_and_replayed_with_other_ends(ck, large):
    codes, scales, x, dy = large
    ends = _ends([375] * 4)
    _both(ck, x, dy, codes, scales, ends)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, dx = _both(ck, x, dy, codes, scales, ends)
    for sizes in ([375] * 4, [1500, 0, 0, 0], [0, 1, 2, 1497], [0, 0, 0, 3], [0, 0, 0, 0], [257, 255, 513, 400]):
        ends.copy_(_ends(sizes))
        y.fill_(7), dx.fill_(7)
        graph.replay()
        want = _both(ck, x, dy, codes, scales, ends)
        assert torch.equal(y, want[0]) and torch.equal(dx, want[1])
        assert not y[sum(sizes):].any() and not dx[sum(sizes):].any()
    del graph


def test_two_streams_at_once(ck, large):
    codes, scales, *_ = large
    ends = _ends(SIZES)
    inputs = [(_made((1500, K), torch.bfloat16, s), _made((1500, N), torch.bfloat16, s + 10)) for s in (16, 17)]
    want = [_both(ck, x, dy, codes, scales, ends) for x, dy in inputs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(6):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(_both(ck, *inputs[i], codes, scales, ends))
    torch.cuda.synchronize()
    for i in (0, 1):
        for y, dx in got[i]:
            assert torch.equal(y, want[i][0]) and torch.equal(dx, want[i][1])


def test_again_and_again(ck, large):
    codes, scales, x, dy = large
    ends = _ends([375] * 4)
    y, dx = _both(ck, x, dy, codes, scales, ends)
    for _ in range(100):
        again = _both(ck, x, dy, codes, scales, ends)
        assert torch.equal(y, again[0]) and torch.equal(dx, again[1])
