"""Layer norm over many rows, which come through rings in shared memory: against the definition in 64 bits, with the bounds of test_layer_norm_gpu.py."""
from __future__ import annotations

import pytest
import torch
from test_layer_norm_gpu import DTYPES, ROUND, U, _made, _run

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


@pytest.mark.parametrize("dtype,widths", [(torch.bfloat16, (2568, 3064)), (torch.float32, (1284, 1532)), (torch.float16, (2567, 3063))])
def test_calls_of_several_threads(ck, dtype, widths):
    """Host threads with widths that the same kernels take with different amounts of shared memory: no call changes what another one's launch may use.
    The library's functions are called directly, which leaves the interpreter's lock to the other threads for all of their time."""
    import threading

    from comfy_kitchen.backends import cuda as backend
    from comfy_kitchen.ops import DTYPE_TO_CODE

    lib, code, rows = backend.load_library(), DTYPE_TO_CODE[dtype], 300
    calls, kept, refused = [], [], []
    for seed in range(6):
        cols = widths[seed % 2]
        x, dy, w = _made((rows, cols), dtype, seed), _made((rows, cols), dtype, 9), _made((cols,), dtype, 10)
        y, dx, dw, db = torch.empty_like(x), torch.empty_like(x), torch.empty_like(w), torch.empty_like(w)
        mean, rstd = (torch.empty(rows, device="cuda") for _ in range(2))
        need = lib.ck_layer_norm_backward_workspace_bytes(rows, cols, 1)
        ws, stream = torch.empty(need, dtype=torch.uint8, device="cuda"), torch.cuda.Stream()
        forward = (x.data_ptr(), code, rows, cols, rows, 0, cols, w.data_ptr(), None, code, 1, 0, 0, 0.0, 1e-5, y.data_ptr(), mean.data_ptr(), rstd.data_ptr(), None,
                   None, stream.cuda_stream)
        backward = (dy.data_ptr(), code, rows, cols, rows, 0, cols, x.data_ptr(), rows, 0, cols, None, None, mean.data_ptr(), rstd.data_ptr(), w.data_ptr(), code, 1, 0,
                    0.0, dx.data_ptr(), dw.data_ptr(), db.data_ptr(), ws.data_ptr(), need, stream.cuda_stream)
        calls.append((forward, backward))
        kept.append((x, dy, w, y, dx, dw, db, mean, rstd, ws, stream))
    torch.cuda.synchronize()

    def run(forward, backward):
        for _ in range(3000):
            if lib.ck_layer_norm_forward(*forward) or lib.ck_layer_norm_backward(*backward):
                refused.append(lib.ck_last_error())

    threads = [threading.Thread(target=run, args=pair) for pair in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not refused, (len(refused), refused[0])
    for x, dy, w, y, dx, dw, db, mean, rstd, _, _ in kept:
        want_y, want_mean, want_rstd = backend.layer_norm_forward(x, w)
        want_dx, want_dw, want_db = backend.layer_norm_backward(dy, x, want_mean, want_rstd, w)
        assert torch.equal(y, want_y) and torch.equal(dx, want_dx) and torch.equal(dw, want_dw[0]) and torch.equal(db, want_db[0])


# teams of one warp and of several, forward and backward, on 16-byte boundaries, on those of pairs and on none
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(300, 520), (2400, 1000), (400, 3072), (2400, 3072), (300, 5120), (300, 12288), (600, 1002), (400, 3070), (2400, 3071), (300, 9001)])
def test_constant_rows(ck, dtype, rows, cols):
    """A row of equal numbers is its own mean, which fp32 holds, as it holds the sums (numbers of seven bits at most, fewer than 2^14 of them): h is 0
    to the last bit, although 1/std is 316, y is the bias and the weight's gradient is 0.  As few rows, so many."""
    value = torch.tensor([1000.0, -13.0, 88.0, 3.0 / 64, 57344.0, 0.0], device="cuda").repeat(rows)[:rows]
    x = value.to(dtype).unsqueeze(1).expand(rows, cols).contiguous()
    w, b = _made((cols,), dtype, 60, 0.2, 1.0), _made((cols,), dtype, 61)
    y, mean, rstd = ck.layer_norm_forward(x, w, b)
    assert torch.equal(mean, value)
    assert torch.equal(y, b.expand(rows, cols)) and torch.equal(ck.layer_norm_forward(x[:6], w, b)[0], y[:6])
    dy = _made((rows, cols), dtype, 62)
    dx, dw, _ = ck.layer_norm_backward(dy, x, mean, rstd, w)
    assert not dw.any()
    # dx = (g - mean g) / sqrt(eps): 128 u of the mean of |g| for the sum, 4 roundings of g
    g = dy.double() * w.double()
    want = (g - g.mean(1, keepdim=True)) / 1e-5**0.5
    limit = (128 * U * g.abs().mean(1, keepdim=True) + 8 * U * g.abs()) / 1e-5**0.5
    assert ((dx.double() - want).abs() <= limit + ROUND[dtype] * (want.abs() + limit)).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("checkpoint", [False, True])
@pytest.mark.parametrize("rows,cols", [(400, 3072), (2400, 3072), (300, 12288), (2400, 3071), (600, 3070)])
def test_rows_that_are_nearly_constant(ck, dtype, checkpoint, rows, cols):
    """One number of a row differs by a step of the type.  All sums are exact (multiples of 8, below 2^24 of them), so the mean is off by
    at most two roundings, or four where warps meet, and h by that over the deviation."""
    if checkpoint and cols % 32:
        pytest.skip("a copy has rows of a multiple of 32")
    x = torch.full((rows, cols), 1024.0, dtype=dtype, device="cuda")
    x[torch.arange(rows), torch.arange(rows) * 37 % cols] = 1032.0
    y, mean, rstd = ck.layer_norm_forward(x)
    d = x.double()
    exact_mean, var = d.mean(1, keepdim=True), d.var(1, correction=0, keepdim=True)
    exact_rstd = 1 / torch.sqrt(var + 1e-5)
    off = 4 * U * 1024
    assert ((mean.double().unsqueeze(1) - exact_mean).abs() <= off).all()
    # var: the squares about a mean that is off add off^2 and cross terms that vanish; 8 u for its own sums and root
    limit_r = exact_rstd * (16 * U + off**2 * exact_rstd**2 + 128 * U)
    assert ((rstd.double().unsqueeze(1) - exact_rstd).abs() <= limit_r).all()
    h = (d - exact_mean) * exact_rstd
    limit = off * exact_rstd + h.abs() * (160 * U + off**2 * exact_rstd**2)
    assert ((y.double() - h).abs() <= limit + ROUND[dtype] * (h.abs() + limit)).all()
    dy = torch.ones_like(x)  # the weight's gradient is the sum of h
    if checkpoint:
        _, mean, rstd, codes, scales = ck.layer_norm_forward_mxfp8(x)
        kept = ck.dequantize_mxfp8(codes, scales, torch.float32).double()
        _, dw, _ = ck.layer_norm_backward_mxfp8(dy, codes, scales, mean, rstd, param_dtype=torch.float32)
    else:
        kept = d
        _, dw, _ = ck.layer_norm_backward(dy, x, mean, rstd, param_dtype=torch.float32)
    hk = (kept - exact_mean) * exact_rstd
    limit = (off * exact_rstd + hk.abs() * (160 * U + off**2 * exact_rstd**2)).sum(0, keepdim=True) + rows * U * hk.abs().sum(0, keepdim=True)
    assert ((dw.double() - hk.sum(0, keepdim=True)).abs() <= limit).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("checkpoint", [False, True])
@pytest.mark.parametrize("rows,cols", [(300, 544), (700, 5120), (320, 6016), (1500, 8192), (500, 12288), (310, 13824), (420, 16384), (300, 18432)])
def test_teams_of_several_warps(ck, dtype, checkpoint, rows, cols):
    """Whole vectors, a row over two to sixteen warps, up to the widest row that the ring takes: threads that are full, that are not, and that have nothing."""
    x = _made((rows, cols), dtype, 70, 2.0, 0.3)
    _run(ck, x, _made((cols,), dtype, 71, 0.2, 1.0), _made((cols,), dtype, 72, 0.2), checkpoint=checkpoint)
    if cols % 2048 == 0:
        x = _made((2, rows, cols), dtype, 73)
        _run(ck, x, _made((2, cols), torch.float32, 74, 0.2), _made((2, cols), torch.float32, 75), 1.0, checkpoint)
