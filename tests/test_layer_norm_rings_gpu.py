"""Layer norm over many rows, which come through rings in shared memory: against the definition in 64 bits, with the bounds of test_layer_norm_gpu.py."""
from __future__ import annotations

import pytest
import torch
from test_layer_norm_gpu import DTYPES, _made, _run

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
