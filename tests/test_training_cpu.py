"""The training operators where there is no GPU: shapes under tracing, refusals of tensors elsewhere, the C entry points' checks of arguments."""
from __future__ import annotations

import ctypes
import importlib.util
import os

import pytest
import torch
from conftest import PKG_DIR
from torch._subclasses.fake_tensor import FakeTensorMode

import comfy_kitchen as ck

FAKE = 0x10000  # an aligned address that no call reads


@pytest.fixture(scope="module")
def lib():
    spec = importlib.util.spec_from_file_location("ck_build", os.path.join(PKG_DIR, "build.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    lib = ctypes.CDLL(mod.build())
    from comfy_kitchen.backends import cuda

    for name, types in cuda._SIGNATURES.items():
        getattr(lib, name).argtypes = types
    for name in ("ck_layer_norm_backward_workspace_bytes", "ck_linear_grad_mxfp8_workspace_bytes"):
        getattr(lib, name).restype = ctypes.c_int64
    lib.ck_last_error.restype = ctypes.c_char_p
    return lib


def _refused(lib, call, said):
    assert call != 0
    assert said in lib.ck_last_error().decode(), lib.ck_last_error()


def _norm(lib, **kw):
    a = dict(x=FAKE, dtype=2, rows=4, cols=64, inner=4, outer=0, stride=64, w=None, b=None, pdtype=2, groups=1, ws=0, bs=0, offset=0.0, eps=1e-5, y=FAKE,
             mean=FAKE, rstd=FAKE, codes=None, scales=None, stream=None)
    a.update(kw)
    return lib.ck_layer_norm_forward(*a.values())


def test_layer_norm_arguments(lib):
    _refused(lib, _norm(lib, x=None), "null")
    _refused(lib, _norm(lib, y=None), "null")
    _refused(lib, _norm(lib, rstd=None), "mean and rstd")
    _refused(lib, _norm(lib, codes=FAKE), "codes and block_scales")
    _refused(lib, _norm(lib, codes=FAKE + 4, scales=FAKE), "aligned")
    _refused(lib, _norm(lib, codes=FAKE, scales=FAKE, cols=40, stride=40), "multiple of 32")
    _refused(lib, _norm(lib, dtype=7), "dtype")
    _refused(lib, _norm(lib, pdtype=1), "dtype")
    _refused(lib, _norm(lib, rows=0), "empty")
    _refused(lib, _norm(lib, cols=0), "empty")
    _refused(lib, _norm(lib, groups=3), "group")
    assert lib.ck_layer_norm_backward_workspace_bytes(0, 64, 1) == 0


def test_gelu_arguments(lib):
    _refused(lib, lib.ck_gelu_mxfp8_forward(None, 2, FAKE, FAKE, FAKE, 4, 64, None), "null")
    _refused(lib, lib.ck_gelu_mxfp8_forward(FAKE, 2, FAKE, FAKE, None, 4, 64, None), "go together")
    _refused(lib, lib.ck_gelu_mxfp8_forward(FAKE, 2, FAKE, FAKE, FAKE, 4, 40, None), "shape")
    _refused(lib, lib.ck_gelu_mxfp8_forward(FAKE, 9, FAKE, FAKE, FAKE, 4, 64, None), "dtype")
    _refused(lib, lib.ck_gelu_mxfp8_backward(FAKE + 16, 2, FAKE, FAKE, FAKE, 4, 64, None), "aligned")
    _refused(lib, lib.ck_gelu_mxfp8_backward(FAKE, 2, None, None, FAKE, 4, 64, None), "null")


def test_linear_gradient_arguments(lib):
    size = lib.ck_linear_grad_mxfp8_workspace_bytes
    assert size(1, 2, 1, 64, 64, 64) > 0 and size(0, 2, 0, 64, 64, 64) > 0
    assert size(1, 2, 1, 64, 12, 64) == 0 and size(1, 2, 1, 64, 64, 40) == 0 and size(1, 9, 1, 64, 64, 64) == 0
    need = 1 << 30
    for entry in ("weight", "input"):
        def call(dy=FAKE, dtype=2, codes=FAKE, scales=FAKE, out=FAKE, out_dtype=2, m=64, n=64, k=64, ws=FAKE, need=need, entry=entry):
            if entry == "weight":
                return lib.ck_linear_weight_grad_mxfp8(dy, dtype, codes, scales, out, out_dtype, None, m, n, k, ws, need, None)
            return lib.ck_linear_input_grad_mxfp8(dy, dtype, codes, scales, out, out_dtype, m, n, k, ws, need, None)

        _refused(lib, call(dy=None), "null")
        _refused(lib, call(out=None), "null")
        _refused(lib, call(dy=FAKE + 8), "aligned")
        _refused(lib, call(codes=FAKE + 16), "aligned")
        _refused(lib, call(dtype=5), "dtype")
        _refused(lib, call(out_dtype=5), "dtype")
        _refused(lib, call(k=40), "")
        _refused(lib, call(n=12), "")
        _refused(lib, call(ws=None), "null")
        _refused(lib, call(need=0), "workspace")


@pytest.mark.parametrize("shape", [(4, 64), (2, 3, 64), (64,)])
def test_shapes_under_tracing(shape):
    rows = 1
    for s in shape[:-1]:
        rows *= s
    ops = torch.ops.comfy_kitchen
    with FakeTensorMode():
        x = torch.empty(shape, device="cuda", dtype=torch.bfloat16)
        w = torch.empty(64, device="cuda", dtype=torch.bfloat16)
        y, mean, rstd, codes, scales = ops.layer_norm_forward_mxfp8(x, w, None, 1e-5, 0.0)
        assert y.shape == x.shape and mean.shape == rstd.shape == (rows,) and codes.shape == (rows, 64) and scales.shape == (128, 4)
        assert mean.dtype == torch.float32 and codes.dtype == torch.float8_e4m3fn and scales.dtype == torch.float8_e8m0fnu
        dx, dw, db = ops.layer_norm_backward_mxfp8(y, codes, scales, mean, rstd, w, 0.0, 1, 0)
        assert dx.shape == x.shape and dw.shape == db.shape == (1, 64) and dw.dtype == torch.float32
        assert ops.layer_norm_forward(x, None, None, 1e-5, 0.0)[0].dtype == x.dtype
        x2 = x.reshape(-1, 64)
        h, codes, scales = ops.gelu_mxfp8_forward(x2)
        assert h.shape == codes.shape == x2.shape and ops.gelu_mxfp8_backward(h, codes, scales).shape == x2.shape
        dy = torch.empty(rows, 24, device="cuda", dtype=torch.float16)
        dw, db = ops.linear_weight_grad_mxfp8(dy, codes, scales, 0, True)
        assert dw.shape == (24, 64) and db.shape == (24,) and dw.dtype == db.dtype == torch.float32
        wc, ws = torch.empty(24, 64, device="cuda", dtype=torch.float8_e4m3fn), torch.empty(128, 4, device="cuda", dtype=torch.float8_e8m0fnu)
        assert ops.linear_input_grad_mxfp8(dy, wc, ws, 1).shape == (rows, 64)


def test_traced_modules():
    """The public functions on traced tensors go through the dispatcher, whose operators carry the gradients."""
    with FakeTensorMode():
        mlp = ck.training.CheckpointedMLP(64, 96, device="cuda", dtype=torch.bfloat16)
        x = torch.empty(2, 5, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        y = mlp(x)
        assert y.shape == x.shape and y.requires_grad
        z = ck.layer_norm(x, torch.empty(2, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True), weight_offset=1.0, checkpoint=True)
        assert z.shape == x.shape and z.requires_grad


def test_refusals_without_a_gpu():
    x, w = torch.zeros(4, 64), torch.zeros(16, 64)
    codes, scales = torch.zeros(4, 64, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.zeros(128, 4, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    stats = torch.zeros(4)
    for call in (lambda: ck.layer_norm(x), lambda: ck.layer_norm(x, checkpoint=True), lambda: ck.layer_norm_forward(x),
                 lambda: ck.layer_norm_backward(x, x, stats, stats), lambda: ck.layer_norm_backward_mxfp8(x, codes, scales, stats, stats),
                 lambda: ck.gelu_checkpointed(x), lambda: ck.gelu_mxfp8_backward(x, codes, scales), lambda: ck.linear_weight_grad_mxfp8(x, codes, scales),
                 lambda: ck.linear_input_grad_mxfp8(torch.zeros(2, 4), codes, scales), lambda: ck.linear_checkpointed(x, w.requires_grad_())):
        with pytest.raises(ck.NoCapableBackendError):
            call()
    with pytest.raises(ValueError, match="multiple of 32"):
        ck.layer_norm(torch.zeros(4, 40), checkpoint=True)
    with pytest.raises(ValueError, match="multiple of 32"):
        ck.gelu_checkpointed(torch.zeros(()))
    with pytest.raises(ValueError, match="output features"):
        ck.linear_checkpointed(x, torch.zeros(12, 64))


def test_norm_backward_takes_a_weight_with_one_row_for_each_group(monkeypatch):
    """A weight whose first dimension is not the groups has its rows elsewhere than a group's number times its stride: refused before any launch."""
    from comfy_kitchen.backends import cuda

    monkeypatch.setattr(cuda, "load_library", lambda: None)  # nothing is launched, whatever is here
    with FakeTensorMode():
        dy, stats = torch.empty(8, 64, device="cuda"), torch.empty(8, device="cuda")
        codes = torch.empty(8, 64, device="cuda", dtype=torch.float8_e4m3fn)
        scales = torch.empty(128, 4, device="cuda", dtype=torch.float8_e8m0fnu)
        for shape in ((2, 2, 64), (1, 4, 64), (2, 1, 2, 64)):
            w = torch.empty(shape, device="cuda")
            for call in (lambda: cuda.layer_norm_backward(dy, dy, stats, stats, w, 0.0, 4),
                         lambda: cuda.layer_norm_backward_mxfp8(dy, codes, scales, stats, stats, w, 0.0, 4)):
                with pytest.raises(AssertionError, match="weight"):
                    call()


def test_gradients_take_operands_of_one_device(monkeypatch):
    """A kernel on one GPU cannot read another one's memory: operands that lie elsewhere are refused before any launch."""
    from comfy_kitchen.backends import cuda

    monkeypatch.setattr(cuda, "load_library", lambda: None)  # nothing is launched, whatever is here
    monkeypatch.setattr(cuda, "_host", None)
    with FakeTensorMode():
        def made(shape, dtype=torch.float32):
            return [torch.empty(shape, device=d, dtype=dtype) for d in ("cuda:0", "cuda:1")]

        dy, stats, w = made((8, 64)), made((8,)), made((64,))
        codes, scales = made((8, 64), torch.float8_e4m3fn), made((128, 4), torch.float8_e8m0fnu)
        for other in range(3):
            mean, rstd, weight = (t[i == other] for i, t in enumerate((stats, stats, w)))
            with pytest.raises(AssertionError, match="device"):
                cuda.layer_norm_backward(dy[0], dy[0], mean, rstd, weight)
        for c, s in ((codes[1], scales[0]), (codes[0], scales[1])):
            for call in (lambda: cuda.layer_norm_backward_mxfp8(dy[0], c, s, stats[0], stats[0]), lambda: cuda.gelu_mxfp8_backward(dy[0], c, s),
                         lambda: cuda.linear_weight_grad_mxfp8(dy[0], c, s), lambda: cuda.linear_input_grad_mxfp8(dy[0][:, :8], c, s)):
                with pytest.raises(AssertionError, match="device"):
                    call()


def test_only_the_results_carry_gradients(monkeypatch):
    """Statistics and copies have no gradient, and say so, instead of one of zeros: the operators' formulas over stand-ins for their kernels."""
    from comfy_kitchen import ops

    def stand_in(name, kwargs):
        if name.endswith("backward") or name.endswith("backward_mxfp8"):
            dy = kwargs["dy"]
            return 2 * dy if name.startswith("gelu") else (2 * dy, 3 * dy.sum(0, keepdim=True), 5 * dy.sum(0, keepdim=True))
        x = kwargs["x"].detach()
        copy = torch.zeros(x.shape, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.zeros(128, 4, dtype=torch.uint8).view(torch.float8_e8m0fnu)
        return (2 * x, *(() if name.startswith("gelu") else (x.mean(-1), x.std(-1))), *(copy if name.endswith("mxfp8") or name.startswith("gelu") else ()))

    monkeypatch.setattr(ops, "_impl", stand_in)
    x, w, b = (torch.ones(s, requires_grad=True) for s in ((4, 64), (64,), (64,)))
    op = torch.ops.comfy_kitchen
    for leaves, out in (((x, w, b), op.layer_norm_forward(x, w, b, 1e-5, 0.0)), ((x, w, b), op.layer_norm_forward_mxfp8(x, w, b, 1e-5, 0.0)),
                        ((x,), op.gelu_mxfp8_forward(x)), ((x, w), ck.layer_norm_forward(x, w))):
        assert out[0].requires_grad and not any(t.requires_grad for t in out[1:])
        grads = torch.autograd.grad(out[0], leaves, torch.ones_like(x))
        assert all(torch.equal(g, torch.full_like(t, c)) for g, t, c in zip(grads, leaves, (2, 12, 20)))
        if out[1].dtype == torch.float32:  # a loss of the result and a statistic: the result's part alone
            mixed = torch.autograd.grad((ck.layer_norm_forward(x, w)[0] + out[1].unsqueeze(1)).sum(), x)[0]
            assert torch.equal(mixed, torch.full_like(x, 2))
            with pytest.raises(RuntimeError, match="does not require grad"):
                torch.autograd.grad(out[1].sum(), x)
