"""RMS norm, clipping and the experts' products where there is no GPU: shapes under tracing, refusals of tensors elsewhere, the C entry points' checks."""
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
BIG = 1 << 40


@pytest.fixture(scope="module")
def lib():
    spec = importlib.util.spec_from_file_location("ck_build", os.path.join(PKG_DIR, "build.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    lib = ctypes.CDLL(mod.build())
    from comfy_kitchen.backends import cuda

    for name, types in cuda._SIGNATURES.items():
        getattr(lib, name).argtypes = types
    for name, kind in cuda._RESTYPE.items():
        getattr(lib, name).restype = kind
    lib.ck_last_error.restype = ctypes.c_char_p
    return lib


def _refused(lib, call, said):
    assert call != 0
    assert said in lib.ck_last_error().decode(), lib.ck_last_error()


def _rms(lib, **kw):
    a = dict(x=FAKE, dtype=2, rows=4, cols=64, inner=4, outer=0, stride=64, residual=None, r_inner=4, r_outer=0, r_stride=64, w=None, pdtype=2, offset=0.0,
             eps=1e-6, y=FAKE, h=None, rstd=FAKE, codes=None, scales=None, stream=None)
    a.update(kw)
    return lib.ck_rms_norm_forward(*a.values())


def test_rms_norm_arguments(lib):
    _refused(lib, _rms(lib, x=None), "null")
    _refused(lib, _rms(lib, y=None), "null")
    _refused(lib, _rms(lib, codes=FAKE, scales=FAKE), "null")  # both kinds of results
    _refused(lib, _rms(lib, y=None, codes=FAKE), "null")
    _refused(lib, _rms(lib, residual=FAKE), "belong together")
    _refused(lib, _rms(lib, h=FAKE), "belong together")
    _refused(lib, _rms(lib, y=None, codes=FAKE, scales=FAKE, cols=40, stride=40), "multiple of 32")
    _refused(lib, _rms(lib, y=None, codes=FAKE + 16, scales=FAKE), "boundaries")
    _refused(lib, _rms(lib, y=None, codes=FAKE, scales=FAKE + 2), "boundaries")
    _refused(lib, _rms(lib, y=None, codes=FAKE, scales=FAKE, stride=72), "boundaries")
    _refused(lib, _rms(lib, dtype=7), "dtype")
    _refused(lib, _rms(lib, pdtype=1), "weight")
    _refused(lib, _rms(lib, rows=0), "shape")
    _refused(lib, _rms(lib, cols=0), "shape")
    _refused(lib, _rms(lib, rows=1 << 31), "shape")
    _refused(lib, _rms(lib, cols=1 << 31), "shape")
    _refused(lib, _rms(lib, inner=0), "strides")
    _refused(lib, _rms(lib, inner=3), "strides")


def test_rms_norm_backward_arguments(lib):
    size = lib.ck_rms_norm_backward_workspace_bytes
    assert size(2, 4, 64) >= 256 and size(0, 1 << 20, 4096) >= 4096 * 4
    assert size(2, 0, 64) == 0 and size(2, 4, 0) == 0 and size(9, 4, 64) == 0

    def call(dy=FAKE, dtype=2, rows=4, cols=64, inner=4, outer=0, stride=64, h=FAKE, rstd=FAKE, w=None, pdtype=2, dx=FAKE, dw=None, ws=FAKE,
             need=BIG):
        return lib.ck_rms_norm_backward(dy, dtype, rows, cols, inner, outer, stride, h, rows, 0, cols, None, rows, 0, cols, rstd, w, pdtype, 0.0, dx, dw, ws,
                                        need, None)

    for name in ("dy", "h", "rstd", "dx"):
        _refused(lib, call(**{name: None}), "null")
    _refused(lib, call(dtype=5), "dtype")
    _refused(lib, call(pdtype=5), "weight")
    _refused(lib, call(rows=0, inner=1), "shape")
    _refused(lib, call(inner=0), "strides")
    _refused(lib, call(inner=3), "strides")
    _refused(lib, call(dw=FAKE, ws=None), "workspace")
    _refused(lib, call(dw=FAKE, ws=FAKE + 4), "workspace")
    _refused(lib, call(dw=FAKE, need=255), "workspace")


def test_clip_arguments(lib):
    size = lib.ck_clip_grad_norm_workspace_bytes
    assert size(0) > 0 and size(1025) > size(1024) and size(-1) == 0 and size((1 << 24) + 1) == 0

    def call(grads, counts=None, dtypes=None, max_norm=1.0, norm=FAKE, ws=FAKE, need=BIG, n=None):
        count = len(grads) if n is None else n
        counts, dtypes = counts or [16] * len(grads), dtypes or [0] * len(grads)
        return lib.ck_clip_grad_norm((ctypes.c_void_p * len(grads))(*grads), (ctypes.c_int64 * len(grads))(*counts), (ctypes.c_int * len(grads))(*dtypes), count,
                                     max_norm, norm, ws, need, None)

    _refused(lib, call([FAKE], norm=None), "null")
    _refused(lib, call([FAKE], ws=None), "null")
    _refused(lib, lib.ck_clip_grad_norm(None, None, None, 1, 1.0, FAKE, FAKE, BIG, None), "null")
    _refused(lib, call([FAKE], n=-1), "tensors")
    _refused(lib, call([FAKE], n=(1 << 24) + 1), "tensors")
    _refused(lib, call([FAKE], need=16), "workspace")
    _refused(lib, call([FAKE], max_norm=float("nan")), "no number")
    _refused(lib, call([FAKE], dtypes=[4]), "not supported")
    _refused(lib, call([FAKE], counts=[-1]), "not supported")
    _refused(lib, call([None]), "not supported")
    _refused(lib, call([FAKE + 2]), "not supported")
    _refused(lib, call([FAKE + 1], dtypes=[2]), "not supported")
    _refused(lib, call([FAKE, FAKE]), "overlap")
    _refused(lib, call([FAKE + 64, FAKE + 2048, FAKE + 60], counts=[4, 4, 2]), "overlap")  # the third reaches into the first


def test_grouped_arguments(lib):
    size = lib.ck_grouped_mm_mxfp8_workspace_bytes
    assert size(1, 8, 64, 4) > size(0, 8, 64, 4) > 0
    assert size(0, 0, 64, 4) == 0 and size(0, 8, 0, 4) == 0 and size(0, 8, 64, 0) == 0 and size(0, 8, 64, 1025) == 0
    grad = lib.ck_grouped_input_grad_mxfp8_workspace_bytes
    assert grad(2, 8, 64, 64, 4) > 0 and grad(9, 8, 64, 64, 4) == 0 and grad(2, 8, 64, 64, 1025) == 0 and grad(2, 0, 64, 64, 4) == 0

    base = dict(x=FAKE, dtype=2, sx=FAKE, w=FAKE, sw=FAKE, ends=FAKE, bias=None, bdtype=0, out=FAKE, odtype=2, m=8, n=64, k=64, e=4, ws=FAKE, need=BIG)

    def mm(**kw):
        a = {**base, **kw}
        return lib.ck_grouped_mm_mxfp8(a["x"], a["w"], a["sx"], a["sw"], a["ends"], a["bias"], a["bdtype"], a["out"], a["odtype"], a["m"], a["n"], a["k"], a["e"],
                                       a["ws"], a["need"], None)

    def linear(**kw):
        a = {**base, **kw}
        return lib.ck_grouped_linear_mxfp8(a["x"], a["dtype"], a["w"], a["sw"], a["ends"], a["bias"], a["bdtype"], a["out"], a["odtype"], a["m"], a["n"], a["k"],
                                           a["e"], a["ws"], a["need"], None)

    def input_grad(**kw):
        a = {**base, **kw}
        return lib.ck_grouped_input_grad_mxfp8(a["x"], a["dtype"], a["w"], a["sw"], a["ends"], a["out"], a["odtype"], a["m"], a["n"], a["k"], a["e"], a["ws"],
                                               a["need"], None)

    for call in (mm, linear, input_grad):
        for name in ("x", "w", "sw", "ends", "out", "ws"):
            _refused(lib, call(**{name: None}), "null")
        for name in ("x", "w", "sw", "out"):
            _refused(lib, call(**{name: FAKE + 8}), "aligned")
        _refused(lib, call(odtype=5), "dtype")
        for bad in ({"m": 0}, {"n": 0}, {"k": 0}, {"m": 1 << 30}, {"n": 1 << 30}, {"k": 1 << 30}):
            _refused(lib, call(**bad), "shape")
        for bad in ({"e": 0}, {"e": 1025}, {"e": -1}):
            _refused(lib, call(**bad), "group")
        for bad in ({"k": 48}, {"n": 12}):
            _refused(lib, call(**bad), "multiple")
        _refused(lib, call(need=64), "workspace")
    _refused(lib, mm(sx=None), "null")
    for call in (linear, input_grad):
        _refused(lib, call(dtype=5), "dtype")
    for call in (mm, linear):
        _refused(lib, call(bias=FAKE, bdtype=4), "dtype")


@pytest.mark.parametrize("shape", [(4, 64), (2, 3, 64), (64,)])
def test_shapes_under_tracing(shape):
    rows = 1
    for s in shape[:-1]:
        rows *= s
    ops = torch.ops.comfy_kitchen
    with FakeTensorMode():
        x = torch.empty(shape, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        w = torch.empty(64, device="cuda", requires_grad=True)
        y = ck.rms_norm(x, w)
        assert y.shape == x.shape and y.dtype == x.dtype and y.requires_grad
        y, h = ck.rms_norm(x, w, x.detach(), weight_offset=1.0)
        assert y.shape == h.shape == x.shape and y.requires_grad and h.requires_grad
        codes, scales = ck.rms_norm_mxfp8(x.detach(), w.detach())
        assert codes.shape == (rows, 64) and scales.shape == (128, 4) and codes.dtype == torch.float8_e4m3fn and scales.dtype == torch.float8_e8m0fnu
        y, h, rstd = ck.rms_norm_forward(x.detach(), w.detach())
        assert y.shape == x.shape and h is None and rstd.shape == (rows,) and rstd.dtype == torch.float32
        dx, dw = ck.rms_norm_backward(y, x.detach(), rstd, w.detach())
        assert dx.shape == x.shape and dw.shape == (64,) and dw.dtype == torch.float32
        codes, scales = torch.empty(5, 24, 64, device="cuda", dtype=torch.float8_e4m3fn), torch.empty(5, 128, 4, device="cuda", dtype=torch.float8_e8m0fnu)
        ends = torch.empty(5, device="cuda", dtype=torch.int32)
        x2 = x.reshape(-1, 64)
        out = ck.grouped_linear_mxfp8(x2, codes, scales, ends)
        assert out.shape == (rows, 24) and out.dtype == x.dtype and out.requires_grad
        assert ck.grouped_input_grad_mxfp8(out.detach(), codes, scales, ends, torch.float32).shape == (rows, 64)
        q, s = torch.empty(rows, 64, device="cuda", dtype=torch.float8_e4m3fn), torch.empty(128, 4, device="cuda", dtype=torch.float8_e8m0fnu)
        out = ck.grouped_mm_mxfp8(q, codes, s, scales, ends, out_dtype=torch.float16)
        assert out.shape == (rows, 24) and out.dtype == torch.float16
        assert ops.grad_norm([x.detach(), w.detach()]).shape == ()


def test_traced_modules():
    """The public functions on traced tensors go through the dispatcher, whose operators carry the gradients."""
    with FakeTensorMode():
        mlp = ck.training.CheckpointedMLP(64, 96, device="cuda", dtype=torch.bfloat16, norm="rms")
        x = torch.empty(2, 5, 64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        y = mlp(x)
        assert y.shape == x.shape and y.requires_grad
        z = ck.norms.RMSNorm(64, device="cuda", dtype=torch.bfloat16)(x)
        assert z.shape == x.shape and z.requires_grad


def test_refusals_without_a_gpu():
    x = torch.zeros(4, 64)
    codes, scales = torch.zeros(2, 16, 64, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.zeros(2, 128, 4, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    ends = torch.tensor([2, 4], dtype=torch.int32)
    w = torch.nn.Parameter(torch.zeros(4))
    w.grad = torch.ones(4)
    for call in (lambda: ck.rms_norm(x), lambda: ck.rms_norm(x.clone().requires_grad_()), lambda: ck.rms_norm_forward(x, x[0]), lambda: ck.rms_norm_mxfp8(x),
                 lambda: ck.rms_norm_backward(x, x, torch.zeros(4)), lambda: ck.grad_norm([x]), lambda: ck.clip_grad_norm_([w], 1.0),
                 lambda: ck.grouped_linear_mxfp8(x, codes, scales, ends), lambda: ck.grouped_input_grad_mxfp8(x[:, :16].contiguous(), codes, scales, ends),
                 lambda: ck.grouped_mm_mxfp8(codes[0, :4], codes, scales[0], scales, ends)):
        with pytest.raises(ck.NoCapableBackendError):
            call()
    with pytest.raises(ValueError, match="max_norm"):
        ck.clip_grad_norm_([w], -1.0)
    with pytest.raises(ValueError, match="max_norm"):
        ck.clip_grad_norm_([w], float("nan"))
    with pytest.raises(ValueError, match="norm is"):
        ck.training.CheckpointedMLP(64, 96, norm="batch")
    assert torch.equal(w.grad, torch.ones(4))
