"""The training layers as a user has them: linear layers over the gradient products, modules, the MLP as a chain of the operators.

A layer's gradients are the operators' own (checked against 64 bits in their own tests), so what is a composition has to give the
same bits as the operators called by hand.  The whole MLP is held against its gradients in 64 bits with the values that stand in the copies: in fp32
a chain of at most seven results, each within 1e-5 of its norm (sums of at most 512 products of fp32 numbers, 2^-24 each, and the norm's and GELU's
few roundings), whose errors pass through the layers behind them without growing: 1e-4.
"""
from __future__ import annotations

import sys

import pytest
import torch
import torch.nn.functional as F
from conftest import PKG_DIR

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def ck(cuda_device):
    import comfy_kitchen

    assert comfy_kitchen.list_backends()["cuda"]["available"]
    return comfy_kitchen


def _made(shape, dtype, seed, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,n", [((1, 32), 8), ((77, 160), 72), ((2, 3, 64), 24), ((96,), 16), ((300, 1024), 512)])
@pytest.mark.parametrize("bias", [False, True])
def test_linear_with_a_dense_weight(ck, dtype, shape, n, bias):
    x, w = _made(shape, dtype, 1).requires_grad_(), _made((n, shape[-1]), dtype, 2, 0.1).requires_grad_()
    b = _made((n,), dtype, 3).requires_grad_() if bias else None
    y = ck.linear_checkpointed(x, w, b)
    assert torch.equal(y, F.linear(x.reshape(-1, shape[-1]), w, b).view(*shape[:-1], n))
    dy = _made(y.shape, dtype, 4)
    dx, dw, *db = torch.autograd.grad(y, (x, w, b) if bias else (x, w), dy)
    codes, scales = ck.quantize_mxfp8(x.detach().reshape(-1, shape[-1]))
    want_dw, want_db = ck.linear_weight_grad_mxfp8(dy.reshape(-1, n), codes, scales, dtype, bias)
    assert torch.equal(dw, want_dw) and (not bias or torch.equal(db[0], want_db))
    assert torch.equal(dx, (dy.reshape(-1, n) @ w).view(shape))
    # an E4M3 number is within 2^-4 of the value (or 2^-10 of the block's largest number, below its normal ones)
    d64, x64 = dy.reshape(-1, n).double(), x.detach().reshape(-1, shape[-1]).double()
    off = (dw.double() - d64.t() @ x64).norm()
    assert off <= (2.0**-4 + 2.0**-7) * torch.linalg.matrix_norm(d64, 2) * x64.norm()


@pytest.mark.parametrize("dtype", DTYPES[:2])
@pytest.mark.parametrize("rows,n,k", [(40, 64, 96), (5, 40, 100), (130, 129, 257), (1, 512, 1024)])
@pytest.mark.parametrize("bias", [False, True])
def test_linear_with_a_frozen_mxfp8_weight(ck, dtype, rows, n, k, bias):
    from comfy_kitchen.tensor import QuantizedTensor

    x = _made((rows, k), dtype, 5).requires_grad_()
    w = QuantizedTensor.from_float(_made((n, k), dtype, 6, 0.1), "TensorCoreMXFP8Layout")
    b = _made((n,), dtype, 7).requires_grad_() if bias else None
    y = ck.linear_checkpointed(x, w, b)
    xq = QuantizedTensor.from_float(x.detach(), "TensorCoreMXFP8Layout")
    every = None if b is None else F.pad(b.detach(), (0, w._qdata.shape[0] - n))  # the codes' rows are padded to 32
    want = ck.scaled_mm_mxfp8(xq._qdata, w._qdata, xq._params.scale, w._params.scale, bias=every, out_dtype=dtype)[:rows, :n]
    assert y.shape == (rows, n) and torch.equal(y.detach(), want)
    dy = _made(y.shape, dtype, 8)
    dx, *db = torch.autograd.grad(y, (x, b) if bias else (x,), dy)
    w64 = w.dequantize().double()
    value, magnitude = dy.double() @ w64, dy.double().abs() @ w64.abs()
    limit = (n / 8 + 64) * 2.0**-22 * magnitude + {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}[dtype] * (value.abs() + 2.0**-12 * magnitude) + 2.0**-24
    assert ((dx.double() - value).abs() <= limit).all()
    if bias:
        assert torch.equal(db[0], dy.sum(0))


def test_linear_keeps_the_copy_only(ck):
    x, w = _made((256, 512), torch.bfloat16, 9).requires_grad_(), _made((64, 512), torch.bfloat16, 10).requires_grad_()
    seen = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: seen.append(t) or t, lambda t: t):
        ck.linear_checkpointed(x, w)
    assert sorted(str(t.dtype) for t in seen) == ["torch.bfloat16", "torch.float8_e4m3fn", "torch.float8_e8m0fnu"]
    assert [t for t in seen if t.dtype == torch.bfloat16][0].data_ptr() == w.data_ptr()
    seen.clear()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: seen.append(t) or t, lambda t: t):
        ck.linear_checkpointed(x, w.detach())  # no gradient of the weight: nothing of x
    assert [t.data_ptr() for t in seen] == [w.data_ptr()]


def test_gradients_that_are_not_wanted(ck):
    x, w, b = _made((40, 64), torch.float32, 11), _made((16, 64), torch.float32, 12), _made((16,), torch.float32, 13)
    dy = _made((40, 16), torch.float32, 14)
    full = torch.autograd.grad(ck.linear_checkpointed(x.clone().requires_grad_(), w.requires_grad_(), b.requires_grad_()), (w, b), dy)
    only_w = torch.autograd.grad(ck.linear_checkpointed(x, w, b.detach()), w, dy)
    only_b = torch.autograd.grad(ck.linear_checkpointed(x, w.detach(), b), b, dy)
    assert torch.equal(full[0], only_w[0])
    torch.testing.assert_close(only_b[0], full[1], rtol=1e-5, atol=1e-5)
    with torch.no_grad():
        assert not ck.linear_checkpointed(x, w, b).requires_grad and not ck.gelu_checkpointed(x).requires_grad


@pytest.mark.parametrize("shape", [(0, 64), (2, 0, 64)])
def test_no_tokens(ck, shape):
    from comfy_kitchen.tensor import QuantizedTensor

    mlp = ck.training.CheckpointedMLP(64, 96, device="cuda")
    x = torch.empty(shape, device="cuda", requires_grad=True)
    mlp(x).sum().backward()
    assert x.grad.shape == shape and all((p.grad == 0).all() for p in mlp.parameters())
    frozen = QuantizedTensor.from_float(_made((96, 64), torch.float32, 42), "TensorCoreMXFP8Layout")
    y = ck.linear_checkpointed(x, frozen)
    assert y.shape == (*shape[:-1], 96) and torch.autograd.grad(y.sum(), x)[0].shape == shape


def test_more_than_2_31_elements(ck):
    x = _made((66000, 32768), torch.bfloat16, 43)
    last = x[-128:]
    y, mean, rstd, codes, scales = ck.layer_norm_forward_mxfp8(x)
    want = ck.layer_norm_forward_mxfp8(last.clone())
    assert torch.equal(y[-128:], want[0]) and torch.equal(codes[-128:].view(torch.uint8), want[3].view(torch.uint8))
    dx = ck.layer_norm_backward_mxfp8(x, codes, scales, mean, rstd)[0]
    held = ck.dequantize_mxfp8(want[3], want[4], torch.float32).double()
    h = (held - want[1].double().unsqueeze(1)) * want[2].double().unsqueeze(1)
    d = last.double()
    exact = want[2].double().unsqueeze(1) * (d - d.mean(1, keepdim=True) - h * (d * h).mean(1, keepdim=True))
    assert (dx[-128:].double() - exact).norm() <= 2.0**-8 * exact.norm()
    del y, dx
    u, gelu_codes, _ = ck.gelu_mxfp8_forward(x)
    assert torch.equal(gelu_codes[-128:].view(torch.uint8), want[3].view(torch.uint8)) and torch.equal(u[-128:], ck.gelu_mxfp8_forward(last.clone())[0])


def test_expanded_gradient(ck):
    """The gradient of a sum is one number for all elements, with strides of zero."""
    x, w = _made((40, 64), torch.float32, 15), _made((16, 64), torch.float32, 16).requires_grad_()
    ck.linear_checkpointed(x, w).sum().backward()
    held = ck.dequantize_mxfp8(*ck.quantize_mxfp8(x), torch.float32).double()
    want = held.sum(0).expand(16, 64)
    assert ((w.grad.double() - want).abs() <= 2.0**-16 * held.abs().sum(0)).all()


def test_under_autocast(ck):
    x, layer = _made((40, 64), torch.float32, 17).requires_grad_(), ck.training.CheckpointedLinear(64, 16, device="cuda")
    with torch.autocast("cuda", torch.bfloat16):
        y = layer(x)
    assert y.dtype == torch.bfloat16
    y.float().sum().backward()
    assert x.grad.dtype == layer.weight.grad.dtype == layer.bias.grad.dtype == torch.float32
    assert torch.equal(layer.bias.grad, torch.full((16,), 40.0, device="cuda"))


def _mlp_by_hand(ck, mlp, x, dy):
    """The module's forward and backward passes as calls of the operators."""
    p = {n: t.detach() for n, t in mlp.named_parameters()}
    normed, mean, rstd, nc, ns = ck.layer_norm_forward_mxfp8(x, p["norm.weight"], p["norm.bias"], mlp.norm.eps)
    c1, s1 = ck.quantize_mxfp8(normed)
    u = F.linear(normed, p["fc1.weight"], p["fc1.bias"])
    h, gc, gs = ck.gelu_mxfp8_forward(u)
    c2, s2 = ck.quantize_mxfp8(h)
    y = x + F.linear(h, p["fc2.weight"], p["fc2.bias"])
    dw2, db2 = ck.linear_weight_grad_mxfp8(dy, c2, s2, bias_grad=True)
    du = ck.gelu_mxfp8_backward(dy @ p["fc2.weight"], gc, gs)
    dw1, db1 = ck.linear_weight_grad_mxfp8(du, c1, s1, bias_grad=True)
    dx, dw, db = ck.layer_norm_backward_mxfp8(du @ p["fc1.weight"], nc, ns, mean, rstd, p["norm.weight"])
    grads = {"fc2.weight": dw2, "fc2.bias": db2, "fc1.weight": dw1, "fc1.bias": db1, "norm.weight": dw[0], "norm.bias": db[0]}
    copies = [ck.dequantize_mxfp8(c, s, torch.float32).double() for c, s in ((nc, ns), (c1, s1), (gc, gs), (c2, s2))]
    return y, dx + dy, grads, copies


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,features,hidden", [(1, 32, 64), (77, 128, 512), (300, 256, 512)])
def test_mlp(ck, dtype, rows, features, hidden):
    torch.manual_seed(0)
    mlp = ck.training.CheckpointedMLP(features, hidden, device="cuda", dtype=dtype)
    with torch.no_grad():
        mlp.norm.weight.copy_(_made((features,), dtype, 20, 0.2) + 1)
        mlp.norm.bias.copy_(_made((features,), dtype, 21, 0.2))
    x = _made((rows, features), dtype, 22).requires_grad_()
    dy = _made((rows, features), dtype, 23)
    y = mlp(x)
    y.backward(dy)
    want_y, want_dx, grads, copies = _mlp_by_hand(ck, mlp, x.detach(), dy)
    assert torch.equal(y.detach(), want_y) and torch.equal(x.grad, want_dx)
    for name, p in mlp.named_parameters():
        assert p.grad.dtype == dtype and torch.equal(p.grad, grads[name]), name
    if dtype != torch.float32:
        return
    # in 64 bits from the same copies
    p = {n: t.detach().double() for n, t in mlp.named_parameters()}
    x64, d64 = x.detach().double(), dy.double()
    mean, var = x64.mean(1, keepdim=True), x64.var(1, keepdim=True, unbiased=False)
    rstd = (var + mlp.norm.eps).rsqrt()
    kept_x, kept_normed, kept_u, kept_h = copies
    leaf = kept_u.clone().requires_grad_()
    (slope,) = torch.autograd.grad(F.gelu(leaf, approximate="tanh").sum(), leaf)
    du = (d64 @ p["fc2.weight"]) * slope
    g = du @ p["fc1.weight"]
    hat, gf = (kept_x - mean) * rstd, g * p["norm.weight"]
    dx = rstd * (gf - gf.mean(1, keepdim=True) - hat * (gf * hat).mean(1, keepdim=True)) + d64
    want = {"fc2.weight": d64.t() @ kept_h, "fc2.bias": d64.sum(0), "fc1.weight": du.t() @ kept_normed, "fc1.bias": du.sum(0),
            "norm.weight": (g * hat).sum(0), "norm.bias": g.sum(0)}
    for name, t in mlp.named_parameters():
        assert (t.grad.double() - want[name]).norm() <= 1e-4 * want[name].norm(), name
    assert (x.grad.double() - dx).norm() <= 1e-4 * dx.norm()


@pytest.mark.parametrize("dtype", DTYPES)
def test_same_without_the_native_host_half(ck, dtype, monkeypatch):
    from comfy_kitchen.backends import cuda as backend

    torch.manual_seed(1)
    mlp = ck.training.CheckpointedMLP(64, 160, device="cuda", dtype=dtype)
    x, dy = _made((2, 9, 64), dtype, 24).requires_grad_(), _made((2, 9, 64), dtype, 25)
    leaves = (x, *mlp.parameters())
    scale, shift = _made((2, 64), dtype, 26).requires_grad_(), _made((2, 64), dtype, 27).requires_grad_()

    def both():
        with torch.no_grad():
            quiet = (ck.layer_norm(x, scale, shift, weight_offset=1.0), ck.gelu_checkpointed(x), mlp(x))
        y = mlp(x)
        z = ck.layer_norm(x, scale, shift, weight_offset=1.0)
        return (*quiet, y.detach(), z.detach(), *torch.autograd.grad(y, leaves, dy), *torch.autograd.grad(z, (x, scale, shift), dy))

    native = both()
    assert torch.equal(native[0], native[4]) and torch.equal(native[2], native[3])
    with monkeypatch.context() as m:
        m.setattr(backend, "_host", None)
        plain = both()
    assert all(torch.equal(a, b) for a, b in zip(native, plain))


def test_modulated_and_strided_norm_on_another_stream(ck):
    """The text tokens of a longer buffer, each sample with a scale and shift of its own, on a stream that is not the default one."""
    wide = _made((3, 40, 256), torch.bfloat16, 28)
    scale, shift = _made((3, 256), torch.bfloat16, 29, 0.2).requires_grad_(), _made((3, 256), torch.bfloat16, 30).requires_grad_()
    x = wide[:, :11].requires_grad_()
    dy = _made((3, 11, 256), torch.bfloat16, 31)
    here = torch.autograd.grad(ck.layer_norm(x, scale, shift, weight_offset=1.0, checkpoint=True), (x, scale, shift), dy)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        there = torch.autograd.grad(ck.layer_norm(x, scale, shift, weight_offset=1.0, checkpoint=True), (x, scale, shift), dy)
    torch.cuda.current_stream().wait_stream(stream)
    assert all(torch.equal(a, b) for a, b in zip(here, there))


def test_compiled(ck):
    torch.manual_seed(2)
    mlp = ck.training.CheckpointedMLP(64, 96, device="cuda", dtype=torch.bfloat16)
    x, dy = _made((20, 64), torch.bfloat16, 32).requires_grad_(), _made((20, 64), torch.bfloat16, 33)
    leaves = (x, *mlp.parameters())
    eager = torch.autograd.grad(mlp(x), leaves, dy)
    traced = torch.autograd.grad(torch.compile(mlp, backend="aot_eager")(x), leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip(eager, traced))


def test_recomputed_activations(ck):
    """Inside torch's own checkpointing, which runs the forward pass again."""
    from torch.utils.checkpoint import checkpoint

    torch.manual_seed(3)
    mlp = ck.training.CheckpointedMLP(64, 96, device="cuda")
    x, dy = _made((20, 64), torch.float32, 34).requires_grad_(), _made((20, 64), torch.float32, 35)
    leaves = (x, *mlp.parameters())
    plain = torch.autograd.grad(mlp(x), leaves, dy)
    again = torch.autograd.grad(checkpoint(mlp, x, use_reentrant=False), leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip(plain, again))


def test_the_example(ck):
    if PKG_DIR not in sys.path:
        sys.path.insert(0, PKG_DIR)
    import train_mlp

    said = []
    ours = train_mlp.run(256, 128, 512, 2, 12, report=said.append)
    dense = train_mlp.run(256, 128, 512, 2, 12, dense=True, report=said.append)
    assert len(said) == 2 and ours["losses"][-1] < ours["losses"][0]
    assert abs(ours["losses"][0] - dense["losses"][0]) <= 0.02 * dense["losses"][0]  # the same forward pass up to bf16's roundings
    assert ours["kept_bytes"] < 0.7 * dense["kept_bytes"]


def test_strict_mode_reports_a_wait_that_gave_up(ck, monkeypatch):
    """The status word is set from the host here; no kernel is made to fail."""
    from comfy_kitchen.backends import cuda as backend

    lib = backend.load_library()
    x, w = _made((600, 64), torch.bfloat16, 44).requires_grad_(), _made((16, 64), torch.bfloat16, 45).requires_grad_()
    codes, scales = ck.quantize_mxfp8(x.detach())
    dy = _made((600, 16), torch.bfloat16, 46)
    backend.check_device_status("clean start")
    monkeypatch.setenv("CK_STRICT", "1")
    for call in (lambda: ck.layer_norm(x), lambda: ck.layer_norm(x.detach()), lambda: ck.layer_norm(x, checkpoint=True),
                 lambda: ck.linear_weight_grad_mxfp8(dy, codes, scales), lambda: ck.linear_input_grad_mxfp8(x.detach(), *ck.quantize_mxfp8(w.detach().t().contiguous()
                                                                                                           .repeat(1, 2)))):
        call()
        assert lib.ck_debug_set_gemm_status(1) == 0
        with pytest.raises(RuntimeError, match="gave up"):
            call()
    monkeypatch.setenv("CK_STRICT", "0")
    backend.check_device_status("cleared")


def test_refusals(ck):
    from comfy_kitchen.tensor import QuantizedTensor

    x = _made((4, 64), torch.bfloat16, 36).requires_grad_()
    with pytest.raises(ValueError, match="input features"):
        ck.linear_checkpointed(x[:, :40], _made((16, 40), torch.bfloat16, 37))
    with pytest.raises(ValueError, match="output features"):
        ck.linear_checkpointed(x, _made((12, 64), torch.bfloat16, 37))
    with pytest.raises(ValueError, match="input"):
        ck.linear_checkpointed(x, _made((16, 96), torch.bfloat16, 37))
    with pytest.raises(ValueError, match="float32"):
        ck.linear_checkpointed(x, _made((16, 64), torch.float32, 37))
    nv = QuantizedTensor.from_float(_made((64, 64), torch.bfloat16, 38), "TensorCoreNVFP4Layout")
    with pytest.raises(ValueError, match="MXFP8"):
        ck.linear_checkpointed(x, nv)
    frozen = QuantizedTensor.from_float(_made((64, 64), torch.bfloat16, 39), "TensorCoreMXFP8Layout")
    with pytest.raises(ValueError, match="MXFP8"):
        ck.linear_checkpointed(x, frozen.t())
    with pytest.raises(ValueError, match="last dimension"):
        ck.training.CheckpointedLayerNorm((4, 64), device="cuda", dtype=torch.bfloat16)(x)
    with pytest.raises(ValueError, match="rows of 32"):
        ck.training.CheckpointedLayerNorm(32, elementwise_affine=False)(x)
    with pytest.raises(RuntimeError):  # no gradients of gradients
        w = _made((16, 64), torch.bfloat16, 40).requires_grad_()
        (g,) = torch.autograd.grad(ck.linear_checkpointed(x, w), w, _made((4, 16), torch.bfloat16, 41).requires_grad_(), create_graph=True)
        g.sum().backward()
