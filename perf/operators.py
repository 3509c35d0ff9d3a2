"""Cases of the training operators: layer norm, 8-bit activation checkpoints and the gradients that read them.

A case is a dict of plain values.  ``kind`` names the operator:

* ``norm``         ``ck.layer_norm`` in inference: one pass over the rows
* ``norm_step``    ``ck.layer_norm`` and its backward pass, with or without an MXFP8 copy of the input in between
* ``gelu_step``    ``ck.gelu_checkpointed`` and its backward pass from the MXFP8 copy of its input
* ``weight_grad``  ``ck.linear_weight_grad_mxfp8``: a linear's weight and bias gradient from the MXFP8 copy of its input
* ``input_grad``   ``ck.linear_input_grad_mxfp8``: a linear's input gradient through its MXFP8 weight

``m`` counts tokens, ``k`` features (``weight_grad`` and ``input_grad``: input features, ``n`` output features), ``groups`` the samples
that have a scale and a shift of their own (0: one learned weight and bias).  Sizes are those of the MMDiT-shaped stack
and of the benchmark: hidden 3072, MLP 12288, 512 text and 4096 image tokens, batch up to 8; the others are generic.

An MXFP8 matrix is held as the package holds it: E4M3 codes ``[rows, cols]`` and one E8M0 byte for 32 of a row, in tiles of 128 rows
by 4 blocks (512 bytes: 32 rows of 16, four rows 32 apart in each).
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

_PACKAGE = os.path.join(os.getcwd(), "comfy-kitchen_b200")
if _PACKAGE not in sys.path:
    sys.path.insert(0, _PACKAGE)

DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-5
BLOCK = 32
LARGEST_STEP = 36864 * 3072  # elements of the largest listed norm
LARGEST_GELU = 4608 * 12288
LARGEST_PRODUCT = 4608 * 12288 * 3072  # multiply-adds of the largest listed product


def _case(kind, m, k, dtype, n=0, groups=0, checkpoint=False, sliced=False, out="", bias=True, **name):
    return {**name, "kind": kind, "m": m, "n": n, "k": k, "dtype": dtype, "groups": groups, "checkpoint": checkpoint, "sliced": sliced,
            "out": out or dtype, "bias": bias}


def listed():
    return [
        # one token on its way through a served model: latency
        _case("norm", 1, 3072, "bf16", name="norm_one_token"),
        # rows of an MLP's width, half precision, no multiple of anything in tokens
        _case("norm", 577, 12288, "fp16", name="norm_wide_rows_fp16"),
        # modulated norm of the text stream, batch of 8: the text part of a buffer that holds text and image tokens
        _case("norm_step", 4096, 3072, "bf16", groups=8, sliced=True, name="norm_step_text_slice"),
        # modulated norm over all tokens of a batch of 8, the input kept in 8 bits
        _case("norm_step", 36864, 3072, "bf16", groups=8, checkpoint=True, name="norm_step_batch_checkpoint"),
        # odd width, odd rows, full precision: a small model's learned norm
        _case("norm_step", 1003, 769, "fp32", name="norm_step_odd_fp32"),
        # a prompt's hidden tensor in half precision
        _case("gelu_step", 77, 4096, "fp16", name="gelu_step_prompt_fp16"),
        # the MLP's hidden tensor over image and text tokens of one sample
        _case("gelu_step", 4608, 12288, "bf16", name="gelu_step_mlp"),
        # first MLP projection of one sample, gradients accumulated in fp32
        _case("weight_grad", 4608, 3072, "bf16", n=12288, out="fp32", name="weight_grad_mlp"),
        # few tokens, half precision: the result's write counts
        _case("weight_grad", 77, 2048, "fp16", n=1024, name="weight_grad_prompt_fp16"),
        # second MLP projection's frozen weight over the tokens of one sample
        _case("input_grad", 4608, 12288, "bf16", n=3072, bias=False, name="input_grad_mlp"),
        # modulation vectors of a batch of 8 through a frozen weight: the weight's read counts
        _case("input_grad", 8, 3072, "bf16", n=12288, bias=False, name="input_grad_few_rows"),
        # ragged tokens, full-precision gradients
        _case("input_grad", 333, 2048, "fp32", n=1536, bias=False, name="input_grad_ragged_fp32"),
    ]


def _spread(rng, lo, hi, step=1):
    """A multiple of ``step`` in [lo, hi], uniform over the logarithm."""
    v = lo * (hi / lo) ** rng.random()
    return min(hi // step * step, max(-(-lo // step) * step, int(round(v / step)) * step))


def draw(rng):
    kind = rng.choice(["norm", "norm_step", "norm_step", "gelu_step", "weight_grad", "weight_grad", "input_grad", "input_grad"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind in ("norm", "norm_step"):
        checkpoint = kind == "norm_step" and rng.random() < 0.4
        k = _spread(rng, 32, 16384, BLOCK if checkpoint else rng.choice([1, 2, 8, 64]))
        groups = rng.choice([0, 0, 1, 2, 3, 8])
        m = _spread(rng, 1, max(1, min(36864, LARGEST_STEP // k // (2 if dtype == "fp32" else 1))))
        m = max(1, m // groups) * groups if groups else m
        return _case(kind, m, k, dtype, groups=groups, checkpoint=checkpoint, sliced=groups > 0 and rng.random() < 0.5)
    if kind == "gelu_step":
        k = _spread(rng, 32, 15360, BLOCK)
        return _case(kind, _spread(rng, 1, LARGEST_GELU // k // (2 if dtype == "fp32" else 1)), k, dtype)
    k = _spread(rng, 256, 15360, rng.choice([64, 64, 32]))
    n = _spread(rng, 256, 15360, rng.choice([64, 64, 8]))
    m = _spread(rng, 1, min(16384, max(1, LARGEST_PRODUCT // (n * k) // {"bf16": 1, "fp16": 2, "fp32": 3}[dtype])))
    out = rng.choice([dtype, "fp32"]) if kind == "weight_grad" else dtype
    return _case(kind, m, k, dtype, n=n, out=out, bias=kind == "weight_grad" and rng.random() < 0.7)


# ------------------------------------------------------------------------------------------ the format
def _tiled(scales):
    """[rows, cols] bytes in the order in which the package holds them, the padding zero."""
    rows, cols = scales.shape
    tall, wide = -(-rows // 128), -(-cols // 4)
    full = torch.zeros(tall * 128, wide * 4, dtype=torch.uint8, device=scales.device)
    full[:rows, :cols] = scales
    return full.view(tall, 4, 32, wide, 4).permute(0, 3, 2, 1, 4).reshape(tall * 128, wide * 4)


def _untiled(scales, rows, cols):
    tall, wide = scales.shape[0] // 128, scales.shape[1] // 4
    return scales.view(tall, wide, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(tall * 128, wide * 4)[:rows, :cols]


def _power_of_two(e):
    return (e + 127 << 23).to(torch.int32).view(torch.float32)


def _to_mxfp8(x):
    """E4M3 codes and the scales' bytes (row by row): the smallest power of two that brings the block's largest value to 448 or below."""
    v = x.float().view(x.shape[0], -1, BLOCK)
    most = v.abs().amax(-1)
    mantissa, exponent = torch.frexp((most / 448.0).clamp(min=2.0 ** -126))
    exponent = (exponent - (mantissa == 0.5).int()).clamp(-126, 126)
    codes = (v * _power_of_two(-exponent).unsqueeze(-1)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return codes.view(x.shape), torch.where(most == 0, 0, exponent + 127).to(torch.uint8)


def _from_mxfp8(codes, scale_bytes):
    v = codes.float().view(codes.shape[0], -1, BLOCK)
    return (v * _power_of_two(scale_bytes.int() - 127).unsqueeze(-1)).view(codes.shape)


# ------------------------------------------------------------------------------------------ state
def _activation(gen, shape, dtype):
    """N(0, 1) about a small mean with one entry in a thousand scaled by 20, as the layers of a transformer see."""
    x = torch.randn(shape, generator=gen, device="cuda")
    x = torch.where(torch.rand(shape, generator=gen, device="cuda") < 0.001, x * 20, x).add_(0.1)
    return x.to(dtype)


def _operands(case, seed):
    """The inputs alone, by the seed."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, m, n, k, dtype = case["kind"], case["m"], case["n"], case["k"], DTYPE[case["dtype"]]
    s = {}
    if kind in ("norm", "norm_step"):
        groups = case["groups"]
        if groups:
            tokens = m // groups
            if case["sliced"]:  # the first tokens of each sample of a longer buffer; scale and shift are chunks of one projection's result
                s["x"] = _activation(gen, (groups, tokens + 5, k), dtype)[:, :tokens]
                chunks = (torch.randn(groups, 6 * k, generator=gen, device="cuda") * 0.2).to(dtype).chunk(6, dim=-1)
            else:
                s["x"] = _activation(gen, (groups, tokens, k), dtype)
                chunks = (torch.randn(2, groups, k, generator=gen, device="cuda") * 0.2).to(dtype)
            s["weight"], s["bias"], s["offset"] = chunks[0], chunks[1], 1.0
        else:
            s["x"] = _activation(gen, (m, k), dtype)
            s["weight"] = (1 + 0.2 * torch.randn(k, generator=gen, device="cuda")).to(dtype)
            s["bias"], s["offset"] = (0.2 * torch.randn(k, generator=gen, device="cuda")).to(dtype), 0.0
        if kind == "norm_step":
            s["dy"] = torch.randn(s["x"].shape, generator=gen, device="cuda").to(dtype)
    elif kind == "gelu_step":
        s["x"] = _activation(gen, (m, k), dtype)
        s["dy"] = torch.randn(m, k, generator=gen, device="cuda").to(dtype)
    else:
        s["dy"] = torch.randn(m, n, generator=gen, device="cuda").to(dtype)
        held = _activation(gen, (m, k), dtype) if kind == "weight_grad" else torch.randn(n, k, generator=gen, device="cuda") * 0.02
        codes, scale_bytes = _to_mxfp8(held)
        s["codes"], s["scales"] = codes, _tiled(scale_bytes).view(torch.float8_e8m0fnu)
    return s


def prepare(case, seed):
    s = _operands(case, seed)
    if case["kind"] in ("norm_step", "gelu_step"):
        for name in ("x", "weight", "bias"):
            if name in s:
                s[name] = s[name].detach().requires_grad_()
    s["case"] = case
    return s


# ------------------------------------------------------------------------------------------ a pass
def _run_own(s):
    import comfy_kitchen as ck

    case = s["case"]
    kind, out = case["kind"], DTYPE[case["out"]]
    if kind == "norm":
        with torch.inference_mode():
            return {"y": ck.layer_norm(s["x"], s["weight"], s["bias"], eps=EPS, weight_offset=s["offset"])}
    if kind == "norm_step":
        leaves = (s["x"], s["weight"], s["bias"])
        y = ck.layer_norm(*leaves, eps=EPS, weight_offset=s["offset"], checkpoint=case["checkpoint"])
        dx, dw, db = torch.autograd.grad(y, leaves, s["dy"])
        return {"y": y, "dx": dx, "dw": dw, "db": db}
    if kind == "gelu_step":
        y = ck.gelu_checkpointed(s["x"])
        return {"y": y, "dx": torch.autograd.grad(y, s["x"], s["dy"])[0]}
    if kind == "weight_grad":
        dw, db = ck.linear_weight_grad_mxfp8(s["dy"], s["codes"], s["scales"], out_dtype=out, bias_grad=case["bias"])
        return {"dw": dw, "db": db} if case["bias"] else {"dw": dw}
    return {"dx": ck.linear_input_grad_mxfp8(s["dy"], s["codes"], s["scales"], out_dtype=out)}


def _norm_forward(s):
    x = s["x"].float()
    mean = x.mean(-1, keepdim=True)
    rstd = ((x - mean).square().mean(-1, keepdim=True) + EPS).rsqrt()
    weight, bias = s["offset"] + s["weight"].float(), s["bias"].float()
    if weight.dim() == 2:
        weight, bias = weight.unsqueeze(1), bias.unsqueeze(1)
    return x, mean, rstd, weight, (x - mean) * rstd * weight + bias


def _gelu_parts(u):
    z = math.sqrt(2.0 / math.pi) * (u + 0.044715 * u * u * u)
    return torch.sigmoid(2.0 * z), math.sqrt(2.0 / math.pi) * (1.0 + 3 * 0.044715 * u * u)


def _run_plain(s):
    case = s["case"]
    kind, dtype, out = case["kind"], DTYPE[case["dtype"]], DTYPE[case["out"]]
    if kind == "norm":
        return {"y": _norm_forward(s)[-1].to(dtype)}
    dy = s["dy"].float()
    if kind == "norm_step":
        x, mean, rstd, weight, y = _norm_forward(s)
        if case["checkpoint"]:
            x = _from_mxfp8(*_to_mxfp8(x.reshape(-1, case["k"]))).view(x.shape)
        h = (x - mean) * rstd
        g = dy * weight
        dx = rstd * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
        rows = 1 if case["groups"] else 0
        return {"y": y.to(dtype), "dx": dx.to(dtype), "dw": (dy * h).sum(rows).to(dtype), "db": dy.sum(rows).to(dtype)}
    if kind == "gelu_step":
        u = s["x"].float()
        y = u * _gelu_parts(u)[0]
        v = _from_mxfp8(*_to_mxfp8(u))
        sig, slope = _gelu_parts(v)
        return {"y": y.to(dtype), "dx": (dy * (sig + 2.0 * v * sig * (1.0 - sig) * slope)).to(dtype)}
    held = _from_mxfp8(s["codes"], _untiled(s["scales"].view(torch.uint8), s["codes"].shape[0], case["k"] // BLOCK))
    if kind == "weight_grad":
        dw = {"dw": torch.matmul(dy.t(), held).to(out)}
        return {**dw, "db": dy.sum(0).to(out)} if case["bias"] else dw
    return {"dx": torch.matmul(dy, held).to(out)}


def run(s):
    if own:
        return _run_own(s)
    with torch.no_grad():
        return _run_plain(s)


# ------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    """Each input read once, each result written once; 10 operations an element and pass for the norms, 20 for GELU."""
    kind, m, n, k = case["kind"], case["m"], case["n"], case["k"]
    size, out = SIZE[case["dtype"]], SIZE[case["out"]]
    vectors = 2 * max(1, case["groups"]) * k * size
    if kind == "norm":
        return {"bytes": 2 * m * k * size + vectors, "flops": 10 * m * k}
    if kind == "norm_step":
        return {"bytes": 4 * m * k * size + 2 * vectors, "flops": 20 * m * k}
    if kind == "gelu_step":
        return {"bytes": 4 * m * k * size, "flops": 40 * m * k}
    held = (m if kind == "weight_grad" else n) * (k + k // BLOCK)
    result = n * k + (n if case["bias"] else 0) if kind == "weight_grad" else m * k
    return {"bytes": m * n * size + held + result * out, "flops": 2 * m * n * k}


# ------------------------------------------------------------------------------------------ the definition in 64 bits
def _two_to(e):
    return (e.long() + 1023 << 52).view(torch.float64)


def _held_values(x):
    """The values that stand in an MXFP8 copy of x, by arithmetic on 64-bit numbers."""
    v = x.double().reshape(-1, x.shape[-1] // BLOCK, BLOCK)
    most = v.abs().max(-1, keepdim=True).values
    fraction, above = torch.frexp(torch.clamp(most / 448.0, min=2.0 ** -126))
    step = _two_to(torch.where(fraction == 0.5, above - 1, above))
    scaled = v / step
    # four significant bits down to 2^-6, steps of 2^-9 below; to the nearest, ties to even
    place = _two_to(torch.frexp(scaled.abs().clamp(min=2.0 ** -6)).exponent - 4)
    return (torch.round(scaled / place) * place * step).reshape(x.shape)


def _as_stored(codes, scales):
    """The same from codes and scales: byte r, c of the scales stands at 512 * tile + 16 * (r % 32) + 4 * (r // 32 % 4) + c % 4."""
    rows, cols = codes.shape
    r = torch.arange(rows, device=codes.device).unsqueeze(1)
    c = torch.arange(cols // BLOCK, device=codes.device).unsqueeze(0)
    at = ((r // 128) * (scales.shape[1] // 4) + c // 4) * 512 + (r % 32) * 16 + (r // 32 % 4) * 4 + c % 4
    bytes_ = scales.view(torch.uint8).reshape(-1)[at].long()
    factor = torch.where(bytes_ == 0, 0.0, _two_to(bytes_ - 127))
    return codes.double() * factor.repeat_interleave(BLOCK, 1)


def exact(case, seed):
    s = _operands(case, seed)
    kind, k = case["kind"], case["k"]
    if kind in ("norm", "norm_step"):
        x = s["x"].double()
        groups = x if x.dim() == 3 else x.unsqueeze(0)
        w, b = (s[name].double().reshape(-1, 1, k) for name in ("weight", "bias"))
        var, mean = torch.var_mean(groups, dim=2, correction=0, keepdim=True)
        y = (groups - mean) / torch.sqrt(var + EPS) * (w + s["offset"]) + b
        if kind == "norm":
            return {"y": y.reshape(x.shape)}
        del y
        kept = _held_values(s["x"]).reshape(groups.shape) if case["checkpoint"] else groups
        h = (kept - mean) / torch.sqrt(var + EPS)
        dy = s["dy"].double().reshape(groups.shape)
        dw, db = (dy * h).sum(1).reshape(s["weight"].shape), dy.sum(1).reshape(s["weight"].shape)
        g = dy * (w + s["offset"])
        del dy
        along = torch.einsum("gtk,gtk->gt", g, h).unsqueeze(2) / k
        dx = (g - g.mean(2, keepdim=True) - h * along) / torch.sqrt(var + EPS)
        del g, h
        y = (groups - mean) / torch.sqrt(var + EPS) * (w + s["offset"]) + b
        return {"y": y.reshape(x.shape), "dx": dx.reshape(x.shape), "dw": dw, "db": db}
    if kind == "gelu_step":
        root = math.sqrt(2.0 / math.pi)
        u = s["x"].double()
        y = 0.5 * u * (1.0 + torch.tanh(root * (u + 0.044715 * u ** 3)))
        v = _held_values(s["x"])
        t = torch.tanh(root * (v + 0.044715 * v ** 3))
        slope = 0.5 * (1.0 + t) + 0.5 * v * (1.0 - t * t) * root * (1.0 + 3.0 * 0.044715 * v * v)
        return {"y": y, "dx": s["dy"].double() * slope}
    dy, held = s["dy"].double(), _as_stored(s["codes"], s["scales"])
    if kind == "weight_grad":
        dw = {"dw": dy.t() @ held}
        return {**dw, "db": dy.sum(0)} if case["bias"] else dw
    return {"dx": dy @ held}
