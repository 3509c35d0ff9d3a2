"""Cases of the operators of language-model layers: RMS norm, experts' products on MXFP8 weights, clipping by the global gradient norm.

A case is a dict of plain values.  ``kind`` names the operator:

* ``rms``           ``ck.rms_norm`` in inference, with or without a residual that is added first
* ``rms_mxfp8``     ``ck.rms_norm_mxfp8``: the same with the result in MXFP8, as the next linear layer reads it
* ``rms_step``      ``ck.rms_norm`` and its backward pass
* ``experts``       ``ck.grouped_linear_mxfp8``: rows in the experts' order, each through the MXFP8 weight of its own expert
* ``experts_mm``    ``ck.grouped_mm_mxfp8``: the same on rows that are held in MXFP8 already
* ``experts_grad``  ``ck.grouped_input_grad_mxfp8``: gradients of the rows through the experts' weights
* ``clip``          ``ck.clip_grad_norm_`` over many gradients; with ``clipped`` the norm is above the bound, and new gradients arrive first

``m`` counts rows, ``k`` (input) features, ``n`` output features.  ``skew`` says how unevenly the rows go to the experts (0: alike; 1: the
e-th expert gets about 1 / e of the first one's).  Sizes are generic ones of transformer layers, or odd.

An MXFP8 matrix is held as the package holds it: E4M3 codes ``[rows, cols]`` and one E8M0 byte for 32 of a row, in tiles of 128 rows
by 4 blocks (512 bytes: 32 rows of 16, four rows 32 apart in each).  Where an operator's result is in MXFP8, a pass returns the values
that it stands for.
"""
from __future__ import annotations

import os
import random
import sys

import torch

own = False

_PACKAGE = os.path.join(os.getcwd(), "comfy-kitchen_b200")
if _PACKAGE not in sys.path:
    sys.path.insert(0, _PACKAGE)

DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-6
BLOCK = 32
MAX_NORM = 1.0
LARGEST_NORM = 16384 * 4096  # elements of the largest listed norm
LARGEST_PRODUCT = 8192 * 8192 * 4096  # multiply-adds of the largest listed product
LARGEST_EXPERTS = 8 * 8192 * 4096  # elements of its weights
LARGEST_CLIP = 4 * 2 * 2048 * 8192


def _norm(kind, m, k, dtype, residual=False, heads=0, offset=0.0, **name):
    return {**name, "kind": kind, "m": m, "k": k, "dtype": dtype, "residual": residual, "heads": heads, "offset": offset}


def _experts(kind, m, n, k, experts, dtype, skew=0.5, bias=False, **name):
    return {**name, "kind": kind, "m": m, "n": n, "k": k, "experts": experts, "dtype": dtype, "skew": skew, "bias": bias}


def _clip(tensors, total, dtype, clipped, features=0, **name):
    return {**name, "kind": "clip", "tensors": tensors, "total": total, "dtype": dtype, "clipped": clipped, "features": features}


def listed():
    return [
        # one token on its way into a served layer: latency
        _norm("rms_mxfp8", 1, 4096, "bf16", residual=True, name="rms_one_token_mxfp8"),
        # the rows of a long prompt, normalized into the operand of the next linear layer
        _norm("rms_mxfp8", 8192, 4096, "bf16", residual=True, name="rms_prompt_mxfp8"),
        # the keys of every head, a part of the projection's result
        _norm("rms", 4096 * 24, 128, "fp16", heads=24, name="rms_heads_fp16"),
        # a training step over a batch's tokens
        _norm("rms_step", 16384, 4096, "bf16", residual=True, name="rms_step_batch"),
        # odd width, odd rows, full precision: a small model's norm, its weight held as the distance from one
        _norm("rms_step", 1003, 1777, "fp32", offset=1.0, name="rms_step_odd_fp32"),
        # one token that goes to eight of 64 experts: the weights' read counts
        _experts("experts", 8, 1536, 2048, 64, "bf16", skew=0.0, name="experts_one_token"),
        # a prompt's rows, each token twice, over eight wide experts
        _experts("experts", 8192, 8192, 4096, 8, "bf16", name="experts_prompt"),
        # ragged rows in half precision, experts without rows among them, features that are no multiple of a tile, a bias
        _experts("experts_mm", 777, 1000, 1056, 40, "fp16", skew=1.0, bias=True, name="experts_ragged_fp16"),
        # the gradient of a batch's rows through frozen experts
        _experts("experts_grad", 8192, 8192, 4096, 8, "bf16", name="experts_grad_batch"),
        # full-precision gradients of few rows
        _experts("experts_grad", 333, 1536, 2048, 16, "fp32", skew=1.0, name="experts_grad_ragged_fp32"),
        # the small tensors of a model, most steps of a run: the norm is below the bound
        _clip(300, 1_000_000, "fp32", False, name="clip_many_small_fp32"),
        # four blocks of an MLP, an early step: the norm is above the bound
        _clip(24, 0, "bf16", True, features=2048, name="clip_blocks"),
    ]


def _spread(rng, lo, hi, step=1):
    """A multiple of ``step`` in [lo, hi], uniform over the logarithm."""
    v = lo * (hi / lo) ** rng.random()
    return min(hi // step * step, max(-(-lo // step) * step, int(round(v / step)) * step))


def draw(rng):
    kind = rng.choice(["rms", "rms_mxfp8", "rms_step", "rms_step", "experts", "experts", "experts_mm", "experts_grad", "experts_grad", "clip"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    wide = 2 if dtype == "fp32" else 1
    if kind in ("rms", "rms_mxfp8", "rms_step"):
        residual = rng.random() < 0.6
        heads = rng.choice([1, 5, 24]) if not residual and kind == "rms" and rng.random() < 0.6 else 0
        k = rng.choice([64, 96, 128, 256]) if heads else _spread(rng, 32, 16384, BLOCK if kind == "rms_mxfp8" else rng.choice([1, 2, 8, 64]))
        m = _spread(rng, 1, max(1, min(65536, LARGEST_NORM // k // wide)))
        if heads:
            m = max(1, m // heads) * heads
        return _norm(kind, m, k, dtype, residual=residual, heads=heads, offset=rng.choice([0.0, 0.0, 1.0]))
    if kind == "clip":
        return _clip(_spread(rng, 1, 400), _spread(rng, 1000, LARGEST_CLIP // wide), dtype, rng.random() < 0.5)
    experts = _spread(rng, 1, 128)
    k = _spread(rng, 256, 8192, rng.choice([64, 64, 32]))
    most = max(264, min(8192, LARGEST_EXPERTS // (k * experts)))
    n = _spread(rng, 256, most, rng.choice([64, 64, 8]))
    cost = {"bf16": 1, "fp16": 2, "fp32": 3}[dtype] if kind == "experts_grad" else wide
    m = _spread(rng, 1, max(1, min(16384, LARGEST_PRODUCT // (n * k) // cost)))
    return _experts(kind, m, n, k, experts, dtype, skew=rng.choice([0.0, 0.5, 1.0, 2.0]), bias=kind != "experts_grad" and rng.random() < 0.3)


# ------------------------------------------------------------------------------------------ the format
def _tiled(scales):
    """[..., rows, cols] bytes in the order in which the package holds them, the padding zero."""
    *many, rows, cols = scales.shape
    tall, wide = -(-rows // 128), -(-cols // 4)
    full = torch.zeros(*many, tall * 128, wide * 4, dtype=torch.uint8, device=scales.device)
    full[..., :rows, :cols] = scales
    return full.view(-1, tall, 4, 32, wide, 4).permute(0, 1, 4, 3, 2, 5).reshape(*many, tall * 128, wide * 4)


def _untiled(scales, rows, cols):
    *many, tall, wide = scales.shape
    tiles = scales.reshape(-1, tall // 128, wide // 4, 32, 4, 4).permute(0, 1, 4, 3, 2, 5)
    return tiles.reshape(*many, tall, wide)[..., :rows, :cols]


def _power_of_two(e):
    return (e + 127 << 23).to(torch.int32).view(torch.float32)


def _to_mxfp8(x):
    """E4M3 codes and the scales' bytes (row by row): the smallest power of two that brings the block's largest value to 448 or below."""
    v = x.float().unflatten(-1, (-1, BLOCK))
    most = v.abs().amax(-1)
    mantissa, exponent = torch.frexp((most / 448.0).clamp(min=2.0 ** -126))
    exponent = (exponent - (mantissa == 0.5).int()).clamp(-126, 126)
    codes = (v * _power_of_two(-exponent).unsqueeze(-1)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return codes.flatten(-2), torch.where(most == 0, 0, exponent + 127).to(torch.uint8)


def _from_mxfp8(codes, scale_bytes):
    v = codes.float().unflatten(-1, (-1, BLOCK))
    return (v * _power_of_two(scale_bytes.int() - 127).unsqueeze(-1)).flatten(-2)


# ------------------------------------------------------------------------------------------ state
def _activation(gen, shape, dtype):
    """N(0, 1) with one entry in a thousand scaled by 20, as the layers of a transformer see."""
    x = torch.randn(shape, generator=gen, device="cuda")
    return torch.where(torch.rand(shape, generator=gen, device="cuda") < 0.001, x * 20, x).to(dtype)


def _shares(case):
    """The experts' chances of a row."""
    w = [(e + 1.0) ** -case["skew"] for e in range(case["experts"])]
    return [v / sum(w) for v in w]


def _clip_sizes(case):
    """Elements of each gradient: those of an MLP's blocks, or spread over three orders of magnitude."""
    f = case["features"]
    if f:
        return [f, f, f * 4 * f, 4 * f, 4 * f * f, f] * (case["tensors"] // 6)
    rng = random.Random(case["tensors"])
    parts = [10 ** (3 * rng.random()) for _ in range(case["tensors"])]
    return [max(1, int(case["total"] * p / sum(parts))) for p in parts]


def _operands(case, seed):
    """The inputs alone, by the seed."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, dtype = case["kind"], DTYPE[case["dtype"]]
    s = {}
    if kind in ("rms", "rms_mxfp8", "rms_step"):
        m, k, heads = case["m"], case["k"], case["heads"]
        if heads:  # the middle third of a projection's result
            s["x"] = _activation(gen, (m // heads, 3, heads, k), dtype)[:, 1]
        else:
            s["x"] = _activation(gen, (m, k), dtype)
        s["weight"] = (1 - case["offset"] + 0.2 * torch.randn(k, generator=gen, device="cuda")).to(dtype)
        if case["residual"]:
            s["residual"] = (3 * _activation(gen, (m, k), torch.float32)).to(dtype)
        if kind == "rms_step":
            s["dy"] = torch.randn(m, k, generator=gen, device="cuda").to(dtype)
            if case["residual"]:
                s["dh"] = torch.randn(m, k, generator=gen, device="cuda").to(dtype)
        return s
    if kind == "clip":
        sizes = _clip_sizes(case)
        # views of one buffer, as a trainer that communicates its gradients together holds them
        total = sum(sizes)
        size = 0.5 * MAX_NORM / total ** 0.5 * (20.0 if case["clipped"] else 1.0)
        s["fresh"], s["sizes"] = (torch.randn(total, generator=gen, device="cuda") * size).to(dtype), sizes
        return s
    m, n, k, experts = case["m"], case["n"], case["k"], case["experts"]
    chosen = torch.multinomial(torch.tensor(_shares(case), device="cuda"), m, replacement=True, generator=gen)
    counts = torch.bincount(chosen, minlength=experts)
    s["offsets"], s["sizes"] = counts.cumsum(0).to(torch.int32), counts.tolist()
    s["w_codes"], held = _to_mxfp8(torch.randn(experts, n, k, generator=gen, device="cuda") * 0.02)
    s["w_scales"] = _tiled(held).view(torch.float8_e8m0fnu)
    if kind == "experts_grad":
        s["dy"] = torch.randn(m, n, generator=gen, device="cuda").to(dtype)
        return s
    x = _activation(gen, (m, k), dtype)
    if kind == "experts":
        s["x"] = x
    else:
        s["x_codes"], held = _to_mxfp8(x)
        s["x_scales"] = _tiled(held).view(torch.float8_e8m0fnu)
    s["bias"] = (torch.randn(experts, n, generator=gen, device="cuda") * 0.1).to(dtype) if case["bias"] else None
    return s


def prepare(case, seed):
    s = _operands(case, seed)
    if case["kind"] == "rms_step":
        for name in ("x", "weight", "residual"):
            if name in s:
                s[name] = s[name].detach().requires_grad_()
    if case["kind"] == "clip":
        s["flat"] = s["fresh"].clone()
        s["params"] = [torch.nn.Parameter(torch.zeros_like(g)) for g in s["flat"].split(s["sizes"])]
        for p, g in zip(s["params"], s["flat"].split(s["sizes"])):
            p.grad = g
    s["case"] = case
    return s


# ------------------------------------------------------------------------------------------ a pass
def _run_own(s):
    import comfy_kitchen as ck

    case = s["case"]
    kind, dtype = case["kind"], DTYPE[case["dtype"]]
    if kind == "rms":
        with torch.inference_mode():
            out = ck.rms_norm(s["x"], s["weight"], s.get("residual"), eps=EPS, weight_offset=case["offset"])
        return {"y": out[0], "h": out[1]} if case["residual"] else {"y": out}
    if kind == "rms_mxfp8":
        with torch.inference_mode():
            codes, scales, *h = ck.rms_norm_mxfp8(s["x"], s["weight"], s.get("residual"), eps=EPS, weight_offset=case["offset"])
            y = ck.dequantize_mxfp8(codes, scales, torch.bfloat16)
        return {"y": y, "h": h[0]} if case["residual"] else {"y": y}
    if kind == "rms_step":
        x, weight, residual = s["x"], s["weight"], s.get("residual")
        out = ck.rms_norm(x, weight, residual, eps=EPS, weight_offset=case["offset"])
        if residual is None:
            dx, dw = torch.autograd.grad(out, (x, weight), s["dy"])
            return {"y": out, "dx": dx, "dw": dw}
        dx, dr, dw = torch.autograd.grad(out, (x, residual, weight), (s["dy"], s["dh"]))
        return {"y": out[0], "h": out[1], "dx": dx, "dr": dr, "dw": dw}
    if kind == "experts":
        with torch.inference_mode():
            return {"y": ck.grouped_linear_mxfp8(s["x"], s["w_codes"], s["w_scales"], s["offsets"], s["bias"])}
    if kind == "experts_mm":
        return {"y": ck.grouped_mm_mxfp8(s["x_codes"], s["w_codes"], s["x_scales"], s["w_scales"], s["offsets"], s["bias"], out_dtype=dtype)}
    if kind == "experts_grad":
        return {"dx": ck.grouped_input_grad_mxfp8(s["dy"], s["w_codes"], s["w_scales"], s["offsets"])}
    if case["clipped"]:
        s["flat"].copy_(s["fresh"])
    norm = ck.clip_grad_norm_(s["params"], MAX_NORM)
    return {"norm": norm, "grads": s["flat"]}


def _run_plain(s):
    case = s["case"]
    kind, dtype = case["kind"], DTYPE[case["dtype"]]
    if kind in ("rms", "rms_mxfp8", "rms_step"):
        h = s["x"] if s.get("residual") is None else (s["x"].float() + s["residual"].float()).to(dtype)
        v = h.float()
        rstd = (v.square().mean(-1, keepdim=True) + EPS).rsqrt()
        weight = s["weight"].float() + case["offset"]
        y = (v * rstd * weight).to(dtype)
        if kind == "rms_mxfp8":
            y = _from_mxfp8(*_to_mxfp8(y)).to(torch.bfloat16)  # 4 significant bits: exact
        out = {"y": y, "h": h} if case["residual"] else {"y": y}
        if kind != "rms_step":
            return out
        dy = s["dy"].float()
        g, unit = dy * weight, v * rstd
        dx = rstd * (g - unit * (g * unit).mean(-1, keepdim=True))
        out["dw"] = (dy * unit).sum(0).to(dtype)
        if case["residual"]:
            dx = dx + s["dh"].float()
        out["dx"] = dx.to(dtype)
        return {**out, "dr": out["dx"]} if case["residual"] else out
    if kind == "clip":
        if case["clipped"]:
            s["flat"].copy_(s["fresh"])
        grads = [p.grad for p in s["params"]]
        norm = torch.stack([g.float().square().sum() for g in grads]).sum().sqrt()
        factor = (MAX_NORM / (norm + 1e-6)).clamp(max=1.0)
        for g in grads:
            g.copy_(g.float() * factor)
        return {"norm": norm, "grads": s["flat"]}
    # an expert at a time: their rows differ in number
    n, k = case["n"], case["k"]
    held = _untiled(s["w_scales"].view(torch.uint8), n, k // BLOCK)
    if kind == "experts_grad":
        parts = [d.float() @ _from_mxfp8(c, b) for d, c, b in zip(s["dy"].split(s["sizes"]), s["w_codes"], held) if len(d)]
        return {"dx": torch.cat(parts).to(dtype)}
    if kind == "experts":
        x = _from_mxfp8(*_to_mxfp8(s["x"]))
    else:
        x = _from_mxfp8(s["x_codes"], _untiled(s["x_scales"].view(torch.uint8), case["m"], k // BLOCK))
    bias = s["bias"].float() if case["bias"] else torch.zeros(case["experts"], 1, device="cuda")
    parts = [r @ _from_mxfp8(c, b).t() + z for r, c, b, z in zip(x.split(s["sizes"]), s["w_codes"], held, bias) if len(r)]
    return {"y": torch.cat(parts).to(dtype)}


def run(s):
    if own:
        return _run_own(s)
    with torch.no_grad():
        return _run_plain(s)


# ------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    """Each input read once, each result written once (the gradients that are clipped twice: the norm stands between); the weights of the
    experts that can be expected to have rows."""
    kind, size = case["kind"], SIZE[case["dtype"]]
    if kind == "clip":
        total = sum(_clip_sizes(case))
        return {"bytes": total * size * (5 if case["clipped"] else 1), "flops": total * (3 if case["clipped"] else 2)}
    m, k = case["m"], case["k"]
    if kind in ("rms", "rms_mxfp8", "rms_step"):
        out = size if kind != "rms_mxfp8" else 2 + 2 * (1 + 1 / BLOCK)  # written, read and returned as bf16 values
        elements = m * k * (size + out + (2 * size if case["residual"] else 0))
        if kind == "rms_step":
            elements += m * k * (3 + (1 if case["residual"] else 0)) * size
        return {"bytes": elements + 2 * k * size, "flops": m * k * (16 if kind == "rms_step" else 6)}
    n = case["n"]
    busy = sum(1.0 - (1.0 - p) ** m for p in _shares(case))
    rows = m * k * (1 + 1 / BLOCK) if kind == "experts_mm" else m * k * size
    return {"bytes": rows + m * n * size + busy * n * k * (1 + 1 / BLOCK), "flops": 2 * m * n * k}


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
    kind, dtype = case["kind"], DTYPE[case["dtype"]]
    if kind in ("rms", "rms_mxfp8", "rms_step"):
        total = s["x"].double() + s["residual"].double() if case["residual"] else s["x"].double()
        h = total.to(dtype).double()  # the sum is an output, and the norm is of what stands there
        root = torch.sqrt(torch.linalg.vector_norm(h, dim=-1, keepdim=True) ** 2 / case["k"] + EPS)
        scale = s["weight"].double() + case["offset"]
        # a result in MXFP8 has none: next to a border between two codes, the last bit of 32 says which one a number takes
        out = {"y": None if kind == "rms_mxfp8" else h / root * scale}
        if case["residual"]:
            out["h"] = total
        if kind == "rms_step":
            dy = s["dy"].double()
            out["dw"] = torch.einsum("mk,mk->k", dy, h / root)
            along = torch.einsum("mk,mk->m", dy * scale, h).unsqueeze(-1) / case["k"]
            out["dx"] = dy * scale / root - h * along / root ** 3
            if case["residual"]:
                out["dx"] = out["dr"] = out["dx"] + s["dh"].double()
        return out
    if kind == "clip":
        g = s["fresh"].double()
        norm = torch.linalg.vector_norm(g)
        return {"norm": norm, "grads": g * min(1.0, MAX_NORM / (norm.item() + 1e-6))}
    if kind == "experts_grad":
        rows = s["dy"].double()
    else:
        rows = _held_values(s["x"]) if kind == "experts" else _as_stored(s["x_codes"], s["x_scales"])
    out = torch.empty(case["m"], case["k"] if kind == "experts_grad" else case["n"], dtype=torch.float64, device="cuda")
    ends = s["offsets"].tolist()
    for e, (begin, end) in enumerate(zip([0, *ends], ends)):
        if begin == end:
            continue
        w = _as_stored(s["w_codes"][e], s["w_scales"][e])
        if kind == "experts_grad":
            out[begin:end] = torch.einsum("mn,nk->mk", rows[begin:end], w)
        else:
            out[begin:end] = torch.einsum("mk,nk->mn", rows[begin:end], w)
            if case["bias"]:
                out[begin:end] += s["bias"][e].double()
    return {"dx": out} if kind == "experts_grad" else {"y": out}
