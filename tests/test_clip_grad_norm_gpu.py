"""The gradients' global norm and clipping by it, on the GPU.

Bounds.  u = 2^-24.  A square is off by u, and a thread adds up to 16 in a vector, a few tens of vectors and a tree of ten levels: 64 u of the sum of
squares, half of it behind the root, for the sizes here.  The scaled gradients are what fp32 arithmetic gives from the norm that is returned,
bit for bit.
"""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0**-24


@pytest.fixture(scope="module")
def ck(cuda_device):
    import comfy_kitchen

    assert comfy_kitchen.list_backends()["cuda"]["available"]
    return comfy_kitchen


def _made(shape, dtype, seed, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _params(grads):
    params = []
    for g in grads:
        p = torch.nn.Parameter(torch.zeros_like(g, memory_format=torch.preserve_format))
        p.grad = g
        params.append(p)
    return params


def _check(ck, grads, max_norm):
    before = [g.clone() for g in grads]
    want = torch.stack([g.double().square().sum() for g in before]).sum().sqrt()
    assert (ck.grad_norm(grads).double() - want).abs() <= 32 * U * want
    norm = ck.clip_grad_norm_(_params(grads), max_norm)
    assert norm.shape == () and norm.dtype == torch.float32 and norm.is_cuda
    assert (norm.double() - want).abs() <= 32 * U * want
    factor = torch.tensor(max_norm, device="cuda") / (norm + 1e-6)
    for g, b in zip(grads, before):
        assert torch.equal(g, b if factor >= 1 else (b.float() * factor).to(b.dtype))


SHAPES = [[(1,)], [(5, 7)], [(1000,), (3,), (17, 33)], [(4096, 512)], [(n,) for n in range(1, 80)], [(0,), (9,), (0, 4)], [(70001,), (8,), (65536,), (65535,), (65537,)]]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32, None])
@pytest.mark.parametrize("shapes", SHAPES)
@pytest.mark.parametrize("max_norm", [0.5, 1e9])
def test_clip(ck, shapes, dtype, max_norm):
    cycle = [torch.float32, torch.bfloat16, torch.float16]
    _check(ck, [_made(s, dtype or cycle[i % 3], i, 0.1) for i, s in enumerate(shapes)], max_norm)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_views_of_one_buffer(ck, dtype):
    """Tensors that start anywhere; what stands between them is left as it was."""
    flat = _made((300_000,), dtype, 1)
    sizes, grads, at = [1, 31, 5000, 16, 15, 17, 100_001, 33, 2], [], 3
    for s in sizes:
        grads.append(flat[at:at + s])
        at += s + (s % 2)
    held = flat.clone()
    _check(ck, grads, 1.0)
    mask = torch.ones_like(flat, dtype=torch.bool)
    at = 3
    for s in sizes:
        mask[at:at + s] = False
        at += s + (s % 2)
    assert torch.equal(flat[mask], held[mask])


def test_more_tensors_than_a_launch_has_room_for(ck):
    _check(ck, [_made((1 + i % 70,), torch.float32, i) for i in range(2500)], 2.0)
    _check(ck, [_made((1 + i % 70,), torch.bfloat16, i) for i in range(1024)], 2.0)
    _check(ck, [_made((3,), torch.float16, i) for i in range(65)], 0.25)


def test_large(ck):
    _check(ck, [_made((40_000_000,), torch.bfloat16, 1, 1e-3), _made((3, 5), torch.float32, 2), _made((10_000_001,), torch.float32, 3, 1e-3)], 1.0)


def test_special_values(ck):
    def clipped(*values, max_norm=1.0):
        g = torch.tensor(values, device="cuda")
        return ck.clip_grad_norm_(_params([g]), max_norm).item(), g.tolist()

    norm, g = clipped(3.0, 4.0, max_norm=0.0)
    assert norm == 5.0 and g == [0.0, 0.0]
    norm, g = clipped(float("inf"), 1.0)
    assert norm == float("inf") and g[1] == 0.0 and g[0] != g[0]
    norm, g = clipped(float("nan"), 1.0)
    assert norm != norm and g[0] != g[0] and g[1] != g[1]
    assert clipped(0.0, 0.0) == (0.0, [0.0, 0.0])
    assert clipped(3.0, 4.0, max_norm=float("inf")) == (5.0, [3.0, 4.0])


def test_as_torch_has_it(ck):
    grads = [_made((100, 30), torch.float32, 4), _made((77,), torch.float32, 5)]
    ours, theirs = _params([g.clone() for g in grads]), _params([g.clone() for g in grads])
    norm = ck.clip_grad_norm_(ours, 1.5)
    want = torch.nn.utils.clip_grad_norm_(theirs, 1.5)
    assert (norm - want).abs() <= 64 * U * want
    for p, q in zip(ours, theirs):
        assert ((p.grad - q.grad).abs() <= 80 * U * q.grad.abs()).all()


def test_parameters_as_they_come(ck):
    g = _made((50,), torch.float32, 6)
    p, no_grad = _params([g.clone()])[0], torch.nn.Parameter(torch.zeros(3, device="cuda"))
    once = ck.clip_grad_norm_([p, no_grad, p], 0.1)  # the same parameter twice counts once
    assert torch.equal(once, ck.grad_norm([g]))
    assert ck.clip_grad_norm_([no_grad], 1.0).item() == 0.0 and ck.clip_grad_norm_([], 1.0).item() == 0.0
    p.grad = g.clone()
    assert torch.equal(ck.clip_grad_norm_(p, 0.1), once) and torch.equal(ck.clip_grad_norm_(iter([p]), 1e9), ck.grad_norm(p.grad))
    # a gradient whose memory is in another order
    t = _made((30, 40), torch.float32, 7)
    q = torch.nn.Parameter(torch.zeros(40, 30, device="cuda"))
    q.grad = t.clone().t()
    norm = ck.clip_grad_norm_([q], 0.1)
    assert torch.equal(q.grad, (t * (torch.tensor(0.1, device="cuda") / (norm + 1e-6))).t())


def test_a_change_is_seen_by_autograd(ck):
    g = _made((8,), torch.float32, 8)
    version = g._version
    ck.clip_grad_norm_(_params([g]), 1e-3)
    assert g._version > version


def test_error_if_nonfinite(ck):
    g = torch.tensor([1.0, float("inf")], device="cuda")
    with pytest.raises(RuntimeError, match="inf"):
        ck.clip_grad_norm_(_params([g]), 1.0, error_if_nonfinite=True)
    assert g.tolist() == [1.0, float("inf")]
    ck.clip_grad_norm_(_params([g[:1]]), 1.0, error_if_nonfinite=True)


def test_the_dispatchers_route(ck):
    from torch.utils._python_dispatch import TorchDispatchMode

    class Watch(TorchDispatchMode):
        seen = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.seen.append(str(func))
            return func(*args, **(kwargs or {}))

    grads = [_made((50,), torch.float32, 9), _made((5, 5), torch.float32, 10)]
    other = [g.clone() for g in grads]
    want = ck.clip_grad_norm_(_params(grads), 0.5)
    params = _params(other)
    with Watch():
        got = ck.clip_grad_norm_(params, 0.5)
    assert any("clip_grads" in s for s in Watch.seen) and torch.equal(got, want)
    assert all(torch.equal(a, b) for a, b in zip(grads, other))


def test_captured(ck):
    grads = [_made((1000,), torch.float32, 11), _made((5, 5), torch.bfloat16, 12)]
    fresh = [g.clone() for g in grads]
    params = _params(grads)
    ck.clip_grad_norm_(params, 0.5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = ck.clip_grad_norm_(params, 0.5)
    for scale in (1.0, 2.0, 1e-4):
        for g, f in zip(grads, fresh):
            g.copy_(f * scale)
        other = [g.clone() for g in grads]
        graph.replay()
        assert torch.equal(norm, ck.clip_grad_norm_(_params(other), 0.5))
        assert all(torch.equal(a, b) for a, b in zip(grads, other))
    del graph


def test_refusals(ck):
    flat = torch.zeros(100, device="cuda")
    for bad in (lambda: ck.clip_grad_norm_(_params([flat[:60], flat[50:]]), 1.0), lambda: ck.clip_grad_norm_(_params([flat]), -1.0),
                lambda: ck.clip_grad_norm_(_params([flat]), float("nan")), lambda: ck.clip_grad_norm_(_params([flat.cpu()]), 1.0),
                lambda: ck.clip_grad_norm_(_params([flat, flat.cpu()]), 1.0), lambda: ck.clip_grad_norm_(_params([flat.double()]), 1.0),
                lambda: ck.grad_norm([flat, flat.to(torch.complex64)])):
        with pytest.raises(Exception):
            bad()
