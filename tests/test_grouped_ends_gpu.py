"""Ends of groups that decrease, lie below zero or behind the rows, in every kernel that reads them: calls end, stay inside their buffers, and
do no more than the rows' work.  And results and workspaces with guards on both sides, through the C entry points."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu
GUARD = 4096


@pytest.fixture(scope="module")
def ck(cuda_device):
    import comfy_kitchen

    assert comfy_kitchen.list_backends()["cuda"]["available"]
    return comfy_kitchen


@pytest.fixture(scope="module")
def lib(ck):
    from comfy_kitchen.backends import cuda

    return cuda.load_library()


def _made(shape, dtype, seed, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


class Guarded:
    def __init__(self, size):
        self.size = size
        self.all = torch.full((size + 2 * GUARD,), 0xA5, dtype=torch.uint8, device="cuda")
        self.inside = self.all[GUARD:GUARD + size]
        assert self.inside.data_ptr() % 256 == 0

    def whole(self):
        return bool((self.all[:GUARD] == 0xA5).all() and (self.all[GUARD + self.size:] == 0xA5).all())


# rows, N, K: half tiles and the few-row gradient; single CTAs; pairs and the gradient's GEMM
SHAPES = [(100, 72, 64), (515, 1160, 288), (1500, 1544, 4128)]


def _odd_ends(m):
    return [[m, 0, m, 0], [0, m // 3, m // 4, m], [-5, m // 2, 2**31 - 1, 7], [2 * m, 3 * m, m, -m], [-1, -1, -1, -1], [m // 2, m // 2 - 1, m // 2 + 1, m - 1]]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_guards(ck, lib, m, n, k):
    from comfy_kitchen.backends.cuda import check_device_status

    x, dy = _made((m, k), torch.bfloat16, 1), _made((m, n), torch.float16, 2)
    xc, xs = ck.quantize_mxfp8(x)
    codes, scales = ck.quantize_experts_mxfp8(_made((4, n, k), torch.float32, 3, 0.05))
    stream = torch.cuda.current_stream().cuda_stream
    sound = [[m // 4, m // 2, m // 2, m], [0, 0, 0, 3], [m, m, m, m]]
    for ends in sound + _odd_ends(m):
        e = torch.tensor(ends, dtype=torch.int32, device="cuda")
        out, ws = Guarded(m * n * 2), Guarded(lib.ck_grouped_mm_mxfp8_workspace_bytes(1, m, k, 4))
        assert lib.ck_grouped_linear_mxfp8(x.data_ptr(), 2, codes.data_ptr(), scales.data_ptr(), e.data_ptr(), None, 0, out.inside.data_ptr(), 2, m, n, k, 4,
                                           ws.inside.data_ptr(), ws.size, stream) == 0
        assert out.whole() and ws.whole()
        if ends in sound:
            assert torch.equal(out.inside.view(torch.bfloat16).view(m, n), ck.grouped_linear_mxfp8(x, codes, scales, e))
        out, ws = Guarded(m * n * 4), Guarded(lib.ck_grouped_mm_mxfp8_workspace_bytes(0, m, k, 4))
        assert lib.ck_grouped_mm_mxfp8(xc.data_ptr(), codes.data_ptr(), xs.data_ptr(), scales.data_ptr(), e.data_ptr(), None, 0, out.inside.data_ptr(), 0, m, n,
                                       k, 4, ws.inside.data_ptr(), ws.size, stream) == 0
        assert out.whole() and ws.whole()
        for code in (0, 1, 2):
            out, ws = Guarded(m * k * (4 if code == 0 else 2)), Guarded(lib.ck_grouped_input_grad_mxfp8_workspace_bytes(1, m, n, k, 4))
            assert lib.ck_grouped_input_grad_mxfp8(dy.data_ptr(), 1, codes.data_ptr(), scales.data_ptr(), e.data_ptr(), out.inside.data_ptr(), code, m, n, k, 4,
                                                   ws.inside.data_ptr(), ws.size, stream) == 0
            assert out.whole() and ws.whole()
    check_device_status()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_no_row_is_two_experts(ck, m, n, k, dtype):
    """An end below an earlier one counts as that one (the gradient, whose rows need nothing that was laid out by group)."""
    dy = _made((m, n), dtype, 4)
    codes, scales = ck.quantize_experts_mxfp8(_made((4, n, k), torch.float32, 3, 0.05))

    def grad(ends):
        return ck.grouped_input_grad_mxfp8(dy, codes, scales, torch.tensor(ends, dtype=torch.int32, device="cuda"))

    for ends in _odd_ends(m):
        above, most = [], 0
        for e in ends:
            most = max(most, min(max(e, 0), m))
            above.append(most)
        assert torch.equal(grad(ends), grad(above)), ends


def test_many_groups_that_overlap(ck):
    """A thousand groups that each claim all rows: the work of one."""
    m, n, k = 700, 264, 288
    dy = _made((m, n), torch.bfloat16, 5)
    codes, scales = ck.quantize_experts_mxfp8(_made((2, n, k), torch.float32, 3, 0.05))
    codes, scales = codes.repeat(512, 1, 1), scales.repeat(512, 1, 1)
    ends = torch.tensor([m, 0] * 512, dtype=torch.int32, device="cuda")
    want = ck.grouped_input_grad_mxfp8(dy, codes[:1], scales[:1], ends[:1], out_dtype=torch.float32)
    got = ck.grouped_input_grad_mxfp8(dy, codes, scales, ends, out_dtype=torch.float32)
    # the same exact products; another kernel may add them in another order
    magnitude = dy.double().abs() @ ck.dequantize_mxfp8(codes[0], scales[0], torch.float32).double().abs()
    assert ((got.double() - want.double()).abs() <= 2 * ((n / 16 + 4) * 2.0**-22 + 2.0**-24) * magnitude).all()
