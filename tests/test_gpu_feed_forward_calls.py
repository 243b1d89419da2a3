"""Calls of the feed-forward half that the documentation allows: any leading dimensions, single rows of odd buffers, scales
of any layout, grid caps, every tile shape that the rules may choose."""
import ctypes

import pytest
import torch

import feed_forward_reference as R
import tokenweave_amd as tw
from tokenweave_amd import ops

pytestmark = pytest.mark.gpu
DEV, BF16, FP8 = "cuda:0", torch.bfloat16, torch.float8_e4m3fn


def filled(layer, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    layer = layer.to(DEV)
    for p in layer.parameters():
        p.data.copy_(torch.randn(p.shape, generator=g, device=DEV) * p.shape[-1] ** -0.5)
    return layer


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("shape", [(2, 9), (3, 1, 2), (2, 0), (1,)])
def test_a_block_of_any_leading_dimensions(shape, fp8):
    block = filled(tw.FeedForward(256, 400))
    if fp8:
        block.to_fp8_blocks()
    x = torch.randn(*shape, 256, device=DEV).to(BF16)
    want = block(x.view(-1, 256).clone())
    hidden = x.clone()
    assert block(hidden) is hidden and torch.equal(hidden.view(-1, 256), want)


class KernelNode(ctypes.Structure):
    """hipKernelNodeParams"""
    _fields_ = [("block", ctypes.c_uint32 * 3), ("extra", ctypes.c_void_p), ("func", ctypes.c_void_p),
                ("grid", ctypes.c_uint32 * 3), ("params", ctypes.c_void_p), ("lds", ctypes.c_uint32)]


def grids(call):
    """The workgroups of each kernel that a call launches, from the graph that captures it."""
    hip = ctypes.CDLL("libamdhip64.so.7")
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        call()
    raw, count = ctypes.c_void_p(graph.raw_cuda_graph()), ctypes.c_size_t(0)
    assert hip.hipGraphGetNodes(raw, None, ctypes.byref(count)) == 0
    nodes = (ctypes.c_void_p * count.value)()
    assert hip.hipGraphGetNodes(raw, nodes, ctypes.byref(count)) == 0
    sizes = []
    for node in nodes:
        kind, params = ctypes.c_int(-1), KernelNode()
        assert hip.hipGraphNodeGetType(ctypes.c_void_p(node), ctypes.byref(kind)) == 0 and kind.value == 0
        assert hip.hipGraphKernelNodeGetParams(ctypes.c_void_p(node), ctypes.byref(params)) == 0
        sizes.append(params.grid[0] * params.grid[1] * params.grid[2])
    return sizes


@pytest.mark.parametrize("M,inner,K", [(5, 100, 72), (300, 36, 2048), (160, 748, 6904), (64, 2100, 264), (1001, 704, 1024), (0, 36, 72)])
@pytest.mark.parametrize("cap", [1, 24, 100])
def test_gated_calls_keep_their_cap(M, inner, K, cap):
    """Every kernel of a capped call, the ones beside the products too, leaves the other units alone, and no bit
    depends on the cap."""
    x, w = (torch.randn(n, K, device=DEV).to(BF16) for n in (M, 2 * inner))
    grad = torch.randn(M, inner, device=DEV).to(BF16)

    def outputs():
        return [torch.full(s, 777.0, dtype=BF16, device=DEV) for s in ((M, inner), (M, 2 * inner), (M, K), (2 * inner, K))]

    def run(out, both, gx, gw, max_cus):
        ops.gated_gemm_bf16_nt(out, x, w, "silu", max_cus, gate_up=both)
        ops.gated_gemm_bf16_nt_backward(gx, gw, grad, x, w, both, "silu", max_cus)

    want, got = outputs(), outputs()
    run(*want, None), run(*got, cap)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    sizes = grids(lambda: run(*got, cap))
    assert len(sizes) >= (1 if M == 0 else 3) and max(sizes) <= cap, sizes


@pytest.mark.parametrize("M,N,K", [(5, 700, 528), (96, 1024, 8192), (1000, 1024, 8192), (1000, 1376, 272)])
@pytest.mark.parametrize("cap", [1, 24, 100])
def test_8_bit_products_keep_their_cap(M, N, K, cap):
    codes, scales = torch.empty((M, K), dtype=FP8, device=DEV), ops.fp8_group_scales(M, K)
    ops.quant_fp8_groups(codes, scales, torch.randn(M, K, device=DEV))
    w, sw = R.weight_codes(torch.randn(N, K, device=DEV))
    want, got = (torch.full((M, N), 777.0, dtype=BF16, device=DEV) for _ in range(2))
    ops.gemm_fp8_block_nt(want, codes, scales, w, sw)
    ops.gemm_fp8_block_nt(got, codes, scales, w, sw, cap)
    assert torch.equal(got, want)
    sizes = grids(lambda: ops.gemm_fp8_block_nt(got, codes, scales, w, sw, cap))
    assert sizes and max(sizes) <= cap, sizes


@pytest.mark.parametrize("route", ["direct", "ctypes"])
def test_a_single_row_of_a_buffer_whose_rows_are_odd(route, monkeypatch):
    """One row has no distance to another: its stride, which no alignment fits, is not looked at."""
    if route == "ctypes":
        monkeypatch.setattr(ops, "_fast", None)

    def row(width, dtype=BF16):
        return torch.zeros(3 * (width + 9), dtype=dtype, device=DEV).as_strided((1, width), (width + 9, 1))

    x, w = torch.randn(1, 72, device=DEV).to(BF16), torch.randn(200, 72, device=DEV).to(BF16)
    out, both, grad = row(100), row(200), row(100)
    grad.copy_(torch.randn(1, 100))
    ops.gated_gemm_bf16_nt(out, x, w, gate_up=both)
    want, kept = torch.empty(1, 100, dtype=BF16, device=DEV), torch.empty(1, 200, dtype=BF16, device=DEV)
    ops.gated_gemm_bf16_nt(want, x, w, gate_up=kept)
    assert torch.equal(out, want) and torch.equal(both, kept)
    gw, want_gw = torch.empty_like(w), torch.empty_like(w)
    ops.gated_gemm_bf16_nt_backward(None, gw, grad, x, w, both)
    ops.gated_gemm_bf16_nt_backward(None, want_gw, grad.clone(memory_format=torch.contiguous_format), x, w, kept)
    assert torch.equal(gw, want_gw)
    codes, scales = torch.empty(1, 272, dtype=FP8, device=DEV), ops.fp8_group_scales(1, 272)
    x = row(272)
    x.copy_(torch.randn(1, 272))
    ops.quant_fp8_groups(codes, scales, x)
    w, sw = R.weight_codes(torch.randn(260, 272, device=DEV))
    out, want = row(260), torch.empty(1, 260, dtype=BF16, device=DEV)
    ops.gemm_fp8_block_nt(out, codes, scales, w, sw)
    ops.gemm_fp8_block_nt(want, codes, scales, w, sw)
    assert torch.equal(out, want)


@pytest.mark.parametrize("route", ["direct", "ctypes"])
def test_scales_whose_rows_end_between_two_of_the_next(route, monkeypatch):
    """Every second place of odd rows, and the same turned: no two scales share memory.  Where two do, the call raises."""
    if route == "ctypes":
        monkeypatch.setattr(ops, "_fast", None)
    M, K, groups = 5, 400, 4
    x, codes = torch.randn(M, K, device=DEV), torch.empty((M, K), dtype=FP8, device=DEV)
    want = R.codes(x.double())[1]
    for rows, columns, turn in ((M, groups, False), (groups, M, True)):
        buf = torch.full((rows, 2 * columns - 1), -1.0, device=DEV)
        scales = buf[:, ::2].t() if turn else buf[:, ::2]
        ops.quant_fp8_groups(codes, scales, x)
        assert torch.equal(scales, want) and (buf[:, 1::2] == -1.0).all()
    base = torch.empty(64, device=DEV)
    for strides in ((3, 1), (6, 2), (1, 4), (0, 1), (1, 0), (2, 2)):
        with pytest.raises(RuntimeError, match="share memory"):
            ops.quant_fp8_groups(codes, base.as_strided((M, groups), strides), x)


@pytest.mark.parametrize("kind", R.ACTIVATIONS)
def test_gradients_against_differences_of_the_64_bit_loss(kind):
    """The derivative of the loss along directions near the gradient of each operand: central differences of the 64-bit
    forward pass against the sum of gradient times direction, magnitudes included.

    A gradient may be off by its own bound and by what the rounding of the kept products to bf16 does to it: G and U off by
    `step` of themselves move U act'(G) by 1.13 |U| step + 0.8 |U| |G| step and act(G) by 1.13 |G| step (1.13 and 0.8: the
    largest first and second derivatives of the three)."""
    M, inner, K = 24, 60, 64
    g = torch.Generator(device=DEV).manual_seed(5)
    layer = filled(tw.GatedLinear(K, inner, kind), 6).requires_grad_()
    x = torch.randn(M, K, generator=g, device=DEV).to(BF16).requires_grad_()
    c = torch.randn(M, inner, generator=g, device=DEV).to(BF16)
    layer(x).backward(c)
    w = layer.weight.detach()
    x64, w64 = x.detach().double(), w.double()
    both = x64 @ w64.t()

    def loss(x, w):
        gate, up = (x @ w.t()).chunk(2, 1)
        return float((R.act(gate, kind) * up * c.double()).sum())

    _, bound_x, _, bound_w = R.gated_gradients(c, x.detach(), w, both.to(BF16), kind)
    gate, up = both.abs().chunk(2, 1)
    step = R.half(BF16)
    off = c.double().abs().repeat(1, 2) * step * 1.02 * torch.cat((up * (1.13 + 0.8 * gate), 1.13 * gate), 1)
    for grad, most, at in ((x.grad.double(), bound_x + off @ w64.abs(), lambda d: (x64 + d, w64)),
                           (layer.weight.grad.double(), bound_w + off.t() @ x64.abs(), lambda d: (x64, w64 + d))):
        # the bound means something: along the gradient the derivative is many times it
        assert float((grad * grad).sum()) > 8 * float((most * grad.abs()).sum())
        for _ in range(4):
            d = grad * torch.rand(grad.shape, generator=g, device=DEV, dtype=torch.float64)
            d, h = d / d.norm(), 1e-4
            slope = (loss(*at(h * d)) - loss(*at(-h * d))) / (2 * h)
            # 1e-4: h^2 / 6 of a third derivative of some 1e3, and 2^-48 of a loss of some 1e3 over h
            assert abs(float((grad * d).sum()) - slope) <= float((most * d.abs()).sum()) + 1e-4
