"""The gated product and its gradients against 64 bits: every row count at which another kernel or tile serves, odd
sizes, views, the smallest and the ragged; captured calls; values that are not numbers."""
import pytest
import torch

import feed_forward_reference as R
from tokenweave_amd import ops

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def make(M, inner, K, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((M, K), generator=g, device="cuda").to(BF16)
    w = (torch.randn((2 * inner, K), generator=g, device="cuda") * (scale * K ** -0.5)).to(BF16)
    return x, w


def wide(rows, width, extra=12):
    """A row slice of a wider buffer, and the buffer, whose other places hold a mark."""
    buf = torch.full((rows + 2, width + extra), 777.0, dtype=BF16, device="cuda")
    return buf[1:1 + rows, 4:4 + width], buf


def untouched(buf, rows, width):
    keep = buf.clone()
    keep[1:1 + rows, 4:4 + width] = 777.0
    return bool((keep == 777.0).all())


def check_forward(M, inner, K, kind, seed=0, max_cus=None):
    x, w = make(M, inner, K, seed)
    out, buf = wide(M, inner)
    both, both_buf = wide(M, 2 * inner, 16)
    ops.gated_gemm_bf16_nt(out, x, w, kind, max_cus, gate_up=both)
    want, bound, products, off = R.gated(x, w, kind)
    R.assert_within(out, want, bound, "out")
    R.assert_within(both, products, off, "gate_up")
    assert untouched(buf, M, inner) and untouched(both_buf, M, 2 * inner)
    again = torch.empty((M, inner), dtype=BF16, device="cuda")
    ops.gated_gemm_bf16_nt(again, x, w, kind, max_cus)
    assert torch.equal(again, out), "the same call without gate_up gives other bits"
    return x, w, both.contiguous(), out


@pytest.mark.parametrize("M", [1, 2, 7, 8, 9, 16, 17, 31, 32, 33, 40, 41, 48, 64, 65, 72, 80, 96, 97, 128])
@pytest.mark.parametrize("inner,K", [(4, 8), (100, 72), (704, 1024), (260, 136)])
def test_few_rows(M, inner, K):
    check_forward(M, inner, K, R.ACTIVATIONS[M % 3], seed=M)


@pytest.mark.parametrize("M", [129, 160, 200, 256, 257, 300, 384, 511, 1001])
@pytest.mark.parametrize("inner,K", [(32, 64), (100, 72), (704, 1024), (1376, 520), (36, 8)])
def test_many_rows(M, inner, K):
    check_forward(M, inner, K, R.ACTIVATIONS[M % 3], seed=M)


@pytest.mark.parametrize("M,inner,K", [(1000, 2048, 256), (2458, 1376, 192), (700, 3696, 320), (4096, 512, 64)])
def test_all_tile_shapes(M, inner, K):
    check_forward(M, inner, K, "silu", seed=M)


@pytest.mark.parametrize("M", [5, 64, 300])
def test_grid_caps_give_the_same_bits(M):
    x, w = make(M, 704, 520)
    outs = []
    for cap in (None, 1, 3, 64):
        out = torch.empty((M, 704), dtype=BF16, device="cuda")
        ops.gated_gemm_bf16_nt(out, x, w, "gelu", cap)
        outs.append(out)
    assert all(torch.equal(o, outs[0]) for o in outs)


def test_products_that_are_large_or_no_numbers():
    """An infinity or a NaN stays in its row (of x) or its column (of b); saturated gates are exact zeros and products."""
    for M in (3, 200):
        x, w = make(M, 64, 64)
        x[1, 5] = float("inf")
        w[7, 3] = float("nan")       # a gate row
        w[64 + 9, 3] = float("inf")  # an up row
        out = torch.empty((M, 64), dtype=BF16, device="cuda")
        ops.gated_gemm_bf16_nt(out, x, w)
        ok = torch.ones_like(out, dtype=torch.bool)
        ok[1], ok[:, 7], ok[:, 9] = False, False, False
        assert torch.isfinite(out[ok]).all() and torch.isnan(out[:, 7]).all() and not torch.isfinite(out[:, 9]).any()
        x, w = make(M, 64, 64, scale=100.0)
        for kind in R.ACTIVATIONS:
            ops.gated_gemm_bf16_nt(out, x, w, kind)
            want, bound, _, _ = R.gated(x, w, kind)
            R.assert_within(out, want, bound + 1e-35, kind)


@pytest.mark.parametrize("M,inner,K", [(1, 4, 8), (3, 36, 72), (64, 64, 64), (65, 100, 136), (129, 100, 72), (257, 704, 520),
                                       (1001, 260, 1024), (7, 704, 1024), (64, 1376, 520), (300, 100, 2048),
                                       (64, 2100, 264), (2, 2048, 128), (4000, 36, 72), (130, 4100, 136)])
@pytest.mark.parametrize("kind", R.ACTIVATIONS)
def test_gradients(M, inner, K, kind):
    x, w, both, out = check_forward(M, inner, K, kind)
    grad_buf = torch.randn((M, inner + 8), device="cuda").to(BF16)
    grad = grad_buf[:, 4:4 + inner]
    gx, gw = torch.empty_like(x), torch.empty_like(w)
    ops.gated_gemm_bf16_nt_backward(gx, gw, grad, x, w, both, kind)
    want_x, bound_x, want_w, bound_w = R.gated_gradients(grad, x, w, both, kind)
    R.assert_within(gx, want_x, bound_x, "grad_x")
    R.assert_within(gw, want_w, bound_w, "grad_w")
    only_x, only_w = torch.full_like(x, 5.0), torch.full_like(w, 5.0)
    ops.gated_gemm_bf16_nt_backward(only_x, None, grad, x, w, both, kind)
    ops.gated_gemm_bf16_nt_backward(None, only_w, grad, x, w, both, kind)
    assert torch.equal(only_x, gx) and torch.equal(only_w, gw)


def test_slopes_far_out_are_finite():
    """Gates of +-3e38 and of 0: slopes of 1, 0 and 1/2, not a product of zero and infinity."""
    gate = torch.tensor([[3e38, -3e38, 0.0, -90.0, 90.0, -5e19, 5e19, 1.0]], device="cuda").to(BF16)
    up = torch.ones_like(gate)
    x = torch.ones((1, 8), dtype=BF16, device="cuda")
    w = torch.zeros((16, 8), dtype=BF16, device="cuda")
    for kind in R.ACTIVATIONS:
        gw = torch.empty_like(w)
        ops.gated_gemm_bf16_nt_backward(None, gw, torch.ones_like(gate) * 1e-3, x, w, torch.cat((gate, up), 1), kind)
        assert torch.isfinite(gw).all()
        want = R.slope(gate.double(), kind)[0] * float(torch.tensor(1e-3).to(BF16))
        R.assert_within(gw[:8, 0], want, want.abs() * 2 ** -7 + 1e-8, kind)


@pytest.mark.parametrize("M", [2, 130])
def test_weight_halves_more_than_two_gib_apart(M):
    inner, K = 69632, 16384
    x = make(M, 4, K)[0]
    w = torch.empty((2 * inner, K), dtype=BF16, device="cuda")
    for part in w.split(8192):
        part.normal_(0, K ** -0.5)
    out = torch.empty((M, inner), dtype=BF16, device="cuda")
    ops.gated_gemm_bf16_nt(out, x, w)
    at = torch.tensor([0, 1, 127, 128, 35000, inner - 129, inner - 1], device="cuda")
    want, bound, _, _ = R.gated(x, torch.cat((w[at], w[inner + at])), "silu")
    R.assert_within(out[:, at], want, bound, "out")


def test_no_rows():
    x, w = make(0, 36, 72)
    ops.gated_gemm_bf16_nt(torch.empty((0, 36), dtype=BF16, device="cuda"), x, w,
                           gate_up=torch.empty((0, 72), dtype=BF16, device="cuda"))
    gx, gw = torch.empty_like(x), torch.full_like(w, 3.0)
    ops.gated_gemm_bf16_nt_backward(gx, gw, torch.empty((0, 36), dtype=BF16, device="cuda"), x, w,
                                    torch.empty((0, 72), dtype=BF16, device="cuda"))
    assert (gw == 0).all()


@pytest.mark.parametrize("M", [7, 300])
def test_captured_and_on_another_stream(M):
    x, w = make(M, 100, 136)
    out, both = (torch.empty((M, n), dtype=BF16, device="cuda") for n in (100, 200))
    grad = torch.randn((M, 100), device="cuda").to(BF16)
    gx, gw = torch.empty_like(x), torch.empty_like(w)

    def step():
        ops.gated_gemm_bf16_nt(out, x, w, "gelu_tanh", gate_up=both)
        ops.gated_gemm_bf16_nt_backward(gx, gw, grad, x, w, both, "gelu_tanh")

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for seed in range(3):
        x2, w2 = make(M, 100, 136, seed + 5)
        x.copy_(x2), w.copy_(w2)
        step()
        torch.cuda.synchronize()
        want = [t.clone() for t in (out, both, gx, gw)]
        for t in (out, both, gx, gw):
            t.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(t, o) for t, o in zip((out, both, gx, gw), want)), seed


def test_both_routes_give_the_same_bits(monkeypatch):
    x, w = make(70, 100, 136)
    a, b = (torch.empty((70, 100), dtype=BF16, device="cuda") for _ in range(2))
    ops.gated_gemm_bf16_nt(a, x, w)
    monkeypatch.setattr(ops, "_fast", None)
    ops.gated_gemm_bf16_nt(b, x, w)
    assert torch.equal(a, b)


@pytest.mark.parametrize("M,inner,K", [(1, 4, 8), (70, 100, 136), (300, 36, 200), (64, 2100, 264), (129, 64, 72)])
def test_what_a_workspace_held_does_not_matter(M, inner, K):
    """Not-a-numbers left in the workspace; gradients that begin 8, 16 and 64 bytes into a buffer."""
    from tokenweave_amd import _lib
    x, w = make(M, inner, K)
    both = torch.empty((M, 2 * inner), dtype=BF16, device="cuda")
    ops.gated_gemm_bf16_nt(torch.empty((M, inner), dtype=BF16, device="cuda"), x, w, gate_up=both)
    grad = torch.randn((M, inner), device="cuda").to(BF16)
    L = _lib.lib()
    size = L.tw_gated_gemm_bf16_nt_backward_workspace(M, inner, K, 1, 1)
    space = torch.full((size // 2,), float("nan"), dtype=BF16, device="cuda")
    before = None
    for skip in (4, 8, 32):
        bufs = [torch.full((rows * K + 64,), 777.0, dtype=BF16, device="cuda") for rows in (M, 2 * inner)]
        gx, gw = (b[skip:skip + rows * K].view(rows, K) for b, rows in zip(bufs, (M, 2 * inner)))
        space.fill_(float("nan"))
        _lib.check(L.tw_gated_gemm_bf16_nt_backward(
            gx.data_ptr(), gw.data_ptr(), grad.data_ptr(), inner, x.data_ptr(), w.data_ptr(), both.data_ptr(), 2 * inner,
            M, inner, K, 0, 0, space.data_ptr(), size, torch.cuda.current_stream().cuda_stream))
        want_x, bound_x, want_w, bound_w = R.gated_gradients(grad, x, w, both, "silu")
        R.assert_within(gx, want_x, bound_x, "grad_x")
        R.assert_within(gw, want_w, bound_w, "grad_w")
        for b, rows in zip(bufs, (M, 2 * inner)):
            assert (b[:skip] == 777.0).all() and (b[skip + rows * K:] == 777.0).all()
        if before:
            assert torch.equal(gx, before[0]) and torch.equal(gw, before[1])
        before = gx.clone(), gw.clone()


@pytest.mark.parametrize("M,inner,K", [(129, 136, 72), (300, 8, 64), (257, 100, 72), (1001, 704, 264), (4096, 3584, 64),
                                       (2458, 1376, 192), (64, 136, 72)])
@pytest.mark.parametrize("kind", R.ACTIVATIONS)
def test_outputs_that_begin_anywhere(M, inner, K, kind):
    """out and gate_up 8, 16 and 64 bytes into a buffer, apart from one another: the same bits, and nothing beside them."""
    x, w = make(M, inner, K)

    def place(width, step):
        buf = torch.full((M + 2, (width + step - 1) // step * step + 2 * step), 777.0, dtype=BF16, device="cuda")
        return buf, buf[1:1 + M, step:step + width]

    plain, both = (torch.empty((M, n), dtype=BF16, device="cuda") for n in (inner, 2 * inner))
    ops.gated_gemm_bf16_nt(plain, x, w, kind, gate_up=both)
    want, bound, products, off = R.gated(x, w, kind)
    R.assert_within(plain, want, bound, "out")
    R.assert_within(both, products, off, "gate_up")
    for step, step_both in ((4, 32), (8, 8), (32, 4), (32, 8), (8, 32), (32, 32)):
        buf, out = place(inner, step)
        both_buf, kept = place(2 * inner, step_both)
        ops.gated_gemm_bf16_nt(out, x, w, kind, gate_up=kept)
        assert torch.equal(out, plain) and torch.equal(kept, both), (step, step_both)
        out.fill_(777.0), kept.fill_(777.0)
        assert (buf == 777.0).all() and (both_buf == 777.0).all(), (step, step_both)


@pytest.mark.parametrize("M,inner,K", [(129, 100, 72), (1001, 704, 264), (1000, 1376, 520), (2458, 260, 1024), (4096, 512, 64),
                                       (700, 2100, 136)])
@pytest.mark.parametrize("max_cus", [None, 1, 7, 24, 100])
def test_gradients_together_and_alone(M, inner, K, max_cus):
    """Both gradients asked for at once, by whatever share of the units each then has, have the bits of either alone."""
    x, w = make(M, inner, K)
    both = torch.empty((M, 2 * inner), dtype=BF16, device="cuda")
    ops.gated_gemm_bf16_nt(torch.empty((M, inner), dtype=BF16, device="cuda"), x, w, gate_up=both)
    grad = torch.randn((M, inner), device="cuda").to(BF16)
    alone = torch.empty_like(x), torch.empty_like(w)
    ops.gated_gemm_bf16_nt_backward(alone[0], None, grad, x, w, both)
    ops.gated_gemm_bf16_nt_backward(None, alone[1], grad, x, w, both)
    want_x, bound_x, want_w, bound_w = R.gated_gradients(grad, x, w, both, "silu")
    R.assert_within(alone[0], want_x, bound_x, "grad_x")
    R.assert_within(alone[1], want_w, bound_w, "grad_w")
    gx, gw = torch.full_like(x, 777.0), torch.full_like(w, 777.0)
    ops.gated_gemm_bf16_nt_backward(gx, gw, grad, x, w, both, max_cus=max_cus)
    assert torch.equal(gx, alone[0]) and torch.equal(gw, alone[1])


@pytest.mark.parametrize("M,inner,K", [(33, 4, 8192), (64, 100, 6152), (96, 748, 6904), (129, 1376, 4096), (160, 748, 6904),
                                       (160, 3584, 8192), (256, 2048, 6144), (300, 1376, 4096), (256, 3584, 8192), (300, 36, 2048),
                                       (384, 3584, 8192), (512, 748, 6904), (1000, 36, 2048), (1024, 100, 4104)])
@pytest.mark.parametrize("kind", R.ACTIVATIONS)
def test_divided_along_k(M, inner, K, kind):
    """Some hundred rows, whose inner dimension is dealt out: against 64 bits, under grid caps, from any workspace."""
    from tokenweave_amd import _lib
    L = _lib.lib()
    size = L.tw_gated_gemm_bf16_nt_workspace(M, inner, K)
    assert size > 0, "this size is not divided any more: the test needs another"
    x, w, both, out = check_forward(M, inner, K, kind)
    for max_cus in (1, 24, 100):
        again, kept = torch.full_like(out, 777.0), torch.full_like(both, 777.0)
        ops.gated_gemm_bf16_nt(again, x, w, kind, max_cus, gate_up=kept)
        assert torch.equal(again, out) and torch.equal(kept, both), max_cus
    space = torch.full((size // 4 + 64,), float("nan"), device="cuda")
    again = torch.empty((M, inner), dtype=BF16, device="cuda")
    _lib.check(L.tw_gated_gemm_bf16_nt(again.data_ptr(), None, x.data_ptr(), w.data_ptr(), M, inner, K, inner, 0,
                                       R.ACTIVATIONS.index(kind), 0, space.data_ptr(), size,
                                       torch.cuda.current_stream().cuda_stream))
    assert torch.equal(again, out) and torch.isnan(space[size // 4:]).all()


def test_divided_along_k_captured():
    """Two captured calls beside each other on two streams, replayed between eager ones."""
    shapes = ((160, 748, 2048), (96, 748, 6904))
    sets = []
    for seed, (M, inner, K) in enumerate(shapes):
        x, w = make(M, inner, K, seed)
        sets.append((torch.empty((M, inner), dtype=BF16, device="cuda"), x, w))
    for s in sets:
        ops.gated_gemm_bf16_nt(*s)
    torch.cuda.synchronize()
    graphs, streams = [], [torch.cuda.Stream() for _ in sets]
    for s, stream in zip(sets, streams):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=stream):
            ops.gated_gemm_bf16_nt(*s)
    for turn in range(4):
        wants = []
        for seed, (s, (M, inner, K)) in enumerate(zip(sets, shapes)):
            x, w = make(M, inner, K, 10 * turn + seed)
            s[1].copy_(x), s[2].copy_(w)
            ops.gated_gemm_bf16_nt(*s)
            wants.append(s[0].clone())
            s[0].fill_(777.0)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for s, want in zip(sets, wants):
            assert torch.equal(s[0], want), turn
