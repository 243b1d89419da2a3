"""GatedLinear and its gradients through autograd, 8-bit linear layers, and FeedForward as both schedules' mlp_fn,
against plain torch arithmetic."""
import pytest
import torch

import feed_forward_reference as R
import tokenweave_amd as tw
from tokenweave_amd import ops

pytestmark = pytest.mark.gpu
DEV, BF16 = "cuda:0", torch.bfloat16
H, INNER, EPS = 256, 400, 1e-5


def filled(layer, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    layer = layer.to(DEV)
    for p in layer.parameters():
        p.data.copy_(torch.randn(p.shape, generator=g, device=DEV) * p.shape[-1] ** -0.5)
    return layer


@pytest.mark.parametrize("shape", [(5,), (3, 7), (2, 3, 50), (0,), (300,)])
@pytest.mark.parametrize("kind", R.ACTIVATIONS)
def test_autograd(shape, kind):
    layer = filled(tw.GatedLinear(H, INNER, kind)).requires_grad_()
    x = torch.randn(*shape, H, device=DEV).to(BF16).requires_grad_()
    out = layer(x)
    assert out.shape == shape + (INNER,)
    grad = torch.randn(out.shape, device=DEV).to(BF16)
    out.backward(grad)
    rows, w = x.detach().reshape(-1, H), layer.weight.detach()
    want, bound, both, off = R.gated(rows, w, kind)
    R.assert_within(out.detach().view(-1, INNER), want, bound, "out")
    kept = torch.empty((rows.shape[0], 2 * INNER), dtype=BF16, device=DEV)
    ops.gated_gemm_bf16_nt(torch.empty((rows.shape[0], INNER), dtype=BF16, device=DEV), rows, w, kind, gate_up=kept)
    gx, bx, gw, bw = R.gated_gradients(grad.view(-1, INNER), rows, w, kept, kind)
    R.assert_within(x.grad.view(-1, H), gx, bx, "x.grad")
    R.assert_within(layer.weight.grad, gw, bw, "weight.grad")
    with torch.no_grad():
        assert torch.equal(layer(x), out)


def test_only_what_is_wanted_and_gradients_of_any_layout():
    layer = filled(tw.GatedLinear(H, INNER))
    x = torch.randn(64, H, device=DEV).to(BF16)
    assert not layer(x).requires_grad
    x.requires_grad_()
    layer(x).sum().backward()                  # an expanded gradient
    first = x.grad.clone()
    x.grad = None
    layer(x).backward(torch.ones(INNER, 64, device=DEV, dtype=BF16).t())
    assert torch.equal(x.grad, first) and layer.weight.grad is None
    layer.requires_grad_()
    layer(x.detach()).sum().backward()
    assert layer.weight.grad is not None
    y = layer(x.detach()[:, :]).sum()
    (g,) = torch.autograd.grad(y, layer.weight)
    assert torch.equal(g, layer.weight.grad)


def test_gradients_follow_differences():
    """Along a direction of both operands: the loss moves as the gradients say.  fp32 sums of bf16 outputs: each of
    the outputs is off by 2^-8 of itself or less, so the difference of two sums by twice that of their size."""
    layer = filled(tw.GatedLinear(H, INNER)).requires_grad_()
    x = torch.randn(40, H, device=DEV).to(BF16).requires_grad_()
    c = torch.randn(40, INNER, device=DEV)
    (layer(x).float() * c).sum().backward()
    step = 0.25
    dx, dw = (x.grad.sign() * step).to(BF16), torch.zeros_like(layer.weight)
    with torch.no_grad():
        up, down = ((layer(x + s * dx).double() * c).sum() for s in (1, -1))
        size = (layer(x + dx).abs().double() * c.abs()).sum() + (layer(x - dx).abs().double() * c.abs()).sum()
        # the operands move by what x +- dx is after its rounding; the third derivative is left to the oracle
        hi, lo = (x + dx).double(), (x - dx).double()
        exact = [(R.gated(z, layer.weight, "silu")[0] * c).sum() for z in (hi, lo)]
    assert abs((up - down) - (exact[0] - exact[1])) <= 2 ** -8 * size
    assert up > down and float(dw.abs().sum()) == 0


def test_a_capture_is_refused_where_a_gradient_is_recorded(monkeypatch):
    layer = filled(tw.GatedLinear(H, INNER)).requires_grad_()
    x = torch.randn(4, H, device=DEV).to(BF16)
    y = layer(x)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="gated_gemm_bf16_nt_backward"):
        layer(x)
    with pytest.raises(RuntimeError, match="gated_gemm_bf16_nt_backward"):
        y.sum().backward()
    assert layer.weight.grad is None


def test_ranks_of_a_whole_weight():
    gate, up = (torch.randn(INNER, H, device=DEV).to(BF16) for _ in range(2))
    x = torch.randn(9, H, device=DEV).to(BF16)
    whole = tw.GatedLinear(H, INNER).to(DEV)
    parts = [tw.GatedLinear(H, INNER, tp_rank=r, tp_size=4).to(DEV) for r in range(4)]
    for layer in (whole, *parts):
        layer.weight_loader(layer.weight, gate, 0)
        layer.weight_loader(layer.weight, up, 1)
    assert torch.equal(torch.cat([p(x) for p in parts], -1), whole(x))


@pytest.mark.parametrize("M", [1, 40, 300])
def test_row_parallel_layer_of_8_bits(M):
    layer = filled(tw.RowParallelLinear(400, 264, bias=True))
    whole = layer.weight.data.clone()
    tw.Fp8BlockLinearMethod().process_weights(layer)
    assert layer.weight.dtype == torch.float8_e4m3fn and layer.weight_scale.shape == (3, 4)
    x = torch.randn(M, 400, device=DEV).to(BF16)
    got = layer(x)[0]
    codes, scales = R.codes(x.double())
    w_codes, w_scales = R.weight_codes(whole)
    assert torch.equal(layer.weight_scale, w_scales) and torch.equal(layer.weight.float(), w_codes.float())
    want, off = R.block_product(codes, scales, w_codes, w_scales)
    rounded = want.to(BF16).double()
    # the product rounded, the bias added to it, the sum rounded
    bound = off + R.half(BF16) * (want.abs() * 2 + (rounded + layer.bias.double()).abs()) + 1e-30
    R.assert_within(got, want + layer.bias.double(), bound, "out")
    out = torch.zeros(M, 264, dtype=BF16, device=DEV)
    assert torch.equal(layer(x, out, is_tokenweave=True)[0], got)


@pytest.mark.parametrize("T", [1, 24, 330])
@pytest.mark.parametrize("fp8", [False, True])
def test_block(T, fp8):
    block = filled(tw.FeedForward(H, INNER))
    gate_up, down = block.gate_up.weight.data.clone(), block.down.weight.data.clone()
    if fp8:
        block.to_fp8_blocks()
    x = torch.randn(T, H, device=DEV).to(BF16)
    hidden = x.clone()
    assert block(hidden) is hidden
    inner = R.gated(x, gate_up, "silu")[0]
    want = inner @ down.double().t()
    rel = float((hidden.double() - want).norm() / want.norm())
    # bf16: one rounding inside, one at the end, 2^-9 of their values each in the mean square at most; 8 bits: four
    # roundings to codes, 2^-4 each at most, which add up as squares (and the rounded sums between)
    assert rel <= (2 * 2 ** -4 + 2 ** -7 if fp8 else 2 ** -7), rel
    if fp8:
        c, s = R.codes(x.double())
        both = R.block_product(c, s, *R.weight_codes(gate_up))[0].to(BF16)
        c, s = R.codes(R.act(both.double()[:, :INNER], "silu") * both.double()[:, INNER:])
        want = R.block_product(c, s, *R.weight_codes(down))[0]
        # against the same steps: codes that land on the other side of a border, few, 2^-3 of a value each
        assert float((hidden.double() - want).norm() / want.norm()) <= 2 ** -6


class Layer:
    """A decoder layer with the package's feed-forward block and an attention that is a projection."""

    def __init__(self, seed, fp8):
        self.input_layernorm, self.post_attention_layernorm = (tw.RMSNorm(H, eps=EPS, dtype=BF16).to(DEV) for _ in range(2))
        self.o = filled(tw.RowParallelLinear(H, H, bias=False), seed)
        # a rank of two has 200 channels inside, which 8-bit rows cannot have
        self.mlp = filled(tw.FeedForward(H, INNER, tp_rank=0, tp_size=1 if fp8 else 2), seed + 1)
        if fp8:
            self.mlp.to_fp8_blocks()

    def self_attn(self, positions, hidden_states, gemm_cus=None, **kwargs):
        self.o(hidden_states.clone(), hidden_states, is_tokenweave=True, gemm_cus=gemm_cus)


def run_layers(T, woven, fp8, cus=0):
    buf = tw.PartialsBuffer(2, T, H, rank=0, device=DEV)
    buf.storage.zero_()
    stack = [Layer(20 + 2 * i, fp8) for i in range(2)]
    final = tw.RMSNorm(H, eps=EPS, dtype=BF16).to(DEV)
    g = torch.Generator(device=DEV).manual_seed(9)
    hidden = buf.hidden_states(T)
    hidden.copy_(torch.randn(T, H, generator=g, device=DEV).to(BF16))
    residual, positions = torch.empty_like(hidden), torch.arange(T, device=DEV)
    cur, side = torch.cuda.current_stream(), torch.cuda.Stream()
    for i, layer in enumerate(stack):
        nxt = stack[i + 1].input_layernorm if i + 1 < len(stack) else final
        if woven:
            tw.tokenweave_overlap(layer, positions, hidden, residual, buf, i, end_layer=2, rank=0, world_size=2,
                                  current_stream=cur, copy_stream=side, next_layer_norm=nxt,
                                  split_size=tw.tokenweave_split_size(T), actual_tokens=T, num_tokens_padded=T,
                                  MAX_CTAS_ATTN=16, MAX_CTAS_MLP=16, mlp_fn=layer.mlp, all_ranks=True, gemm_cus=cus)
        else:
            tw.tokenweave_with_fuse_only(layer, positions, hidden, residual, buf, i, rank=0, world_size=2,
                                         next_layer_norm=nxt, actual_tokens=T, nearest_multiple_of_world_size=T,
                                         MAX_CTAS_ATTN=0, MAX_CTAS_MLP=0, mlp_fn=layer.mlp, all_ranks=True)
    torch.cuda.synchronize()
    return hidden.clone(), residual.clone()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("cus", [0, 96])
def test_as_the_schedules_mlp(fp8, cus):
    """Both splits have the kernels of the whole batch's size here, whose sums do not depend on the rows beside them:
    the woven layers' results are the unsplit ones' to the bit."""
    T = 1024
    y0, r0 = run_layers(T, False, fp8)
    y1, r1 = run_layers(T, True, fp8, cus)
    assert torch.equal(r0, r1) and torch.equal(y0, y1)


def test_two_streams_at_once():
    """The whole of it on two streams with operands of their own, many times: nothing is shared."""
    def work(seed, T):
        g = torch.Generator(device=DEV).manual_seed(seed)
        x = torch.randn(T, H, generator=g, device=DEV).to(BF16)
        w = (torch.randn(2 * INNER, H, generator=g, device=DEV) * H ** -0.5).to(BF16)
        dh = torch.randn(T, INNER, generator=g, device=DEV).to(BF16)
        block = filled(tw.FeedForward(H, INNER), seed).to_fp8_blocks()
        out, both = (torch.empty(T, n, dtype=BF16, device=DEV) for n in (INNER, 2 * INNER))
        dx, dw = torch.empty_like(x), torch.empty_like(w)

        def run():
            ops.gated_gemm_bf16_nt(out, x, w, gate_up=both)
            ops.gated_gemm_bf16_nt_backward(dx, dw, dh, x, w, both)
            return [t.clone() for t in (out, both, dx, dw)] + [block(x.clone())]
        return run

    pair = [work(1, 300), work(2, 40)]
    want = [run() for run in pair]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in pair]
    got = [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(pair[i]())
    torch.cuda.synchronize()
    for i in range(2):
        for results in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(results, want[i]))
