"""Plain forms in 64 bits of the gated product, its gradients, the 8-bit codes and their product, with the
bounds that the arithmetic of a kernel has to keep.  `half(t)`: the most that a rounding to type t is off, relative
to the value."""
import math

import torch

GROUP = 128
ACTIVATIONS = ("silu", "gelu", "gelu_tanh")
SUM = 2.0 ** -23     # a step of a sum in fp32, whatever the way it rounds
ACT = 2.0 ** -18     # the fp32 activation: a reciprocal, an exponential and a few products, of 2^-22 each or less


def half(dtype):
    return torch.finfo(dtype).eps / 2


def act(x, kind):
    if kind == "silu":
        return x * torch.sigmoid(x)
    if kind == "gelu":
        return x * 0.5 * torch.special.erfc(-x / math.sqrt(2))
    return x * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3))


def slope(x, kind):
    if kind == "silu":
        s = torch.sigmoid(x)
        return s + x * s * (1 - s)
    if kind == "gelu":
        return 0.5 * torch.special.erfc(-x / math.sqrt(2)) + x * torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)
    z = 2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)
    s = torch.sigmoid(z)
    return s + x * s * torch.sigmoid(-z) * 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * x ** 2)


def products(x, w):
    """Gate and up sums in 64 bits, and the most that fp32 sums of them can be off."""
    x, w = x.double(), w.double()
    return x @ w.t(), x.shape[1] * SUM * (x.abs() @ w.abs().t())


def gated(x, w, kind):
    """(out, its bound, both products, their bound)."""
    both, off = products(x, w)
    gate, up = both.chunk(2, 1)
    off_gate, off_up = off.chunk(2, 1)
    a = act(gate, kind)
    out = a * up
    # |act'| <= 1.13; the two errors meet in one product
    bound = (half(torch.bfloat16) + ACT) * out.abs() + 1.01 * (1.13 * off_gate * (up.abs() + off_up)
                                                              + (a.abs() + ACT) * off_up) + 1e-30
    return out, bound, both, half(torch.bfloat16) * both.abs() + off + 1e-30


def gated_gradients(grad, x, w, gate_up, kind):
    """(grad_x, bound, grad_w, bound) from the rounded products that the forward call kept."""
    gate, up = gate_up.double().chunk(2, 1)
    g, x, w = grad.double(), x.double(), w.double()
    d = torch.cat((g * up * slope(gate, kind), g * act(gate, kind)), 1)
    # of the slope, a sum of terms of both signs, the terms' sizes count
    size = torch.cat(((g * up).abs() * (1 + gate.abs() / 2), (g * act(gate, kind)).abs()), 1)
    off = half(torch.bfloat16) * d.abs() + ACT * size
    gx, gw = d @ w, d.t() @ x
    most = half(torch.bfloat16) + 1e-30
    bound_x = most * gx.abs() + (off + d.shape[1] * SUM * 1.01 * d.abs()) @ w.abs() + 1e-30
    bound_w = most * gw.abs() + (off + d.shape[0] * SUM * 1.01 * d.abs()).t() @ x.abs() + 1e-30
    return gx, bound_x, gw, bound_w


def spread(scales, n, axis):
    return scales.repeat_interleave(GROUP, axis).narrow(axis, 0, n)


def codes(y):
    """(codes as 64-bit values, scales in fp32) of rows y in 64 bits: the nearest of the 253 finite values, ties to the
    even code, found by looking."""
    rows, K = y.shape
    padded = torch.nn.functional.pad(y, (0, -K % GROUP)).view(rows, -1, GROUP)
    scales = (padded.abs().amax(2).clamp(min=float(torch.tensor(1e-10))) / 448).float()
    values = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().to(y.device)
    q = y / spread(scales, K, 1).double()
    above = torch.searchsorted(values, q.abs().contiguous()).clamp(1, 126)
    low, high = q.abs() - values[above - 1], values[above] - q.abs()
    at = torch.where((low < high) | ((low == high) & (above % 2 == 1)), above - 1, above)
    return torch.copysign(values[at], q), scales


def block_product(a, a_scales, b, b_scales):
    """(product, the most that a kernel's sums of it are off).

    The matrix instruction for 8-bit codes adds aligned eights of products first: it shifts them to the largest
    product's exponent E and keeps 13 bits below it (`test_what_the_instruction_keeps` looks at that), so each of
    the eight is off by at most half of 2^(E - 13), with 2^E <= the largest product <= the largest |a| times the
    largest |b| of the eight.  All sums above that are fp32's."""
    M, K = a.shape
    x = a.double() * spread(a_scales, K, 1).double()
    w = b.double() * spread(spread(b_scales, b.shape[0], 0), K, 1).double()
    eights = x.abs().view(M, -1, 8).amax(2) @ w.abs().view(b.shape[0], -1, 8).amax(2).t()
    return x @ w.t(), 8 * 2.0 ** -14 * eights + (K + 8) * SUM * (x.abs() @ w.abs().t()) + 1e-30


def weight_codes(w):
    """e4m3 codes and scales of 128 x 128 blocks, as a checkpoint holds them."""
    N, K = w.shape
    padded = torch.nn.functional.pad(w.float(), (0, -K % GROUP, 0, -N % GROUP))
    blocks = padded.view(padded.shape[0] // GROUP, GROUP, -1, GROUP)
    scales = (blocks.abs().amax((1, 3)).clamp(min=1e-10).double() / 448).float().contiguous()   # (one rounding)
    return (w.float() / spread(spread(scales, N, 0), K, 1)).clamp(-448, 448).to(torch.float8_e4m3fn), scales


def assert_within(got, want, bound, what):
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} outside, first at {bad.nonzero()[0].tolist()}: "
                           f"got {got[bad][0].item()}, want {want[bad][0].item()}, bound {bound[bad][0].item():.3g}")
