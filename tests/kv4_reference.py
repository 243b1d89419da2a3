"""The rotation, the 4-bit cache and attention over it in 64 bits on the CPU, from the definitions, and
what the kernels may be off by."""
import math

import torch

GRID = torch.tensor((0, 0.5, 1, 1.5, 2, 3, 4, 6), dtype=torch.float64)
# unit roundoffs: half the distance of neighbouring values over the value
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
# half the distance of the smallest values
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}


def rotate(x, positions, cos_sin, interleaved, inverse=False):
    """[tokens, heads, D] in float64 by the table's own (fp32) values."""
    n = cos_sin.shape[1]
    x, row = x.double().cpu(), cos_sin.double().cpu()[positions.cpu()]
    z = torch.complex(row[:, None, :n // 2], row[:, None, n // 2:] * (-1 if inverse else 1))
    y = x.clone()
    if interleaved:
        pairs = torch.view_as_complex(x[..., :n].reshape(*x.shape[:-1], n // 2, 2).contiguous())
        y[..., :n] = torch.view_as_real(pairs * z).flatten(-2)
    else:
        pairs = torch.complex(x[..., :n // 2].contiguous(), x[..., n // 2:n].contiguous()) * z
        y[..., :n // 2], y[..., n // 2:n] = pairs.real, pairs.imag
    return y


def rotate_bound(x, want, dtype, n, interleaved, largest=1.0):
    """One rounding to the output's type; two products and a sum in fp32, each off by at most 2^-24 of what
    it rounds, of values up to `largest` (|x1| + |x2|)."""
    a = x.double().cpu().abs()
    s = torch.zeros_like(a)
    if interleaved:
        s[..., :n] = (a[..., 0:n:2] + a[..., 1:n:2]).repeat_interleave(2, -1)
    else:
        s[..., :n] = (a[..., :n // 2] + a[..., n // 2:n]).repeat(1, 1, 2)
    return U[dtype] * want.abs() * (1 + 2.0 ** -10) + 3 * 2.0 ** -24 * s * largest + 2.0 ** -126 + TINY[dtype]


def quantise(x):
    """What the cache holds of [..., D]: per 32 channels the nearest value of the grid at the smallest
    power of two that keeps the block within 7, in [2^-23, 2^13]; ties to the even code."""
    b = x.double().cpu().unflatten(-1, (-1, 32))
    most = b.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(torch.where(most.isfinite(), most, torch.ones_like(most)))   # most = m 2^e, m in [0.5, 1)
    e = torch.where(m > 0.875, e - 2, e - 3)                                        # 7 2^e = 0.875 2^(e + 3)
    e = torch.where(most == 0, torch.full_like(e, -23), e).clamp(-23, 13)
    size = 2.0 ** e.double()
    # (far behind the grid's end all its values are equally far in 64 bits)
    away = ((b.abs() / size).clamp(max=8.0)[..., None] - GRID).abs() + torch.tensor((0, 1) * 4, dtype=torch.float64) * 1e-13
    y = GRID[away.nan_to_num(0.0).argmin(-1)] * torch.where(b < 0, -1.0, 1.0) * size
    return torch.where(most.isfinite(), y, torch.full_like(y, math.nan)).flatten(-2)


def page_bytes(k, v):
    """Bytes of whole pages [pages, heads, page * (D + D/16)] from keys and values [pages, heads, page, D]
    that the cache holds exactly: byte by byte from the layout's definition."""
    N, H, P, D = k.shape
    out = torch.zeros((N, H, P * (D + D // 16)), dtype=torch.uint8)
    for first, scales, x in ((0, P * D, k), (P * D // 2, P * D + P * (D // 32), v)):
        b = x.double().unflatten(-1, (-1, 32))
        e = torch.full(b.shape[:-1], -23, dtype=torch.float64)
        # the smallest scale at which every value is on the grid
        for step in range(13, -24, -1):
            on = ((b.abs() / 2.0 ** step)[..., None] == GRID).any(-1).all(-1)
            e = torch.where(on, torch.full_like(e, step), e)
        code = ((b.abs() / 2.0 ** e[..., None])[..., None] == GRID).int().argmax(-1)
        assert (GRID[code] * 2.0 ** e[..., None] == b.abs()).all()
        code = (code + 8 * (b < 0)).flatten(-2)
        byte = (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8)             # [N, H, P, D/2]
        w = D // 32
        for t in range(P):
            for i in range(D // 2):
                at = t * (D // 2) + i if first == 0 else (t // 4) * 2 * D + (i // w) * 4 * w + (t % 4) * w + i % w
                out[:, :, first + at] = byte[:, :, t, i]
            for g in range(D // 32):
                out[:, :, scales + g * P + t] = (e[:, :, t, g] + 127).to(torch.uint8)
    return out


def attend(q, keys, values, lengths, news, scale, window=0):
    """Per sequence: keys, values [heads, length, D] in float64.  Returns the output, and for every value of
    it the p-weighted mean of |v| and the row's largest sum of |q k| scale, which bound its error."""
    out, mean, size, first = [], [], [], 0
    G = q.shape[1] // (keys[0].shape[0] if keys else 1)
    for k, v, n, m in zip(keys, values, lengths, news):
        x = q[first:first + m].double().cpu().transpose(0, 1)
        first += m
        k, v = k.repeat_interleave(G, 0), v.repeat_interleave(G, 0)
        last = n - m + torch.arange(m)[:, None]
        t = torch.arange(n)
        sees = (t <= last) & ((t > last - window) if window else torch.ones_like(t, dtype=torch.bool))
        s = (x @ k.transpose(1, 2) * scale).masked_fill(~sees, -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300)) if n else s
        p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
        p = torch.where(sees, p, torch.zeros_like(p))
        v = torch.where(torch.ones_like(v, dtype=torch.bool), v, v)
        out.append((p @ v).transpose(0, 1))
        mean.append((p @ v.abs()).transpose(0, 1))
        big = ((x.abs() @ k.abs().transpose(1, 2)) * scale).masked_fill(~sees, 0.0)
        size.append((big.amax(-1) if n else torch.zeros(G * k.shape[0] // max(G, 1), m))[..., None].expand(-1, -1, q.shape[2]).transpose(0, 1))
    return torch.cat(out), torch.cat(mean), torch.cat(size)


def attend_bound(out, mean, size, dtype, tokens):
    """The output's rounding; the probabilities' rounding to fp16 (2^-11 each) and their sums in fp32; a
    score's error, at most 2^-21 of the sum of |q k| (fp32 sums of up to 256 products, matrix units that
    may cut instead of round), twice: in the probability and in the sum that it is divided by."""
    return (U[dtype] * out.abs() * (1 + 2.0 ** -8) + mean * (2.0 ** -11 + 2 * size * 2.0 ** -21 + tokens * 2.0 ** -24)
            + 2.0 ** -25)
