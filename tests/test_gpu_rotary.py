"""Rotation of queries and keys against complex multiplication in 64 bits."""
import pytest
import torch

import tokenweave_amd as tw
from kv4_reference import rotate, rotate_bound
from tokenweave_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def inputs(T, Hq, Hk, D, dtype, seed=1, length=5000):
    g = torch.Generator(device=DEV).manual_seed(seed)
    qkv = torch.randn(T, (Hq + 2 * Hk) * D, generator=g, device=DEV).to(dtype)
    q, k, v = (x.view(T, -1, D) for x in qkv.split((Hq * D, Hk * D, Hk * D), 1))
    return q, k, v, torch.randint(0, length, (T,), generator=g, device=DEV)


def check(got, x, positions, table, interleaved, inverse=False):
    want = rotate(x, positions, table, interleaved, inverse)
    far = (got.double().cpu() - want).abs()
    bound = rotate_bound(x, want, got.dtype, table.shape[1], interleaved, float(table.abs().max()))
    assert (far <= bound).all(), float((far - bound).max())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T, Hq, Hk, D, dim", [(1, 8, 1, 128, 128), (64, 8, 1, 128, 128), (33, 6, 1, 64, 32),
                                               (17, 12, 12, 96, 32), (5, 3, 3, 80, 80), (7, 2, 1, 80, 20),
                                               (3, 5, 1, 70, 34), (2, 1, 1, 3, 2), (1031, 28, 4, 256, 128)])
def test_against_complex_products(T, Hq, Hk, D, dim, interleaved, dtype):
    q, k, v, positions = inputs(T, Hq, Hk, D, dtype)
    layer = tw.RotaryPositions(D, dim, 5000, 500000.0, interleaved).to(DEV)
    q0, k0, v0 = q.clone(), k.clone(), v.clone()
    qo, ko = torch.empty_like(q0), torch.empty_like(k0)
    got = layer(positions, q, k, qo, ko)
    assert got[0] is qo and got[1] is ko
    assert torch.equal(q, q0) and torch.equal(k, k0)          # the inputs stay
    check(qo, q0, positions, layer.cos_sin, interleaved)
    check(ko, k0, positions, layer.cos_sin, interleaved)
    layer(positions, q, k)                                     # in place, views of the projections' output
    assert torch.equal(q, qo) and torch.equal(k, ko) and torch.equal(v, v0)


@pytest.mark.parametrize("scaling", [None, {"type": "linear", "factor": 4.0}, {"type": "ntk", "factor": 4.0},
                                     {"type": "bands", "factor": 8.0, "original_max_position": 8192},
                                     {"type": "yarn", "factor": 16.0, "original_max_position": 4096}])
def test_scaled_tables_and_far_positions(scaling):
    layer = tw.RotaryPositions(128, None, 131072, 500000.0, scaling=scaling).to(DEV)
    q, _, _, _ = inputs(9, 4, 1, 128, torch.float32)
    positions = torch.tensor([131071, 0, 1, 65536, 131070, 8191, 8192, 4097, 100000], device=DEV)
    qo = torch.empty_like(q, memory_format=torch.contiguous_format)
    layer(positions, q, None, qo)
    check(qo, q, positions, layer.cos_sin, False)


@pytest.mark.parametrize("interleaved", [False, True])
def test_inverse_is_the_gradient(interleaved):
    """The gradient of sum(y g) by x is the rotation of g the other way: against the formula, and against
    central differences of the 64-bit rotation (which is linear, so they are exact up to rounding)."""
    T, H, D, dim = 6, 3, 64, 48
    x, g, _, positions = inputs(T, H, H, D, torch.float32)
    layer = tw.RotaryPositions(D, dim, 5000, 10000.0, interleaved).to(DEV)
    got = torch.empty(T, H, D, device=DEV)
    layer(positions, g, None, got, inverse=True)
    check(got, g, positions, layer.cos_sin, interleaved, inverse=True)
    x64, g64 = x.double().cpu(), g.double().cpu()
    for at in ((0, 0, 0), (1, 2, 1), (2, 1, 23), (3, 0, 24), (4, 2, 47), (5, 1, 63)):
        step = torch.zeros_like(x64)
        step[at] = 1e-3
        up, down = (rotate(x64 + s * step, positions, layer.cos_sin, interleaved) for s in (1, -1))
        slope = float(((up - down) * g64).sum() / 2e-3)
        assert abs(float(got[at]) - slope) <= 1e-5     # 1e-16 / 1e-3 * values of some 10, and fp32's 1e-7 of some 10


def test_wide_narrow_and_strided_layouts_agree_bit_for_bit():
    """The vector form (16-byte accesses) and the scalar one (any alignment) compute the same."""
    T, H, D = 21, 5, 128
    layer = tw.RotaryPositions(D, D, 5000).to(DEV)
    q, _, _, positions = inputs(T, H, 1, D, torch.bfloat16)
    a = q.contiguous()
    odd = torch.empty(T * H * D + 1, dtype=torch.bfloat16, device=DEV)[1:].view(T, H, D).copy_(a)
    by_head = torch.empty(H, T, D, dtype=torch.bfloat16, device=DEV).transpose(0, 1).copy_(a)
    gaps = torch.empty(T, H, D + 3, dtype=torch.bfloat16, device=DEV)[..., :D].copy_(a)
    layer(positions, a)
    for other in (odd, by_head, gaps):
        layer(positions, other)
        assert torch.equal(a, other)


def test_position_outside_the_table_gives_nan_and_touches_nothing_else():
    layer = tw.RotaryPositions(64, 32, 100).to(DEV)
    q = torch.randn(4, 2, 64, device=DEV)
    q0 = q.clone()
    layer(torch.tensor([5, 100, -1, 99], device=DEV), q)
    assert q[1:3, :, :32].isnan().all() and not q[[0, 3]].isnan().any()
    assert torch.equal(q[:, :, 32:], q0[:, :, 32:])


def test_direct_and_ctypes_routes_agree(monkeypatch):
    if ops._fast is None:
        pytest.skip("no compiled binding")
    layer = tw.RotaryPositions(128).to(DEV)
    q, k, _, positions = inputs(10, 8, 2, 128, torch.float16)
    a, b = torch.empty_like(q), torch.empty_like(k)
    layer(positions, q, k, a, b)
    assert ops._fast.rotary_positions(q, k, positions, layer.cos_sin, False, False, a, b) is True
    monkeypatch.setattr(ops, "_fast", None)
    c, d = torch.empty_like(q), torch.empty_like(k)
    layer(positions, q, k, c, d)
    assert torch.equal(a, c) and torch.equal(b, d)


def test_no_tokens():
    layer = tw.RotaryPositions(128).to(DEV)
    q = torch.empty(0, 8, 128, device=DEV)
    assert layer(torch.empty(0, dtype=torch.int64, device=DEV), q)[0].shape == (0, 8, 128)


def test_refusals():
    layer = tw.RotaryPositions(64, 32, 100).to(DEV)
    q, pos = torch.randn(4, 2, 64, device=DEV), torch.arange(4, device=DEV)
    for bad, match in (((pos.int(), q), "positions"), ((pos[:3], q), "positions holds 3"), ((pos, q[..., 0]), "shape"),
                       ((pos, q, q.half()), "dtype"), ((pos, q, q[:3]), "k has shape"), ((pos, q.transpose(1, 2)), "channels"),
                       ((pos.cpu(), q), "positions"), ((pos, q, None, q[:, :1]), "q_out"),
                       ((pos, q, None, None, q), "k_out without k"), ((pos, torch.randn(4, 2, 16, device=DEV)), "cos_sin")):
        with pytest.raises(RuntimeError, match=match):
            layer(*bad)
    with pytest.raises(NotImplementedError):
        layer(pos, q.double())
    with pytest.raises(RuntimeError, match="GPU only|expected"):
        ops.rotary_positions(q.cpu(), None, pos, layer.cos_sin)
