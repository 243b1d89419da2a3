"""Argument checks of the gated product, the 8-bit codes and their product: nothing is launched, so no GPU is needed."""
import ctypes

import pytest
import torch

from tokenweave_amd import _lib, ops

BUF = ctypes.create_string_buffer(4096 + 256)
AT = (ctypes.addressof(BUF) + 255) & ~255   # host memory: never read by these calls
BAD, ALIGN, DTYPE = _lib.TW_ERR_INVALID_ARGUMENT, _lib.TW_ERR_ALIGNMENT, _lib.TW_ERR_DTYPE


def gated(out=AT, both=None, a=AT, b=AT, M=4, inner=8, K=16, ldc=8, ld_both=0, act=0):
    return _lib.lib().tw_gated_gemm_bf16_nt(out, both, a, b, M, inner, K, ldc, ld_both, act, 0, None)


def test_gated_product():
    assert gated(M=0, out=None, a=None, b=None) == _lib.TW_OK
    for call in (dict(out=None), dict(a=None), dict(b=None), dict(M=-1), dict(inner=0), dict(K=0), dict(ldc=4),
                 dict(act=3), dict(act=-1), dict(both=AT, ld_both=12), dict(both=AT, ld_both=18), dict(K=(1 << 24) + 8),
                 dict(inner=1 << 30, ldc=1 << 30)):
        assert gated(**call) == BAD, call
    for call in (dict(inner=6), dict(K=12), dict(ldc=10), dict(a=AT + 8), dict(b=AT + 8), dict(out=AT + 4),
                 dict(both=AT + 4, ld_both=16)):
        assert gated(**call) == ALIGN, call


def backward(ga=AT, gb=AT, grad=AT, ld_grad=8, a=AT, b=AT, both=AT, ld_both=16, M=4, inner=8, K=16, act=0, ws=AT, size=None):
    L = _lib.lib()
    if size is None:
        size = L.tw_gated_gemm_bf16_nt_backward_workspace(4, 8, 16, ga is not None, gb is not None)
    return L.tw_gated_gemm_bf16_nt_backward(ga, gb, grad, ld_grad, a, b, both, ld_both, M, inner, K, act, 0, ws, size, None)


def test_gated_gradients():
    L = _lib.lib()
    size = L.tw_gated_gemm_bf16_nt_backward_workspace
    # D, b turned; D turned and a turned over 64 rows: 2 bytes each, 256-byte places
    assert size(4, 8, 16, 1, 0) == 256 + 512
    assert size(4, 8, 16, 0, 1) == 2 * (16 * 64 + 16 * 64)
    assert size(4, 8, 16, 1, 1) == size(4, 8, 16, 1, 0) + size(4, 8, 16, 0, 1)
    assert size(0, 8, 16, 1, 1) == 0 and size(4, 8, 16, 0, 0) == 0
    assert size(4, 6, 16, 1, 1) == ALIGN and size(-1, 8, 16, 1, 1) == BAD
    assert backward(ga=None, gb=None) == _lib.TW_OK
    assert backward(M=0, gb=None) == _lib.TW_OK
    for call in (dict(grad=None), dict(a=None), dict(b=None), dict(both=None), dict(ws=None), dict(size=100),
                 dict(ld_grad=4), dict(ld_grad=10), dict(ld_both=8), dict(ld_both=18), dict(act=3), dict(K=0), dict(M=-1)):
        assert backward(**call) == BAD, call
    for call in (dict(inner=6), dict(K=12), dict(a=AT + 8), dict(b=AT + 8), dict(ws=AT + 64), dict(ga=AT + 4),
                 dict(gb=AT + 4), dict(grad=AT + 4), dict(both=AT + 4)):
        assert backward(**call) == ALIGN, call


def quant(out=AT, scales=AT, s0=1, s1=4, x=AT, ld=64, M=4, K=64, act=-1, dtype=0):
    return _lib.lib().tw_quant_fp8_groups(out, scales, s0, s1, x, ld, M, K, act, dtype, None)


def test_codes():
    assert quant(M=0, out=None, scales=None, x=None) == _lib.TW_OK
    for call in (dict(out=None), dict(scales=None), dict(x=None), dict(M=-1), dict(K=0), dict(ld=32), dict(act=0), dict(act=3)):
        assert quant(**call) == BAD, call
    assert quant(dtype=3) == DTYPE
    for call in (dict(x=AT + 1), dict(x=AT + 2, dtype=2), dict(scales=AT + 2)):
        assert quant(**call) == ALIGN, call


def block(out=AT, a=AT, sa=AT, b=AT, sb=AT, M=4, N=8, K=32, ldc=8, dtype=0):
    return _lib.lib().tw_gemm_fp8_block_nt(out, a, sa, 1, 4, b, sb, M, N, K, ldc, dtype, 0, None)


def test_block_product():
    assert block(M=0, out=None, a=None, sa=None, b=None, sb=None) == _lib.TW_OK
    for call in (dict(out=None), dict(a=None), dict(sa=None), dict(b=None), dict(sb=None), dict(M=-1), dict(N=0), dict(K=0),
                 dict(ldc=4), dict(K=(1 << 22) + 16)):
        assert block(**call) == BAD, call
    assert block(dtype=2) == DTYPE
    for call in (dict(N=6), dict(K=24), dict(ldc=10), dict(a=AT + 8), dict(b=AT + 8), dict(out=AT + 4), dict(sa=AT + 2),
                 dict(sb=AT + 2)):
        assert block(**call) == ALIGN, call


def bf16(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def test_the_ops_run_on_the_gpu_only():
    codes, scales = torch.zeros((4, 128), dtype=torch.float8_e4m3fn), torch.zeros((4, 1))
    for call in (lambda: ops.gated_gemm_bf16_nt(bf16(4, 8), bf16(4, 16), bf16(16, 16)),
                 lambda: ops.gated_gemm_bf16_nt_backward(bf16(4, 16), None, bf16(4, 8), bf16(4, 16), bf16(16, 16), bf16(4, 16)),
                 lambda: ops.quant_fp8_groups(codes, scales, bf16(4, 128)),
                 lambda: ops.gemm_fp8_block_nt(bf16(4, 4), codes, scales, codes, scales[:1])):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_names_and_types_are_checked():
    with pytest.raises(ValueError, match="unknown activation 'relu'"):
        ops.gated_gemm_bf16_nt(bf16(4, 8), bf16(4, 16), bf16(16, 16), "relu")
    with pytest.raises(ValueError, match="unknown activation"):
        ops.quant_fp8_groups(torch.zeros((4, 8), dtype=torch.float8_e4m3fn), torch.zeros((4, 1)), bf16(4, 16), "tanh")
    with pytest.raises(NotImplementedError):
        ops.gated_gemm_bf16_nt(bf16(4, 8), torch.zeros(4, 16), bf16(16, 16))
    with pytest.raises(NotImplementedError):
        ops.gemm_fp8_block_nt(bf16(4, 4), bf16(4, 128), torch.zeros(4, 1), bf16(4, 128), torch.zeros(1, 1))
    with pytest.raises(NotImplementedError):
        ops.quant_fp8_groups(torch.zeros((4, 8), dtype=torch.int8), torch.zeros((4, 1)), torch.zeros(4, 8, dtype=torch.int32))


def test_a_tensor_that_wants_its_gradient_is_refused():
    x = bf16(4, 16).requires_grad_()
    with pytest.raises(RuntimeError, match="records no gradient"):
        ops.gated_gemm_bf16_nt(bf16(4, 8), x, bf16(16, 16))
    with pytest.raises(RuntimeError, match="records no gradient"):
        ops.quant_fp8_groups(torch.zeros((4, 16), dtype=torch.float8_e4m3fn), torch.zeros((4, 1)), x)
