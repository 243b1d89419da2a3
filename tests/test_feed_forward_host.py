"""Argument checks of the gated product, the 8-bit codes and their product: nothing is launched, so no GPU is needed."""
import ctypes

import pytest
import torch

from tokenweave_amd import _lib, ops

BUF = ctypes.create_string_buffer(4096 + 256)
AT = (ctypes.addressof(BUF) + 255) & ~255   # host memory: never read by these calls
BAD, ALIGN, DTYPE = _lib.TW_ERR_INVALID_ARGUMENT, _lib.TW_ERR_ALIGNMENT, _lib.TW_ERR_DTYPE


def gated(out=AT, both=None, a=AT, b=AT, M=4, inner=8, K=16, ldc=8, ld_both=0, act=0, ws=None, size=0):
    return _lib.lib().tw_gated_gemm_bf16_nt(out, both, a, b, M, inner, K, ldc, ld_both, act, 0, ws, size, None)


def test_gated_product():
    assert gated(M=0, out=None, a=None, b=None) == _lib.TW_OK
    for call in (dict(out=None), dict(a=None), dict(b=None), dict(M=-1), dict(inner=0), dict(K=0), dict(ldc=4),
                 dict(act=3), dict(act=-1), dict(both=AT, ld_both=12), dict(both=AT, ld_both=18), dict(K=(1 << 24) + 8),
                 dict(inner=1 << 30, ldc=1 << 30)):
        assert gated(**call) == BAD, call
    for call in (dict(inner=6), dict(K=12), dict(ldc=10), dict(a=AT + 8), dict(b=AT + 8), dict(out=AT + 4),
                 dict(both=AT + 4, ld_both=16)):
        assert gated(**call) == ALIGN, call


def test_gated_product_divided_along_k():
    size = _lib.lib().tw_gated_gemm_bf16_nt_workspace
    # few rows, many, few slabs, many columns: nothing to add; else the fp32 sums of both products, of some parts
    for M, inner, K in ((0, 8, 8192), (1, 748, 6904), (32, 748, 6904), (1025, 748, 6904), (300, 704, 440), (4096, 3584, 8192)):
        assert size(M, inner, K) == 0, (M, inner, K)
    for M, inner, K in ((96, 748, 6904), (160, 3584, 8192), (160, 748, 6904), (1000, 36, 2048)):
        assert size(M, inner, K) >= 2 * 8 * M * inner and size(M, inner, K) % (8 * M * inner) == 0, (M, inner, K)
    assert size(4, 6, 16) == ALIGN and size(-1, 8, 16) == BAD and size(4, 8, 0) == BAD
    shape = dict(M=160, inner=748, K=6904, ldc=748)
    need = size(160, 748, 6904)
    assert gated(**shape) == BAD and gated(**shape, ws=AT, size=need - 1) == BAD
    assert gated(**shape, ws=AT + 64, size=need) == ALIGN


def backward(ga=AT, gb=AT, grad=AT, ld_grad=8, a=AT, b=AT, both=AT, ld_both=16, M=4, inner=8, K=16, act=0, ws=AT, size=None):
    L = _lib.lib()
    if size is None:
        size = L.tw_gated_gemm_bf16_nt_backward_workspace(4, 8, 16, ga is not None, gb is not None)
    return L.tw_gated_gemm_bf16_nt_backward(ga, gb, grad, ld_grad, a, b, both, ld_both, M, inner, K, act, 0, ws, size, None)


def test_gated_gradients():
    L = _lib.lib()
    size = L.tw_gated_gemm_bf16_nt_backward_workspace
    # the gradient of both products, 2 bytes a value, and the same turned; rows of whole slabs of 64
    assert size(4, 8, 16, 1, 0) == 4 * 64 * 2 and size(4, 8, 16, 0, 1) == 16 * 64 * 2
    assert size(65, 40, 16, 1, 1) == (65 * 128 + 80 * 128) * 2
    assert size(0, 8, 16, 1, 1) == 0 and size(4, 8, 16, 0, 0) == 0
    assert size(4, 6, 16, 1, 1) == ALIGN and size(-1, 8, 16, 1, 1) == BAD
    assert backward(ga=None, gb=None) == _lib.TW_OK
    assert backward(M=0, gb=None) == _lib.TW_OK
    for call in (dict(grad=None), dict(a=None), dict(b=None), dict(both=None), dict(ws=None), dict(size=2559),
                 dict(K=(1 << 21) + 8), dict(inner=1 << 21, ld_grad=1 << 21, ld_both=1 << 22, gb=None, size=1 << 60),
                 dict(M=(1 << 21) + 1, ga=None, size=1 << 60),
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


def block(out=AT, a=AT, sa=AT, b=AT, sb=AT, M=4, N=8, K=32, ldc=8, dtype=0, ws=None, size=0):
    return _lib.lib().tw_gemm_fp8_block_nt(out, a, sa, 1, 4, b, sb, M, N, K, ldc, dtype, 0, ws, size, None)


def test_block_product():
    assert block(M=0, out=None, a=None, sa=None, b=None, sb=None) == _lib.TW_OK
    for call in (dict(out=None), dict(a=None), dict(sa=None), dict(b=None), dict(sb=None), dict(M=-1), dict(N=0), dict(K=0),
                 dict(ldc=4), dict(K=(1 << 22) + 16)):
        assert block(**call) == BAD, call
    assert block(dtype=2) == DTYPE
    for call in (dict(N=6), dict(K=24), dict(ldc=10), dict(a=AT + 8), dict(b=AT + 8), dict(out=AT + 4), dict(sa=AT + 2),
                 dict(sb=AT + 2)):
        assert block(**call) == ALIGN, call


def test_block_product_divided_along_k():
    size = _lib.lib().tw_gemm_fp8_block_nt_workspace
    for M, N, K in ((0, 1024, 8192), (1, 1024, 8192), (64, 1024, 8192), (1025, 1024, 8192), (300, 1024, 384), (1000, 8192, 3696),
                    (96, 7168, 8192)):
        assert size(M, N, K) == 0, (M, N, K)
    for M, N, K in ((96, 1024, 8192), (200, 1024, 8192), (1000, 1024, 8192), (300, 100, 4112)):
        assert size(M, N, K) >= 2 * 4 * M * N and size(M, N, K) % (4 * M * N) == 0, (M, N, K)
    assert size(-1, 8, 16) == BAD and size(4, 0, 16) == BAD and size(4, 8, (1 << 22) + 16) == BAD
    shape = dict(M=200, N=1024, K=8192, ldc=1024)
    need = size(200, 1024, 8192)
    assert block(**shape) == BAD and block(**shape, ws=AT, size=need - 1) == BAD
    assert block(**shape, ws=AT + 64, size=need) == ALIGN


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


def test_the_formulas_gradients_follow_differences():
    """The 64-bit gradients that the kernel's are compared with, against central differences."""
    import feed_forward_reference as R
    g = torch.Generator().manual_seed(3)
    x, w, c = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((3, 8), (12, 8), (3, 6)))
    for kind in R.ACTIVATIONS:
        both = x @ w.t()
        gx, _, gw, _ = R.gated_gradients(c, x, w, both, kind)

        def loss(x, w):
            gate, up = (x @ w.t()).chunk(2, 1)
            return float((R.act(gate, kind) * up * c).sum())

        for t, grad in ((x, gx), (w, gw)):
            for i in range(0, t.numel(), 5):
                keep, h = t.view(-1)[i].item(), 1e-5
                t.view(-1)[i] = keep + h
                above = loss(x, w)
                t.view(-1)[i] = keep - h
                below = loss(x, w)
                t.view(-1)[i] = keep
                # a third derivative of order 100 times h^2, and 2^-50 of the loss over h
                assert abs((above - below) / (2 * h) - grad.view(-1)[i].item()) < 1e-7


def test_layers_check_their_sizes():
    import tokenweave_amd as tw
    with pytest.raises(ValueError, match="not divisible"):
        tw.GatedLinear(16, 30, tp_size=4)
    with pytest.raises(ValueError, match="Invalid rank"):
        tw.GatedLinear(16, 32, tp_rank=4, tp_size=4)
    with pytest.raises(ValueError, match="unknown activation"):
        tw.FeedForward(16, 32, "swish")


def test_sizes_without_8_bit_rows_are_refused_when_a_model_is_loaded():
    import tokenweave_amd as tw
    with pytest.raises(ValueError, match="multiple of 16"):
        tw.FeedForward(64, 400, tp_size=2).to_fp8_blocks()
    with pytest.raises(ValueError, match="multiple of 16"):
        tw.Fp8BlockLinearMethod().process_weights(tw.RowParallelLinear(24, 64, bias=False))


def test_weight_codes_on_the_cpu():
    import feed_forward_reference as R
    import tokenweave_amd as tw
    w = torch.randn(300, 200)
    codes, scales = tw.quantize_fp8_blocks(w)
    want, want_scales = R.weight_codes(w)
    assert codes.dtype == torch.float8_e4m3fn and scales.shape == (3, 2)
    assert torch.allclose(scales, want_scales, rtol=2 ** -23, atol=0) and (codes.float() - want.float()).abs().max() <= 32


def test_a_capture_is_refused_where_a_gradient_is_recorded(monkeypatch):
    from tokenweave_amd import feed_forward
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="gated_gemm_bf16_nt_backward"):
        feed_forward.gated_linear(bf16(4, 16).requires_grad_(), bf16(16, 16))


def test_a_models_type_leaves_codes_and_scales_as_they_are():
    import tokenweave_amd as tw
    block = tw.FeedForward(64, 96)
    for p in block.parameters():
        p.data.normal_()
    block.to_fp8_blocks()
    before = {k: v.clone() for k, v in block.state_dict().items()}
    for model in (block.half(), block.bfloat16(), block.to(torch.float32)):
        for name, value in model.state_dict().items():
            assert value.dtype == before[name].dtype == (torch.float32 if "scale" in name else torch.float8_e4m3fn)
            assert torch.equal(value.view(torch.uint8), before[name].view(torch.uint8))
    plain = tw.RowParallelLinear(64, 64, bias=True).half()
    assert plain.weight.dtype == plain.bias.dtype == torch.float16
