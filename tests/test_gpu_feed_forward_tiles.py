"""Every tile shape of the feed-forward half's products, against 64 bits: each alone in one round, each walking several
tiles under a grid cap, inner dimensions of whole and of partial slabs, short ones and ones of more than 64 slabs, each
divided form.  The sizes are the smallest found at which the rules choose the shape on 256 compute units."""
import pytest
import torch

import feed_forward_reference as R
from tokenweave_amd import ops

pytestmark = pytest.mark.gpu
DEV, BF16, FP8 = "cuda", torch.bfloat16, torch.float8_e4m3fn


def normal(shape, seed, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * std).to(BF16)


def guarded(rows, width):
    buf = torch.full((rows + 2, width), 777.0, dtype=BF16, device=DEV)
    return buf[1:1 + rows], buf


def check_gated(M, inner, K, cap, kind):
    x, w = normal((M, K), M), normal((2 * inner, K), inner, K ** -0.5)
    (out, out_buf), (both, both_buf) = guarded(M, inner), guarded(M, 2 * inner)
    ops.gated_gemm_bf16_nt(out, x, w, kind, cap, gate_up=both)
    want, bound, products, off = R.gated(x, w, kind)
    R.assert_within(out, want, bound, "out")
    R.assert_within(both, products, off, "gate_up")
    for buf in (out_buf, both_buf):
        assert (buf[0] == 777.0).all() and (buf[-1] == 777.0).all()


# tile rows x columns of b, M, I, cap
GATED = [("256x256", 1731, 3348, None), ("192x256", 1130, 4104, None), ("160x256", 1028, 3588, None),
         ("128x256", 4041, 644, None), ("96x256", 387, 4228, None), ("128x128", 295, 4144, None), ("96x128", 194, 4104, None),
         ("64x128", 234, 36, None),
         ("256x256", 641, 68, 1), ("192x256", 536, 80, 1), ("160x256", 134, 264, 1), ("128x256", 193, 280, 2),
         ("96x256", 167, 264, 2), ("128x128", 449, 32, 1), ("96x128", 261, 32, 1)]


@pytest.mark.parametrize("shape,M,inner,cap", GATED)
@pytest.mark.parametrize("K", [192, 200])
def test_gated_tiles(shape, M, inner, cap, K):
    check_gated(M, inner, K, cap, R.ACTIVATIONS[M % 3])


@pytest.mark.parametrize("shape,M,inner,cap", [("256x256", 1731, 3348, None), ("192x256", 1130, 4104, None),
                                               ("160x256", 1028, 3588, None), ("128x256", 4041, 644, None)])
@pytest.mark.parametrize("K", [4224, 4232])
def test_gated_tiles_of_many_slabs(shape, M, inner, cap, K):
    check_gated(M, inner, K, cap, "silu")


@pytest.mark.parametrize("M,inner,K", [(132, 4, 1256), (133, 4, 1728), (791, 4, 6120), (783, 4, 6400), (780, 4, 7648), (739, 4, 8448),
                                       (142, 2784, 3728), (155, 2712, 6400)])
@pytest.mark.parametrize("cap", [None, 5])
def test_gated_tiles_divided_along_k(M, inner, K, cap):
    from tokenweave_amd import _lib
    assert _lib.lib().tw_gated_gemm_bf16_nt_workspace(M, inner, K) > 0
    check_gated(M, inner, K, cap, R.ACTIVATIONS[M % 3])


def check_gradients(M, inner, K, cap, wanted):
    x, w = normal((M, K), M), normal((2 * inner, K), inner, K ** -0.5)
    both = normal((M, 2 * inner), 3)
    grad = normal((M, inner), 4)
    (gx, gx_buf), (gw, gw_buf) = guarded(M, K), guarded(2 * inner, K)
    ops.gated_gemm_bf16_nt_backward(gx if "a" in wanted else None, gw if "b" in wanted else None, grad, x, w, both, "silu", cap)
    want_x, bound_x, want_w, bound_w = R.gated_gradients(grad, x, w, both, "silu")
    if "a" in wanted:
        R.assert_within(gx, want_x, bound_x, "grad_x")
    if "b" in wanted:
        R.assert_within(gw, want_w, bound_w, "grad_w")
    for buf in (gx_buf, gw_buf):
        assert (buf[0] == 777.0).all() and (buf[-1] == 777.0).all()


# tile, rows and columns of the product, cap
PRODUCT = [("256x256", 3075, 3848, None), ("192x256", 3089, 3664, None), ("256x192", 4012, 2312, None),
           ("160x256", 3665, 2312, None), ("192x192", 4103, 1808, None), ("128x256", 4103, 1352, None),
           ("96x256", 3215, 1744, None), ("128x192", 4104, 968, None), ("96x192", 780, 4616, None), ("128x128", 4036, 648, None),
           ("96x128", 4131, 400, None), ("64x128", 2, 192, None),
           ("256x256", 194, 624, 1), ("192x256", 184, 584, 1), ("256x192", 690, 136, 1), ("160x256", 143, 616, 1),
           ("192x192", 519, 136, 1), ("128x256", 101, 616, 1), ("96x256", 1, 1000, 1), ("128x192", 97, 560, 1),
           ("96x192", 2, 576, 1), ("128x128", 323, 72, 1), ("96x128", 285, 64, 1), ("64x128", 1, 360, 1)]


@pytest.mark.parametrize("shape,M,N,cap", PRODUCT)
@pytest.mark.parametrize("inner", [32, 36, 220])
def test_gradient_of_the_rows(shape, M, N, cap, inner):
    check_gradients(M, inner, N, cap, "a")


@pytest.mark.parametrize("shape,rows,N,cap", PRODUCT)
@pytest.mark.parametrize("M", [64, 75])
def test_gradient_of_the_weight(shape, rows, N, cap, M):
    """(The nearest count of rows that a weight of gate and up halves of whole fours has.)"""
    check_gradients(M, max(4, rows // 8 * 4), N, cap, "b")


@pytest.mark.parametrize("shape,M,inner,K,cap", [
    ("64x128", 1, 8, 16, None), ("96x128", 138, 40, 7064, None), ("96x192", 162, 96, 8232, None), ("96x256", 419, 132, 7584, None),
    ("128x128", 211, 68, 7560, None), ("128x192", 209, 156, 7120, None), ("128x256", 389, 152, 7688, None),
    ("160x256", 597, 224, 7752, None), ("192x192", 534, 204, 7208, None), ("192x256", 527, 400, 7432, None),
    ("256x192", 556, 348, 7904, None), ("256x256", 899, 356, 7952, None),
    ("64x128", 1, 8, 2080, 16), ("96x128", 923, 520, 16, 16), ("96x192", 81, 44, 2360, 16), ("96x256", 1, 20, 3128, 16),
    ("128x128", 1705, 896, 16, 16), ("128x192", 110, 40, 2240, 16), ("128x256", 116, 44, 3144, 16), ("160x256", 263, 76, 2392, 16),
    ("192x192", 164, 72, 2352, 16), ("192x256", 317, 188, 1568, 16), ("256x192", 218, 76, 2592, 16),
    ("256x256", 422, 196, 1904, 16)])
def test_both_gradients_in_one_launch(shape, M, inner, K, cap):
    check_gradients(M, inner, K, cap, "ab")


def check_block(M, N, K, cap, dtype=BF16):
    g = torch.Generator(device=DEV).manual_seed(M)
    a, a_scales = torch.empty((M, K), dtype=FP8, device=DEV), ops.fp8_group_scales(M, K)
    ops.quant_fp8_groups(a, a_scales, torch.randn((M, K), generator=g, device=DEV)
                         * torch.exp2(torch.randint(-3, 4, (M, 1), generator=g, device=DEV).float()))
    b = torch.randn((N, K), generator=g, device=DEV)
    blocks = torch.exp2(torch.randint(-3, 4, (-(-N // 128), -(-K // 128)), generator=g, device=DEV).float())
    b, b_scales = R.weight_codes(b * blocks.repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K])
    buf = torch.full((M + 2, N), 777.0, dtype=dtype, device=DEV)
    ops.gemm_fp8_block_nt(buf[1:-1], a, a_scales, b, b_scales, cap)
    want, off = R.block_product(a, a_scales, b, b_scales)
    R.assert_within(buf[1:-1], want, off + R.half(dtype) * want.abs(), "out")
    assert (buf[0] == 777.0).all() and (buf[-1] == 777.0).all()


# tile, M, N, cap
BLOCK = [("256x224", 3080, 3852, None), ("256x192", 3652, 3104, None), ("192x256", 2309, 3332, None), ("256x128", 3614, 2060, None),
         ("256x128", 4352, 1920, None), ("128x256", 4101, 908, None), ("128x128", 4175, 388, None), ("64x128", 1062, 64, None),
         ("256x224", 1181, 196, 1), ("256x192", 1074, 132, 1), ("192x256", 1115, 132, 2), ("256x128", 1041, 32, 1),
         ("128x256", 1227, 204, 2), ("128x128", 1040, 32, 3), ("64x128", 1308, 32, 5)]


@pytest.mark.parametrize("shape,M,N,cap", BLOCK)
@pytest.mark.parametrize("K", [128, 640, 656, 8320, 8336])
def test_block_scaled_tiles(shape, M, N, cap, K):
    check_block(M, N, K, cap)


@pytest.mark.parametrize("shape,M,N,K", [("64x128", 65, 4, 3808), ("64x128", 71, 4, 4224), ("128x128", 325, 4, 16368),
                                         ("128x128", 260, 4, 20992), ("128x256", 130, 3920, 9776), ("128x256", 395, 1640, 12160),
                                         ("128x256", 920, 1388, 21968), ("128x256", 920, 1388, 22016)])
@pytest.mark.parametrize("cap", [None, 3])
def test_block_scaled_tiles_divided_along_k(shape, M, N, K, cap):
    from tokenweave_amd import _lib
    assert _lib.lib().tw_gemm_fp8_block_nt_workspace(M, N, K) > 0
    check_block(M, N, K, cap)
