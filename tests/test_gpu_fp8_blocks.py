"""Rows to e4m3 codes by groups of 128 and the block-scaled product, against 64 bits: codes to the bit where the rows are
given, every row count at which another kernel or tile serves, ragged groups and blocks, views, captured calls."""
import pytest
import torch

import feed_forward_reference as R
from tokenweave_amd import ops

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn
DTYPES = (torch.bfloat16, torch.float16, torch.float32)


def rows(M, K, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((M, K), generator=g, device="cuda")
    return (x * torch.exp2(torch.randint(-12, 6, (M, K), generator=g, device="cuda").float())).to(dtype)


def quantised(x, kind=None, scales=None):
    K = x.shape[1] // (1 if kind is None else 2)
    out = torch.empty((x.shape[0], K), dtype=FP8, device="cuda")
    scales = ops.fp8_group_scales(x.shape[0], K) if scales is None else scales
    ops.quant_fp8_groups(out, scales, x, kind)
    return out, scales


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (1, 8), (3, 127), (17, 128), (16, 129), (33, 3696), (5, 8192), (1001, 264)])
def test_codes_to_the_bit(M, K, dtype):
    x = rows(M, K, dtype)
    got, scales = quantised(x)
    want, want_scales = R.codes(x.double())
    assert torch.equal(scales, want_scales)
    assert torch.equal(got.double(), want)
    plain = torch.full((M, -(-K // 128)), 3.0, device="cuda")   # scales in the rows' order
    again, _ = quantised(x, scales=plain)
    assert torch.equal(plain, scales) and torch.equal(again.view(torch.uint8), got.view(torch.uint8))


@pytest.mark.parametrize("dtype", DTYPES)
def test_quotients_on_borders(dtype):
    """Every border of two codes, one step of the type beside it, as multiples of the scale where the scale is a power
    of two and where it is not."""
    values = torch.arange(127, dtype=torch.uint8).view(FP8).double()
    borders = (values[1:] + values[:-1]) / 2
    for scale in (1.0, 0.75, 5.0 / 7, 1.1e-3):
        y = torch.cat((borders * scale, -borders * scale)).to(dtype)
        y = torch.cat((y, torch.nextafter(y.float(), torch.tensor(9e9)).to(dtype), y * (1 + torch.finfo(dtype).eps)))
        y = torch.nn.functional.pad(y, (0, -len(y) % 127)).view(-1, 127)
        top = torch.full((len(y), 1), 448 * scale).to(dtype)
        x = torch.cat((y, top), 1).cuda()
        got, scales = quantised(x)
        want, want_scales = R.codes(x.double())
        assert torch.equal(scales, want_scales) and torch.equal(got.double(), want), scale


def test_every_bf16_value_with_every_small_scale():
    """All finite bf16 magnitudes below a group's largest, for many largest values: 64-bit codes."""
    g = torch.Generator().manual_seed(4)
    for e in (-30, -8, 0, 9, 60):
        top = (1 + torch.rand(512, 1, generator=g)) * 2.0 ** e
        y = top * torch.rand(512, 127, generator=g) ** 3
        x = torch.cat((y, top), 1).bfloat16().cuda()
        x[:, :127] = torch.minimum(x[:, :127], x[:, 127:])
        got, scales = quantised(x)
        want, want_scales = R.codes(x.double())
        assert torch.equal(scales, want_scales) and torch.equal(got.double(), want), e


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", R.ACTIVATIONS)
@pytest.mark.parametrize("M,K", [(1, 4), (19, 136), (130, 3696), (64, 77)])
def test_gated_rows(M, K, kind, dtype):
    g = torch.Generator(device="cuda").manual_seed(M)
    x = (torch.randn((M, 2 * K), generator=g, device="cuda") * 3).to(dtype)
    got, scales = quantised(x, kind)
    y = R.act(x[:, :K].double(), kind) * x[:, K:].double()
    _, want = R.codes(y)
    R.assert_within(scales, want.double(), want.double() * 2 * R.ACT, "scales")
    s = R.spread(scales, K, 1).double()
    # half a step of the code, and what the activation was off before
    R.assert_within(got.double() * s, y, y.abs() * (R.half(FP8) + 2 * R.ACT) + s * 2 ** -10, "values")


def test_zeros_tiny_huge_and_no_numbers():
    x = torch.zeros((6, 256), dtype=torch.float32, device="cuda")
    x[1] = 1e-30
    x[2] = 3e38
    x[3, 7] = float("inf")
    x[4, 130] = float("nan")
    x[5, 0] = -1e-42
    got, scales = quantised(x)
    least = (torch.tensor(1e-10) .double() / 448).float().cuda()
    assert (scales[0] == least).all() and (got[0].float() == 0).all()
    assert (scales[1] == least).all() and (got[1].float() == 0).all()
    assert (got[2].float() == 448).all()
    assert torch.isnan(got[3, :128].float()).all() and (got[3, 128:].float() == 0).all()
    assert torch.isnan(got[4, 128:].float()).all() and (got[4, :128].float() == 0).all()
    assert not torch.isfinite(scales[3, 0]) and not torch.isfinite(scales[4, 1])
    assert (got[5].float() == 0).all()


def test_views_and_alignment():
    """Row slices, rows that begin at any element, scales inside a wider buffer."""
    base = rows(40, 700, torch.bfloat16)
    for first, K in ((0, 256), (8, 264), (1, 255), (3, 130)):
        x = base[3:30, first:first + K]
        buf = torch.full((-(-K // 128) + 1, 60), -1.0, device="cuda")
        scales = buf[:-1, 10:37].t()
        got, _ = quantised(x, scales=scales)
        want, want_scales = R.codes(x.double())
        assert torch.equal(scales, want_scales) and torch.equal(got.double(), want)
        keep = buf.clone()
        keep[:-1, 10:37] = -1.0
        assert (keep == -1.0).all()


def operands(M, N, K, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    a, a_scales = quantised((torch.randn((M, K), generator=g, device="cuda")
                             * torch.exp2(torch.randint(-3, 4, (M, 1), generator=g, device="cuda").float())))
    w = torch.randn((N, K), generator=g, device="cuda") * K ** -0.5
    w = w * torch.exp2(torch.randint(-3, 4, (-(-N // 128), -(-K // 128)), generator=g, device="cuda").float()
                       ).repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
    return (a, a_scales) + R.weight_codes(w)


def check_product(M, N, K, dtype=torch.bfloat16, max_cus=None, seed=0):
    a, a_scales, b, b_scales = operands(M, N, K, seed)
    buf = torch.full((M + 2, N + 12), 777.0, dtype=dtype, device="cuda")
    out = buf[1:1 + M, 4:4 + N]
    ops.gemm_fp8_block_nt(out, a, a_scales, b, b_scales, max_cus)
    want, off = R.block_product(a, a_scales, b, b_scales)
    R.assert_within(out, want, off + R.half(dtype) * want.abs() + (6e-8 if dtype == torch.float16 else 0), "out")
    keep = buf.clone()
    keep[1:1 + M, 4:4 + N] = 777.0
    assert (keep == 777.0).all()
    again = torch.empty((M, N), dtype=dtype, device="cuda")
    ops.gemm_fp8_block_nt(again, a, a_scales.contiguous(), b, b_scales, max_cus)
    assert torch.equal(again, out)


@pytest.mark.parametrize("M", [1, 2, 8, 9, 16, 17, 32, 33, 64, 65, 100, 128])
@pytest.mark.parametrize("N,K", [(4, 16), (100, 128), (132, 144), (520, 1040), (1408, 1024), (8192, 256)])
def test_product_of_few_rows(M, N, K):
    check_product(M, N, K, (torch.bfloat16, torch.float16)[M % 2], seed=M)


@pytest.mark.parametrize("M", [129, 160, 255, 256, 257, 513, 1000])
@pytest.mark.parametrize("N,K", [(4, 16), (100, 128), (132, 144), (520, 1040), (1408, 1024), (8192, 256)])
def test_product_of_many_rows(M, N, K):
    check_product(M, N, K, (torch.bfloat16, torch.float16)[M % 2], seed=M)


@pytest.mark.parametrize("M,N,K", [(2458, 1376, 512), (4096, 2048, 128), (700, 7392, 400), (384, 6144, 2048),
                                   # one round of each shape: 256 x 224, 256 x 192, 192 x 256, 256 x 128, 128 x 256, ...
                                   (4096, 3584, 400), (4090, 3068, 528), (3070, 4092, 1040), (4096, 2044, 9200),
                                   (2047, 4096, 640), (2040, 2048, 144), (1020, 2048, 8336)])
def test_product_of_all_tile_shapes(M, N, K):
    check_product(M, N, K)


@pytest.mark.parametrize("M", [4, 200])
def test_what_the_instruction_keeps(M):
    """Beside 2^16 - 2^16: a product of the same aligned eight counts down to 2^3, one of another eight of the same
    16 down to 2^-8, any other one always.  (On this rest the bounds of this file's products, not the kernel.)"""
    for place, least in ((2, 3), (7, 3), (15, -8), (16, -18), (100, -18)):
        for e in (8, 4, 3, 0, -8, -12, -18):
            a, b = (torch.zeros((n, 128), device="cuda") for n in (M, 4))
            low = max(e // 2, -9)
            a[:, 0], a[:, 1], b[:, :2], a[:, place], b[:, place] = 256, -256, 256, 2.0 ** low, 2.0 ** (e - low)
            out = torch.empty((M, 4), dtype=torch.bfloat16, device="cuda")
            one = torch.ones((M, 1), device="cuda")
            ops.gemm_fp8_block_nt(out, a.to(FP8), one, b.to(FP8), one[:1])
            if e >= least:
                assert (out == 2.0 ** e).all(), (place, e)
            else:
                assert (out.abs() <= 2.0 ** least).all(), (place, e)


@pytest.mark.parametrize("M", [3, 64, 100, 300])
def test_long_inner_dimension(M):
    check_product(M, 68, 33168)


@pytest.mark.parametrize("M", [3, 130])
def test_weight_of_more_than_two_gib(M):
    N, K = 70000, 32768
    a, a_scales, _, _ = operands(M, 4, K)
    b = torch.empty((N, K), dtype=torch.uint8, device="cuda")
    for part in b.split(10000):
        part.copy_(torch.randint(0, 256, part.shape, dtype=torch.uint8, device="cuda"))
        part[(part & 0x7f) == 0x7f] = 1
    b_scales = torch.rand((-(-N // 128), K // 128), device="cuda")
    out = torch.empty((M, N), dtype=torch.bfloat16, device="cuda")
    ops.gemm_fp8_block_nt(out, a, a_scales, b.view(FP8), b_scales)
    for first in (0, 35072, 69888):
        part = b[first:first + 128].view(FP8)
        want, off = R.block_product(a, a_scales, part, b_scales[first // 128:first // 128 + 1])
        R.assert_within(out[:, first:first + 128], want, off + R.half(torch.bfloat16) * want.abs(), first)


def test_scales_of_one_row_at_any_stride():
    a, a_scales, b, b_scales = operands(1, 260, 272)
    wide = torch.empty((1, 1 << 22), device="cuda").as_strided((1, 3), (1 << 22, 5))
    wide.copy_(a_scales)
    out, want = (torch.empty((1, 260), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    ops.gemm_fp8_block_nt(want, a, a_scales, b, b_scales)
    ops.gemm_fp8_block_nt(out, a, wide, b, b_scales)
    assert torch.equal(out, want)
    with pytest.raises(RuntimeError, match="elements apart"):
        rows2 = torch.empty(1 << 22, device="cuda").as_strided((2, 3), (1 << 21, 1))
        ops.gemm_fp8_block_nt(torch.empty((2, 260), dtype=torch.bfloat16, device="cuda"), a.expand(2, -1).contiguous(), rows2,
                              b, b_scales)


@pytest.mark.parametrize("M", [5, 64, 300])
def test_grid_caps_give_the_same_bits(M):
    a, a_scales, b, b_scales = operands(M, 700, 528)
    outs = []
    for cap in (None, 1, 3, 64):
        out = torch.empty((M, 700), dtype=torch.bfloat16, device="cuda")
        ops.gemm_fp8_block_nt(out, a, a_scales, b, b_scales, cap)
        outs.append(out)
    assert all(torch.equal(o, outs[0]) for o in outs)


@pytest.mark.parametrize("M", [3, 200])
def test_codes_that_are_no_numbers_stay_in_their_row(M):
    a, a_scales, b, b_scales = operands(M, 260, 272)
    nan = torch.tensor([0x7f], dtype=torch.uint8, device="cuda").view(FP8)
    a[1, 270] = nan
    b[17, 5] = nan
    out = torch.empty((M, 260), dtype=torch.bfloat16, device="cuda")
    ops.gemm_fp8_block_nt(out, a, a_scales, b, b_scales)
    bad = torch.isnan(out)
    want = torch.zeros_like(bad)
    want[1], want[:, 17] = True, True
    assert torch.equal(bad, want)


def test_no_rows():
    a, a_scales, b, b_scales = operands(1, 260, 272)
    x = torch.empty((0, 260), dtype=torch.bfloat16, device="cuda")
    out, scales = quantised(x)
    assert out.shape == (0, 260) and scales.shape == (0, 3)
    ops.gemm_fp8_block_nt(torch.empty((0, 260), dtype=torch.bfloat16, device="cuda"), a[:0], a_scales[:0], b, b_scales)


@pytest.mark.parametrize("M", [7, 100, 300])
def test_a_run_captured(M):
    """Rows to codes, gate and up projections, activation and codes, down projection: captured and replayed."""
    H, inner = 272, 400
    g = torch.Generator(device="cuda").manual_seed(1)
    w1, s1 = R.weight_codes(torch.randn((2 * inner, H), generator=g, device="cuda") * H ** -0.5)
    w2, s2 = R.weight_codes(torch.randn((H, inner), generator=g, device="cuda") * inner ** -0.5)
    x = rows(M, H, torch.bfloat16)
    c1, t1 = torch.empty((M, H), dtype=FP8, device="cuda"), ops.fp8_group_scales(M, H)
    c2, t2 = torch.empty((M, inner), dtype=FP8, device="cuda"), ops.fp8_group_scales(M, inner)
    mid, out = (torch.empty((M, n), dtype=torch.bfloat16, device="cuda") for n in (2 * inner, H))

    def step():
        ops.quant_fp8_groups(c1, t1, x)
        ops.gemm_fp8_block_nt(mid, c1, t1, w1, s1)
        ops.quant_fp8_groups(c2, t2, mid, "silu")
        ops.gemm_fp8_block_nt(out, c2, t2, w2, s2)

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
        x.copy_(rows(M, H, torch.bfloat16, seed + 9))
        step()
        torch.cuda.synchronize()
        want = [t.clone() for t in (t1, mid, t2, out)]
        for t in (t1, mid, t2, out):
            t.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(t, o) for t, o in zip((t1, mid, t2, out), want)), seed


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K", [(129, 136, 144), (300, 8, 128), (1000, 1376, 272), (700, 7392, 400), (4096, 2048, 128),
                                   (2458, 1440, 512), (2500, 7168, 128)])
def test_outputs_that_begin_anywhere(M, N, K, dtype):
    """Rows 8, 16 and 64 bytes into a buffer, as far apart as keeps that alignment: the same bits, and nothing beside them."""
    x, sx, w, sw = operands(M, N, K)
    plain = torch.empty((M, N), dtype=dtype, device="cuda")
    ops.gemm_fp8_block_nt(plain, x, sx, w, sw)
    want, off = R.block_product(x, sx, w, sw)
    R.assert_within(plain, want, off + R.half(dtype) * want.abs() + (6e-8 if dtype == torch.float16 else 0), "plain")
    for step in (4, 8, 32):
        buf = torch.full((M + 2, (N + step - 1) // step * step + 2 * step), 777.0, dtype=dtype, device="cuda")
        out = buf[1:1 + M, step:step + N]
        ops.gemm_fp8_block_nt(out, x, sx, w, sw)
        assert torch.equal(out, plain), step
        out.fill_(777.0)
        assert (buf == 777.0).all(), step


@pytest.mark.parametrize("M", [130, 300])
def test_rows_of_the_output_far_apart(M):
    """Strides on both sides of what a 32-bit offset of a tile's rows reaches."""
    x, sx, w, sw = operands(M, 40, 272)
    plain = torch.empty((M, 40), dtype=torch.bfloat16, device="cuda")
    ops.gemm_fp8_block_nt(plain, x, sx, w, sw)
    for stride in (1 << 22, (1 << 22) + 64):
        buf = torch.empty(M * stride, dtype=torch.bfloat16, device="cuda")
        out = buf.as_strided((M, 48), (stride, 1))
        out.fill_(777.0)
        ops.gemm_fp8_block_nt(out[:, :40], x, sx, w, sw)
        assert torch.equal(out[:, :40], plain) and (out[:, 40:] == 777.0).all(), stride


@pytest.mark.parametrize("M,N,K", [(65, 4, 8208), (96, 1024, 8192), (128, 1280, 8192), (129, 100, 4112), (200, 1024, 8192),
                                   (257, 132, 6160), (300, 1024, 4096), (512, 768, 3600), (640, 700, 6144), (1000, 1024, 8192),
                                   (1024, 520, 20000)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_divided_along_k(M, N, K, dtype):
    """Few columns and a long inner dimension: against 64 bits, under grid caps, from any workspace."""
    from tokenweave_amd import _lib
    L = _lib.lib()
    size = L.tw_gemm_fp8_block_nt_workspace(M, N, K)
    assert size > 0, "this size is not divided any more: the test needs another"
    check_product(M, N, K, dtype, seed=M)
    x, sx, w, sw = operands(M, N, K, M)
    out = torch.empty((M, N), dtype=dtype, device="cuda")
    ops.gemm_fp8_block_nt(out, x, sx, w, sw)
    for max_cus in (1, 24, 100):
        again = torch.full_like(out, 777.0)
        ops.gemm_fp8_block_nt(again, x, sx, w, sw, max_cus)
        assert torch.equal(again, out), max_cus
    space = torch.full((size // 4 + 64,), float("nan"), device="cuda")
    again = torch.empty_like(out)
    _lib.check(L.tw_gemm_fp8_block_nt(again.data_ptr(), x.data_ptr(), sx.data_ptr(), sx.stride(0), sx.stride(1), w.data_ptr(),
                                      sw.data_ptr(), M, N, K, N, ops._DTYPE_CODE[dtype], 0, space.data_ptr(), size,
                                      torch.cuda.current_stream().cuda_stream))
    assert torch.equal(again, out) and torch.isnan(space[size // 4:]).all()
