"""The feed-forward modules' bookkeeping, without a GPU: what they refuse, what they load, what a model's type leaves
alone."""
import pytest
import torch

import tokenweave_amd as tw

BF16, FP8 = torch.bfloat16, torch.float8_e4m3fn


def filled(layer, seed=0):
    g = torch.Generator().manual_seed(seed)
    for p in layer.parameters():
        p.data.copy_(torch.randn(p.shape, generator=g))
    return layer


@pytest.mark.parametrize("fp8", [False, True])
def test_a_block_whose_gradient_is_wanted_is_refused(fp8):
    """Its result lies where its input lay: autograd would take the block for the identity."""
    leaf = torch.randn(4, 64).to(BF16).requires_grad_()
    block = filled(tw.FeedForward(64, 96))
    if fp8:
        block.to_fp8_blocks()
    with pytest.raises(RuntimeError, match="FeedForward records no gradient"):
        block(2 * leaf)
    for part in (block.gate_up, block.down):
        part.weight.requires_grad_()
        with pytest.raises(RuntimeError, match="FeedForward records no gradient"):
            block(torch.randn(4, 64).to(BF16))
        with torch.no_grad(), pytest.raises(RuntimeError, match="GPU"):   # past the refusal
            block(torch.randn(4, 64).to(BF16))
        part.weight.requires_grad_(False)
    with pytest.raises(RuntimeError, match="GPU"):
        block(torch.randn(4, 64).to(BF16))


@pytest.mark.parametrize("make", [lambda: tw.RowParallelLinear(64, 64, bias=False), lambda: tw.GatedLinear(64, 32)])
def test_a_models_type_is_a_bf16_weights_whatever_stands_beside_it(make):
    """`weight_scale` is any method's name for its scales: only e4m3 codes keep their type."""
    for holder in (torch.nn.Parameter(torch.ones(1), requires_grad=False), torch.ones(1)):
        layer = filled(make())
        layer.weight_scale = holder
        assert layer.half().weight.dtype == torch.float16
        assert layer.weight_scale.dtype == (torch.float16 if isinstance(holder, torch.nn.Parameter) else torch.float32)


def values(codes, scales):
    N, K = codes.shape
    return codes.double() * scales.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]


@pytest.mark.parametrize("tp", [1, 2])
def test_8_bit_weights_are_loaded(tp):
    """A whole model's codes and scales: every rank's layers stand for its part of the whole weights."""
    hidden, inner = 144, 512
    gate, up, down = (tw.quantize_fp8_blocks(torch.randn(s)) for s in ((inner, hidden), (inner, hidden), (hidden, inner)))
    n = inner // tp
    for rank in range(tp):
        block = filled(tw.FeedForward(hidden, inner, tp_rank=rank, tp_size=tp)).to_fp8_blocks()
        for shard, (codes, scales) in enumerate((gate, up)):
            block.gate_up.weight_loader(block.gate_up.weight, codes, shard)
            block.gate_up.weight_loader(block.gate_up.weight_scale, scales, shard)
        block.down.weight_loader(block.down.weight, down[0])
        block.down.weight_loader(block.down.weight_scale, down[1])
        rows = slice(rank * n, (rank + 1) * n)
        want = torch.cat((values(*gate)[rows], values(*up)[rows]))
        assert torch.equal(values(block.gate_up.weight, block.gate_up.weight_scale), want)
        assert torch.equal(values(block.down.weight, block.down.weight_scale), values(*down)[:, rows])
        # one rank's own, as a sharded checkpoint has them
        block.down.weight_loader(block.down.weight_scale, block.down.weight_scale.data * 2)
        assert torch.equal(values(block.down.weight, block.down.weight_scale), 2 * values(*down)[:, rows])


def test_8_bit_weights_that_do_not_fit_are_refused():
    block = filled(tw.FeedForward(64, 96)).to_fp8_blocks()
    with pytest.raises(ValueError, match="holds 8-bit codes"):
        block.gate_up.weight_loader(block.gate_up.weight, torch.zeros(96, 64, dtype=BF16), 0)
    with pytest.raises(ValueError, match="holds 8-bit codes"):
        block.down.weight_loader(block.down.weight, torch.zeros(64, 96, dtype=BF16))
    with pytest.raises(ValueError, match="inside a block of 128"):      # the up rows begin inside the gate rows' last block
        block.gate_up.weight_loader(block.gate_up.weight_scale, torch.ones(1, 1), 0)
    block = filled(tw.FeedForward(64, 384, tp_rank=1, tp_size=2)).to_fp8_blocks()
    with pytest.raises(ValueError, match="inside a block of 128"):
        block.down.weight_loader(block.down.weight_scale, torch.ones(1, 3))


def test_an_8_bit_block_takes_any_leading_dimensions():
    block = filled(tw.FeedForward(64, 96)).to_fp8_blocks()
    with pytest.raises(RuntimeError, match="GPU"):      # no complaint about the shape
        block(torch.zeros(2, 3, 64, dtype=BF16))


def test_a_gated_projection_alone_has_no_8_bit_form():
    layer = tw.GatedLinear(64, 32)
    with pytest.raises(ValueError, match="to_fp8_blocks"):
        tw.Fp8BlockLinearMethod().process_weights(layer)
    assert layer.weight.dtype == BF16 and not hasattr(layer, "weight_scale")


def test_row_counts_next_to_32_bits_are_refused():
    """Before anything is launched: a tile's last rows would be counted past them."""
    from tokenweave_amd import _lib
    L, at = _lib.lib(), 1 << 12
    for M in (2 ** 31 - 1, 2 ** 31 - 16, 2 ** 31):
        assert L.tw_quant_fp8_groups(at, at, 1, M, at, 8, M, 8, -1, 0, None) == _lib.TW_ERR_INVALID_ARGUMENT
        assert L.tw_gated_gemm_bf16_nt(at, at, at, at, M, 4, 8, 4, 8, 0, 0, None, 0, None) == _lib.TW_ERR_INVALID_ARGUMENT


def test_the_build_follows_its_makefiles_and_headers():
    """How many jobs run is the caller's choice; flags and headers that change are compiled in."""
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

    def make(where, *args):
        env = {k: v for k, v in os.environ.items() if k not in ("MAKEFLAGS", "MFLAGS", "MAKELEVEL")}
        return subprocess.run(["make", "-C", os.path.join(root, where), *args], capture_output=True, text=True, env=env).stdout

    csrc = os.path.join("tokenweave_amd", "csrc")
    flags = [line for line in make(csrc, "-pn", "-j2", "lib").splitlines() if line.startswith("MAKEFLAGS")]
    assert flags and not any("-j8" in line for line in flags), flags
    assert make(csrc, "-n", "-W", "Makefile", "lib").count(" -c -o build/") >= 9
    for header in ("tw_activation.h", "tw_store.h"):
        assert "tw_bench.hip" in make("benchlib", "-n", "-W", f"../tokenweave_amd/csrc/{header}")


def test_weight_codes_and_scales_have_no_history():
    """Of a weight in training: what the products take as constants, not tensors that want a gradient."""
    w = torch.randn(130, 144).requires_grad_()
    codes, scales = tw.quantize_fp8_blocks(w)
    assert not codes.requires_grad and not scales.requires_grad
    want = tw.quantize_fp8_blocks(w.detach())
    assert torch.equal(codes.view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(scales, want[1])


def test_an_e4m3_weight_without_scales_is_a_weight_like_others():
    """A type that a layer was made with, not codes of another weight: it follows the model's and takes any values."""
    layer = tw.RowParallelLinear(64, 64, bias=False, params_dtype=FP8)
    layer.weight_loader(layer.weight, torch.ones(64, 64, dtype=BF16))
    assert (layer.weight.float() == 1).all() and layer.half().weight.dtype == torch.float16
