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
