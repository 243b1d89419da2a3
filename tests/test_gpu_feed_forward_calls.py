"""Calls of the feed-forward half that the documentation allows: any leading dimensions, single rows of odd buffers, scales
of any layout, grid caps, every tile shape that the rules may choose."""
import pytest
import torch

import feed_forward_reference as R
import tokenweave_amd as tw
from tokenweave_amd import ops

pytestmark = pytest.mark.gpu
DEV, BF16, FP8 = "cuda:0", torch.bfloat16, torch.float8_e4m3fn


def filled(layer, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    layer = layer.to(DEV)
    for p in layer.parameters():
        p.data.copy_(torch.randn(p.shape, generator=g, device=DEV) * p.shape[-1] ** -0.5)
    return layer


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("shape", [(2, 9), (3, 1, 2), (2, 0), (1,)])
def test_a_block_of_any_leading_dimensions(shape, fp8):
    block = filled(tw.FeedForward(256, 400))
    if fp8:
        block.to_fp8_blocks()
    x = torch.randn(*shape, 256, device=DEV).to(BF16)
    want = block(x.view(-1, 256).clone())
    hidden = x.clone()
    assert block(hidden) is hidden and torch.equal(hidden.view(-1, 256), want)
