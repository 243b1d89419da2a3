"""Rows of tokens that no sequence has: padding behind a step's tokens, or before them."""
import math

import pytest
import torch

import tokenweave_amd as tw
from test_gpu_attention_layer import D, DEV, H, HK, PAGE, attention, batch
from test_gpu_kv4_attention import Case
from tokenweave_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("before, behind", [(0, 1), (0, 700), (3, 0), (5, 40)])
@pytest.mark.parametrize("lengths, news, Hq, Hk, head", [([300, 70], [1, 2], 8, 2, 128), ([5, 3], [1, 1], 6, 1, 64),
                                                         ([300, 70], [120, 70], 4, 1, 128), ([90], [40], 4, 2, 256),
                                                         ([200] * 3, [50] * 3, 2, 1, 64)])
@pytest.mark.parametrize("aligned", [True, False])
def test_rows_without_a_sequence_are_zeros(lengths, news, Hq, Hk, head, before, behind, aligned):
    c = Case(lengths, news, Hq, Hk, head, 16)
    want = c.run()
    T = sum(news)
    q = torch.zeros(before + T + behind, Hq, head, dtype=c.q.dtype, device=DEV)
    q[before:before + T] = c.q
    wide = torch.full((len(q), Hq, head + 8), math.nan, dtype=c.q.dtype, device=DEV)
    out = wide[..., 8:] if aligned else wide[..., 3:3 + head]
    ops.kv4_attention(out, q, c.cache.pages, c.table, c.seq_lens, head ** -0.5, c.starts + before, max(news))
    assert torch.equal(out[before:before + T], want)
    assert not out[:before].any() and not out[before + T:].any()
    assert wide.isnan().sum() == len(q) * Hq * 8


@pytest.mark.parametrize("sequences", [0, 2])
def test_a_step_of_padding_alone(sequences):
    c = Case([9] * 2, [0] * 2, 4, 2)
    q = torch.randn(33, 4, 128, device=DEV).bfloat16()
    starts = torch.zeros(sequences + 1, dtype=torch.int32, device=DEV)
    for most in (0, 4, None):
        out = torch.full_like(q, 3.0)
        c.cache.attend(q, c.table[:sequences], c.seq_lens[:sequences], None, starts, most, 0, out)
        assert not out.any()


def test_padded_rows_of_a_layer_are_the_same_every_time():
    """A step padded to a captured graph's size: what its padding rows bring to the projection is zero, whatever memory
    the output was given."""
    cache = tw.KVCache4(9, PAGE, HK, D, DEV)
    old = torch.randn(9 * PAGE, HK, D, generator=torch.Generator(device=DEV).manual_seed(7), device=DEV)
    cache.append(old, old.flip(0), torch.arange(9 * PAGE, device=DEV))
    attn = attention(cache)
    table = torch.tensor([[5, 0, 7], [1, 8, 2]], dtype=torch.int32, device=DEV)
    positions, step = batch(cache, [20, 33], [20, 1], table)
    pad = 43
    step.slots = torch.cat((step.slots, torch.full((pad,), -1, device=DEV)))
    positions = torch.cat((positions, torch.zeros(pad, dtype=torch.int64, device=DEV)))
    attn.begin(step)
    found = []
    for fill in (math.nan, 1e4):
        x = torch.randn(21 + pad, H, generator=torch.Generator(device=DEV).manual_seed(2), device=DEV).bfloat16()
        # (what the allocator gives next)
        held = [torch.full((21 + pad, 4, D), fill, dtype=torch.bfloat16, device=DEV) for _ in range(8)]
        del held
        attn(positions=positions, hidden_states=x)
        assert not x[21:].any()
        found.append(x)
    assert torch.equal(*found)
