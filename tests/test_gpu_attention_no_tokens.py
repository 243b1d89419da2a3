"""A step, or a half of one, without tokens."""
import pytest
import torch

import tokenweave_amd as tw
from test_gpu_attention_layer import D, DEV, H, HK, PAGE, attention, batch

pytestmark = pytest.mark.gpu


def test_a_half_without_tokens():
    """All of a step's tokens in its first or in its second half: the other call does nothing."""
    cache = tw.KVCache4(9, PAGE, HK, D, DEV)
    attn = attention(cache)
    table = torch.tensor([[5, 0, 7], [1, 8, 2]], dtype=torch.int32, device=DEV)
    positions, step = batch(cache, [20, 33], [20, 33], table)
    x = torch.randn(53, H, generator=torch.Generator(device=DEV).manual_seed(2), device=DEV).bfloat16()
    want = x.clone()
    attn.begin(step)
    attn(positions=positions, hidden_states=want)
    pages = cache.pages.clone()
    for cut in (0, 53):
        got = x.clone()
        for i, part in enumerate((slice(0, cut), slice(cut, 53))):
            attn(positions=positions[part], hidden_states=got[part], split_id=i, split_size=cut, num_actual_tokens=len(got[part]))
        assert torch.equal(got, want) and torch.equal(cache.pages, pages)
    got = x.clone()      # padding behind no tokens stays
    attn(positions=positions[53:], hidden_states=got, split_id=1, split_size=53, num_actual_tokens=0)
    assert torch.equal(got, x)


def test_a_step_without_tokens():
    attn = attention(tw.KVCache4(1, PAGE, HK, D, DEV))
    none = torch.zeros(0, dtype=torch.int64, device=DEV)
    for sequences, starts in ((0, None), (2, torch.zeros(3, dtype=torch.int32, device=DEV))):
        attn.begin(tw.CachedBatch(none, torch.zeros(sequences, 1, dtype=torch.int32, device=DEV),
                                  torch.zeros(sequences, dtype=torch.int32, device=DEV), starts, 0))
        x = torch.empty(0, H, dtype=torch.bfloat16, device=DEV)
        assert attn(positions=none, hidden_states=x) is x
