"""Attention where scores are so large that neighbouring fp32 values are further apart than the exponents' range."""
import pytest
import torch

from kv4_reference import attend, attend_bound
from test_gpu_kv4_attention import DEV, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("news", [1, 3, 100])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("size", [1e5, 4e6, 1e7, 3e7, 1e8, 1e9, 1e20, 1e36])
@pytest.mark.parametrize("dtype, D", [(torch.bfloat16, 128), (torch.float16, 64), (torch.bfloat16, 256)])
def test_the_largest_score_takes_all(dtype, D, size, sign, news):
    """Every product and sum of q k is exact here and tokens 37 and 210 have the same, largest one, by a third of its
    size: the output is their values' mean (or the one that is visible), to the probabilities' and the output's rounding."""
    c = Case([300], [news], 8, 1, D, 32, dtype)
    direction = torch.where(torch.arange(D, device=DEV) % 2 == 0, 1.0, -1.0)
    top, other = (6.0, 4.0) if sign > 0 else (4.0, 6.0)
    by = torch.full((300, 1, 1), other, device=DEV)
    by[[37, 210]] = top
    slots = c.slots(0, 300)
    c.cache.append(by * direction, c.values[0].transpose(0, 1).float().to(DEV).contiguous(), slots)
    c.keys[0] = c.cache.read(slots, torch.float32)[0].double().cpu().transpose(0, 1)
    g = torch.Generator(device=DEV).manual_seed(3)
    each = 1 + torch.rand(news, 8, 1, generator=g, device=DEV)
    c.q = (each * direction * sign).to(dtype)
    scale = size / (top * D)
    got = c.run(scale=scale)
    want, mean, big = attend(c.q, c.keys, c.values, c.lengths, c.news, scale)
    far = (got.double().cpu() - want).abs()
    assert (far <= attend_bound(want, mean, 0 * big, dtype, 300)).all(), (int(got.isnan().sum()), float(far.nan_to_num(0).max()))
