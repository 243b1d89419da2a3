"""A key that is not a number: the rows that see it are not numbers, the others as without it."""
import math

import pytest
import torch

from test_gpu_kv4_attention import DEV, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("lengths, news, D", [([300, 77], [3, 4], 128), ([300, 77], [3, 4], 256), ([140, 33], [1, 1], 64),
                                              ([300, 150], [300, 100], 128), ([410, 70], [200, 70], 64), ([200], [90], 256)])
def test_rows_that_see_the_key(lengths, news, D, window):
    c = Case(lengths, news, 4, 2, D, 16)
    want = c.run(window)
    hit, first = torch.zeros(len(c.q), 4, dtype=torch.bool), 0
    for i, (n, m) in enumerate(zip(lengths, news)):
        at = n - 1 - m // 2
        k = c.keys[i].clone()
        k[1, at, D // 2] = math.nan      # the second key head's, one block of 32 channels
        c.cache.append(k.transpose(0, 1).float().to(DEV).contiguous(), c.values[i].transpose(0, 1).float().to(DEV).contiguous(),
                       c.slots(i, n))
        own = torch.arange(n - m, n)
        hit[first:first + m, 2:] = ((own >= at) & ((own < at + window) if window else True))[:, None]
        first += m
    got = c.run(window)
    assert hit.any() and not hit.all()
    assert torch.equal(got.isnan().all(-1).cpu(), hit) and torch.equal(got.isnan().any(-1).cpu(), hit)
    assert torch.equal(got[~hit.to(DEV)], want[~hit.to(DEV)])
