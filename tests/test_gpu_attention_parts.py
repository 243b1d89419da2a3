"""A batch attended in parts: starts below 0 and past q's tokens are other parts' tokens."""
import pytest
import torch

import tokenweave_amd as tw
from test_gpu_kv4_attention import DEV, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window", [0, 30])
@pytest.mark.parametrize("lengths, news, Hq, Hk, D", [([200, 90, 64], [3, 4, 1], 8, 1, 128), ([40, 300, 9], [4, 4, 4], 4, 2, 64),
                                                      ([300, 77, 5], [120, 70, 5], 4, 1, 128), ([200, 60], [90, 60], 4, 2, 256)])
def test_parts_are_the_whole(lengths, news, Hq, Hk, D, window):
    """Every cut in two, and each token alone against the 64-bit statement's bound."""
    c = Case(lengths, news, Hq, Hk, D, 16)
    T, most = sum(news), max(news)
    for cut in sorted({0, 1, 2, news[0], news[0] + 1, T // 2, T - 1, T}):
        out = torch.full_like(c.q, float("nan"), memory_format=torch.contiguous_format)
        for part in (slice(0, cut), slice(cut, T)):
            c.cache.attend(c.q[part], c.table, c.seq_lens, None, c.starts - part.start, most, window, out[part])
        c.check(out, window)
        # the halves of a batch, by lengths and starts of their own and as the layer takes them
        batch = tw.CachedBatch(torch.zeros(T, dtype=torch.int64, device=DEV), c.table, c.seq_lens, c.starts, most)
        for half, part in zip(batch.split(cut), (slice(0, cut), slice(cut, T))):
            for table, lens, starts, bound in ((half.block_table, half.seq_lens, half.query_starts, half.max_queries),
                                               half._operands()):
                got = torch.empty_like(out[part])
                c.cache.attend(c.q[part], table, lens, None, starts, bound, window, got)
                assert torch.equal(got, out[part])


def test_a_part_in_the_middle():
    c = Case([200, 150], [60, 50], 4, 1, 128, 32)
    out = torch.full_like(c.q, float("nan"), memory_format=torch.contiguous_format)
    for a, b in ((0, 20), (20, 55), (55, 70), (70, 71), (71, 110)):
        c.cache.attend(c.q[a:b], c.table, c.seq_lens, None, c.starts - a, b - a, 0, out[a:b])
    c.check(out)
