"""The halves of a step's tokens: they follow their batch's tensors."""
import pytest
import torch

import tokenweave_amd as tw


def where(half, base):
    """(token, sequence, position) of every new token of a half."""
    s, n = half.query_starts.tolist(), half.seq_lens.tolist()
    return [(base + s[i] + j, i, n[i] - (s[i + 1] - s[i]) + j) for i in range(len(n)) for j in range(s[i + 1] - s[i])]


def test_halves_follow_lengths_and_starts_that_change_in_place():
    """Static buffers: a step writes its lengths and starts over the last step's."""
    starts, lens = (torch.tensor(x, dtype=torch.int32) for x in ([0, 3, 4, 10, 12], [30, 5, 6, 100]))
    batch = tw.CachedBatch(torch.arange(12), torch.zeros(4, 2, dtype=torch.int32), lens, starts, 9)
    halves = batch.split(5)
    for new_starts, new_lens in (([0, 3, 4, 10, 12], [31, 6, 7, 101]), ([0, 1, 2, 11, 12], [8, 50, 9, 4])):
        starts.copy_(torch.tensor(new_starts)), lens.copy_(torch.tensor(new_lens))
        whole = [(t, i, new_lens[i] - new_starts[i + 1] + t) for i in range(4) for t in range(new_starts[i], new_starts[i + 1])]
        for first, second in (halves, batch.split(5)):
            assert where(first, 0) + where(second, 5) == whole


def test_halves_of_single_tokens_follow_their_lengths():
    lens = torch.tensor([30, 40, 50, 60], dtype=torch.int32)
    batch = tw.CachedBatch(torch.arange(4), torch.zeros(4, 2, dtype=torch.int32), lens)
    first, second = batch.split(2)
    lens += 1
    assert first.seq_lens[:2].tolist() == [31, 41] and second.seq_lens[-2:].tolist() == [51, 61]
    again = batch.split(2)
    assert again[0].seq_lens[:2].tolist() == [31, 41] and again[1].seq_lens[-2:].tolist() == [51, 61]


def test_halves_follow_tensors_that_are_replaced():
    batch = tw.CachedBatch(torch.arange(4), torch.zeros(4, 2, dtype=torch.int32), torch.tensor([30, 40, 50, 60], dtype=torch.int32))
    batch.split(2)
    batch.seq_lens, batch.slots = torch.tensor([1, 2, 3, 4], dtype=torch.int32), torch.arange(4) + 7
    first, second = batch.split(2)
    assert first.seq_lens[:2].tolist() == [1, 2] and second.seq_lens[-2:].tolist() == [3, 4]
    assert first.slots.tolist() + second.slots.tolist() == [7, 8, 9, 10]


def test_halves_keep_a_bound_on_a_sequences_new_tokens():
    """The bound picks the kernel: without one, a half with starts counts all its tokens as one sequence's."""
    table = torch.zeros(4, 2, dtype=torch.int32)
    for each, cut in ((1, 2), (1, 4), (3, 6), (3, 5), (3, 0)):
        lens = torch.full((4,), 40, dtype=torch.int32)
        batch = tw.CachedBatch(torch.arange(4 * each), table, lens)
        covered = []
        for half, base in zip(batch.split(cut), (0, cut)):
            n, starts = half.seq_lens.numel(), half.query_starts
            assert half.block_table.shape == (n, 2)
            if starts is None:     # the op's own bound: the same number each
                assert half.max_queries in (None, each) and half.slots.numel() == n * each
                starts = torch.arange(n + 1) * each
            else:
                assert half.max_queries == each
            assert (starts[1:] - starts[:-1]).max() <= each if n else half.slots.numel() == 0
            covered += half.slots[int(starts[0]):int(starts[-1])].tolist()
        assert covered == list(range(4 * each))
    starts = torch.tensor([0, 3, 4], dtype=torch.int32)
    for bound in (None, 3):
        batch = tw.CachedBatch(torch.arange(4), table[:2], torch.tensor([9, 9], dtype=torch.int32), starts, bound)
        assert all(half.max_queries == bound for half in batch.split(2))
    # what the op refuses of a whole batch is refused of its halves
    with pytest.raises(RuntimeError, match="same number for each"):
        tw.CachedBatch(torch.arange(5), table[:2], torch.tensor([9, 9], dtype=torch.int32)).split(2)
