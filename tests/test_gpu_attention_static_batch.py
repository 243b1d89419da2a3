"""`PagedSelfAttention` over a batch in static buffers, as a captured step of the woven schedule keeps it."""
import pytest
import torch

import tokenweave_amd as tw
from test_gpu_attention_layer import D, DEV, H, HK, PAGE, attention

pytestmark = pytest.mark.gpu


class Step:
    """Two calls of one layer, a half of the tokens each, in buffers that stay."""

    def __init__(self, news, even):
        self.news, T = news, sum(news)
        starts = torch.tensor([0] + news).cumsum(0).int()
        self.cache = tw.KVCache4(8 * len(news), PAGE, HK, D, DEV)
        old = torch.randn(8 * len(news) * PAGE, HK, D, generator=torch.Generator(device=DEV).manual_seed(4), device=DEV)
        self.cache.append(old, old.flip(0), torch.arange(len(old), device=DEV))
        self.table = torch.randperm(8 * len(news)).int().view(len(news), 8).to(DEV)
        self.lens = torch.zeros(len(news), dtype=torch.int32, device=DEV)
        self.slots, self.positions = (torch.zeros(T, dtype=torch.int64, device=DEV) for _ in range(2))
        self.rows = torch.cat([torch.full((m,), i) for i, m in enumerate(news)]).to(DEV)
        self.x = torch.randn(T, H, device=DEV, generator=torch.Generator(device=DEV).manual_seed(6)).bfloat16()
        self.hidden = torch.empty_like(self.x)
        self.attn = attention(self.cache)
        self.attn.begin(tw.CachedBatch(self.slots, self.table, self.lens, None if even else starts.to(DEV), max(news)))

    def set(self, lengths):
        self.lens.copy_(torch.tensor(lengths, dtype=torch.int32))
        self.positions.copy_(torch.cat([torch.arange(n - m, n) for n, m in zip(lengths, self.news)]))
        self.slots.copy_(self.table[self.rows, self.positions // PAGE].long() * PAGE + self.positions % PAGE)
        self.hidden.copy_(self.x)

    def run(self, cut):
        for i, part in enumerate((slice(0, cut), slice(cut, None))):
            hs = self.hidden[part]
            self.attn(positions=self.positions[part], hidden_states=hs, split_id=i, split_size=cut, num_actual_tokens=len(hs))

    def whole(self):
        """The same step in one call."""
        self.hidden.copy_(self.x)
        self.attn(positions=self.positions, hidden_states=self.hidden)
        return self.hidden.clone()


@pytest.mark.parametrize("news, even, cut, steps", [
    ([1, 1, 1, 1], True, 2, ([30, 40, 50, 60], [31, 41, 51, 61], [100, 1, 2, 90])),
    ([3, 3, 3], True, 4, ([30, 40, 50], [33, 3, 53], [101, 7, 9])),
    ([5, 40, 1, 20], False, 25, ([30, 40, 50, 60], [35, 80, 51, 80], [100, 41, 2, 20]))])
def test_a_captured_split_step_follows_its_lengths(news, even, cut, steps):
    """Sums of the halves may be cut differently from the whole's: one 16-bit rounding of the attention's output and one of
    the projection's apart."""
    s = Step(news, even)
    s.set(steps[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s.run(cut)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        s.run(cut)
    for lengths in steps + steps:
        s.set(lengths)
        graph.replay()
        torch.cuda.synchronize()
        replayed = s.hidden.clone()
        s.hidden.copy_(s.x)
        s.run(cut)
        assert torch.equal(replayed, s.hidden)
        torch.testing.assert_close(replayed.float(), s.whole().float(), rtol=2.0 ** -7, atol=2.0 ** -6)
