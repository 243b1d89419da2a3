"""Attention over the 4-bit cache against softmax in 64 bits on what the cache holds."""
import math

import pytest
import torch

import tokenweave_amd as tw
from kv4_reference import attend, attend_bound
from tokenweave_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


class Case:
    """Sequences of the given cached and new tokens, in pages taken in random order."""

    def __init__(self, lengths, news, Hq=8, Hk=1, D=128, page=64, dtype=torch.bfloat16, seed=1, std=1.0, spare=3):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.lengths, self.news, self.page, self.D = list(lengths), list(news), page, D
        counts = [-(-n // page) for n in lengths]
        self.cache = tw.KVCache4(sum(counts) + spare, page, Hk, D, DEV)
        # what was never written: not-a-number scales
        self.cache.pages.fill_(0xFF)
        order = torch.randperm(sum(counts) + spare, generator=g, device=DEV).int()
        width = max(counts + [1])
        self.table = torch.full((len(counts), width), -1, dtype=torch.int32, device=DEV)
        self.keys, self.values, first = [], [], 0
        for i, (n, c) in enumerate(zip(lengths, counts)):
            self.table[i, :c] = order[first:first + c]
            first += c
            slots = self.slots(i, n)
            k, v = (torch.randn(n, Hk, D, generator=g, device=DEV) * std for _ in range(2))
            self.cache.append(k, v, slots)
            k, v = self.cache.read(slots, torch.float32)
            self.keys.append(k.double().cpu().transpose(0, 1))
            self.values.append(v.double().cpu().transpose(0, 1))
        T = sum(news)
        qkv = torch.randn(T, (Hq + 2 * Hk) * D, generator=g, device=DEV).to(dtype)
        self.q = qkv[:, :Hq * D].view(T, Hq, D)
        self.seq_lens = torch.tensor(lengths, dtype=torch.int32, device=DEV)
        self.starts = torch.tensor([0] + news, device=DEV).cumsum(0).int()

    def slots(self, i, n):
        t = torch.arange(n, device=DEV)
        return self.table[i].long()[t // self.page] * self.page + t % self.page

    def run(self, window=0, scale=None, **kw):
        out = torch.full(self.q.shape, math.nan, dtype=self.q.dtype, device=DEV)
        return self.cache.attend(self.q, self.table, self.seq_lens, scale, self.starts, max(self.news + [0]), window, out, **kw)

    def check(self, got, window=0, scale=None):
        want, mean, size = attend(self.q, self.keys, self.values, self.lengths, self.news,
                                  self.D ** -0.5 if scale is None else scale, window)
        far = (got.double().cpu() - want).abs()
        bound = attend_bound(want, mean, size, got.dtype, max(self.lengths + [1]))
        assert (far <= bound).all(), (float((far - bound).max()), float((far / bound).max()))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hq, Hk, D", [(8, 1, 128), (6, 1, 128), (16, 2, 128), (4, 4, 64), (8, 2, 256), (32, 1, 64)])
@pytest.mark.parametrize("lengths", [[1], [2, 31, 32, 33], [63, 64, 65, 127, 128, 129], [1000, 5, 300]])
def test_one_new_token_each(lengths, Hq, Hk, D, dtype):
    c = Case(lengths, [1] * len(lengths), Hq, Hk, D, 16 if D == 64 else 64, dtype)
    c.check(c.run())
    # the same without query_starts
    out = c.cache.attend(c.q, c.table, c.seq_lens)
    assert torch.equal(out, c.run())


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_page_sizes_and_a_long_sequence(page):
    c = Case([5000, 3, 4096], [1, 1, 1], page=page)
    c.check(c.run())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lengths, news, Hq, Hk, D", [
    ([100, 7, 64], [4, 4, 4], 6, 1, 128), ([200, 90], [2, 5], 8, 2, 64), ([40, 300, 9], [3, 7, 1], 28, 4, 128),
    ([130, 65], [130, 65], 8, 1, 128), ([300, 77, 1], [100, 77, 1], 4, 2, 256), ([500, 260], [37, 200], 16, 2, 64),
    ([1025], [1025], 2, 1, 128)])
def test_several_new_tokens(lengths, news, Hq, Hk, D, dtype):
    c = Case(lengths, news, Hq, Hk, D, 32, dtype)
    c.check(c.run())


@pytest.mark.parametrize("window", [1, 2, 31, 64, 65, 400, 100000])
@pytest.mark.parametrize("lengths, news", [([700, 33, 5], [1, 1, 1]), ([600, 129], [200, 129]), ([333, 90], [3, 4])])
def test_window(lengths, news, window):
    c = Case(lengths, news, 6, 1, page=16)
    c.check(c.run(window), window)


def test_rows_that_see_nothing_give_zeros():
    """Sequences without tokens, and more new tokens than cached ones: the first see nothing."""
    c = Case([0, 3, 40, 0], [2, 5, 1, 1], 4, 2)
    got = c.run()
    assert not got[:2].any() and not got[2:4].any() and not got[8].any()
    c.check(got)
    # no room in the table at all
    out = c.cache.attend(c.q, c.table[:, :0], c.seq_lens, None, c.starts, 5)
    assert not out.any()


def test_pages_outside_the_cache_are_masked():
    c = Case([200, 70], [1, 1], page=16)
    for i, holes in ((0, {3: -7, 5: 1 << 30}), (1, {0: -1})):
        keep = torch.ones(c.lengths[i], dtype=torch.bool)
        for place, page in holes.items():
            c.table[i, place] = page
            keep[place * 16:place * 16 + 16] = False
        c.keys[i], c.values[i] = c.keys[i][:, keep], c.values[i][:, keep]
    got = c.run()
    c.lengths = [k.shape[1] for k in c.keys]   # one new token each: it sees all that is left
    c.check(got)


def test_a_sequence_ends_inside_a_page_of_not_a_numbers():
    """The pages' unwritten places hold NaN scales; lengths behind what was written are the caller's."""
    c = Case([17, 100, 63], [1, 3, 63], 8, 2, page=64)
    assert not c.run().isnan().any()


def test_large_and_small_scores():
    """Scores of some thousands (one token takes all) and of almost nothing (all alike)."""
    for scale in (20.0, 1e-6, 0.0, -0.3):
        c = Case([300, 65], [1, 40], 4, 1)
        got = c.run(scale=scale)
        want, mean, size = attend(c.q, c.keys, c.values, c.lengths, c.news, scale)
        far = (got.double().cpu() - want).abs()
        assert (far <= attend_bound(want, mean, size.abs(), got.dtype, 300)).all()


@pytest.mark.parametrize("std", [1e-3, 30.0, 1e4])
def test_small_and_large_cached_values(std):
    c = Case([150, 40], [1, 10], 8, 1, std=std)
    c.check(c.run(scale=0.05 / std), scale=0.05 / std)


def test_queries_over_many_orders_of_magnitude():
    c = Case([90, 33], [2, 2], 8, 1)
    size = torch.tensor([1e-20, 1e-6, 1.0, 1e6], device=DEV)[:, None, None]
    q = (c.q.float() * size).bfloat16()
    for i in range(4):
        c.q = q
        # each row with a scale that brings its scores to order 1
        s = float(0.1 / size[i])
        got = c.run(scale=s)[i:i + 1]
        want, mean, big = (x[i:i + 1] for x in attend(q, c.keys, c.values, c.lengths, c.news, s))
        assert ((got.double().cpu() - want).abs() <= attend_bound(want, mean, big, got.dtype, 90)).all()


def test_not_a_number_in_a_query_stays_in_its_row():
    c = Case([90, 33], [3, 1], 4, 1)
    c.q = c.q.clone()
    c.q[1, 2, 7] = math.nan
    got = c.run()
    assert got[1, 2].isnan().all()
    got[1, 2] = 0
    assert not got.isnan().any()


def test_results_do_not_depend_on_the_batch():
    """A sequence alone and among others; the same call twice."""
    c = Case([700, 1200, 64, 9], [1, 1, 1, 1])
    both = c.run()
    assert torch.equal(both, c.run())
    one = c.cache.attend(c.q[1:2], c.table[1:2], c.seq_lens[1:2])
    torch.testing.assert_close(one, both[1:2], rtol=2.0 ** -7, atol=2.0 ** -12)


def test_out_and_q_of_any_stride():
    c = Case([70, 200], [3, 2], 4, 2)
    want = c.run()
    wide = torch.full((5, 4, 140), 7.0, dtype=torch.bfloat16, device=DEV)
    q = torch.empty(4, 5, 131, dtype=torch.bfloat16, device=DEV).transpose(0, 1)[..., :128].copy_(c.q)
    ops.kv4_attention(wide[..., 3:131], q, c.cache.pages, c.table, c.seq_lens, 128 ** -0.5, c.starts, 3)
    assert torch.equal(wide[..., 3:131], want) and bool((wide[..., :3] == 7).all()) and bool((wide[..., 131:] == 7).all())


def test_fewer_queries_than_there_are():
    """Tokens behind max_queries are not computed, and nothing outside q is read or written."""
    c = Case([64, 64], [4, 4])
    out = torch.full(c.q.shape, 5.0, dtype=c.q.dtype, device=DEV)
    c.cache.attend(c.q, c.table, c.seq_lens, None, c.starts, 2, 0, out)
    whole = c.run()
    assert torch.equal(out[[0, 1, 4, 5]], whole[[0, 1, 4, 5]]) and bool((out[[2, 3, 6, 7]] == 5).all())


def test_lengths_may_change_between_replays_of_a_graph():
    c = Case([300, 900], [1, 1])
    out = torch.zeros_like(c.q, memory_format=torch.contiguous_format)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.cache.attend(c.q, c.table, c.seq_lens, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        c.cache.attend(c.q, c.table, c.seq_lens, out=out)
    for lengths in ([300, 900], [10, 64], [299, 1], [150, 900]):
        c.seq_lens.copy_(torch.tensor(lengths, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        eager = c.cache.attend(c.q, c.table, c.seq_lens)
        assert torch.equal(out, eager)


def test_streams():
    """Calls on several streams at once do not disturb each other."""
    cases = [Case([900 + 10 * i, 400], [1, 1], seed=i) for i in range(3)]
    want = [c.run() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(c.cache.attend(c.q, c.table, c.seq_lens))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i % 3]) for i, g in enumerate(got))


def test_direct_and_ctypes_routes_agree(monkeypatch):
    if ops._fast is None:
        pytest.skip("no compiled binding")
    c = Case([300, 65], [2, 5], 8, 2)
    a = c.run()
    monkeypatch.setattr(ops, "_fast", None)
    assert torch.equal(a, c.run())


def test_refusals():
    c = Case([64, 64], [1, 1], 8, 2)
    q, table, lens, starts = c.q, c.table, c.seq_lens, c.starts
    for bad, match in (((q[:, :7], table, lens), "query heads"), ((q, table.long(), lens), "block_table"),
                       ((q, table, lens.long()), "seq_lens"), ((q, table, lens[:1]), "seq_lens holds 1"),
                       ((q, table, lens, None, starts[:2]), "query_starts holds 2"),
                       ((q[:1], table, lens), "same number for each"), ((q, table, lens, None, starts, -1), "negative"),
                       ((q, table, lens, None, starts, 1, -1), "negative"), ((q[..., :64], table, lens), "head_size 128"),
                       ((q, table.t(), lens), "contiguous rows|seq_lens"), ((q.transpose(1, 2), table, lens), "shape|channels")):
        with pytest.raises(RuntimeError, match=match):
            c.cache.attend(*bad)
    with pytest.raises(NotImplementedError):
        c.cache.attend(q.float(), table, lens)
    with pytest.raises(RuntimeError, match="out has shape"):
        c.cache.attend(q, table, lens, out=q[:1])
