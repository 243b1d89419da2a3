"""Attention over the 4-bit cache where it can go wrong: values that are not numbers in masked places, running
maxima that move, more sequences than a wave holds, tiles past the even shares, caches past 32-bit offsets."""
import math

import pytest
import torch

import tokenweave_amd as tw
from kv4_reference import attend, attend_bound
from test_gpu_kv4_attention import DEV, Case

pytestmark = pytest.mark.gpu


def check(c, got, window=0, values=None, tokens=None):
    """Within the bound of the reference, and of probabilities below fp16's normal range: they are held times 2^7
    or more of the largest, so each is off by at most half of 2^-24 2^-7 of it."""
    values = c.values if values is None else values
    want, mean, size = attend(c.q, c.keys, values, c.lengths, c.news, c.D ** -0.5, window)
    most = max([float(v.abs().max()) for v in values if v.numel()] + [0.0])
    bound = attend_bound(want, mean, size, got.dtype, max(c.lengths + [1])) + max(c.lengths + [1]) * 2.0 ** -32 * most
    far = (got.double().cpu() - want).abs()
    ok = far <= bound
    if tokens is not None:
        ok = ok | tokens
    assert ok.all(), (float((far - bound)[~ok].max()), float((far / bound)[~ok].max()))


@pytest.mark.parametrize("window", [0, 1, 37, 150])
@pytest.mark.parametrize("lengths, news, Hq, Hk, D, page", [
    ([300, 77], [3, 4], 4, 1, 128, 16), ([300, 77], [3, 4], 4, 2, 64, 64), ([140, 33], [5, 2], 4, 1, 256, 32),
    ([300, 150], [300, 100], 4, 1, 128, 64), ([410, 70], [200, 70], 6, 2, 64, 16), ([200], [90], 4, 1, 256, 64)])
def test_not_a_number_values_reach_the_rows_that_see_them_alone(lengths, news, Hq, Hk, D, page, window):
    c = Case(lengths, news, Hq, Hk, D, page)
    g = torch.Generator().manual_seed(11)
    values, hit = [], []
    for i, n in enumerate(lengths):
        v = c.values[i].clone()
        bad = torch.zeros((Hk, n, D // 32), dtype=torch.bool)
        for t in {0, n // 2, n - news[i], n - 1} | set(torch.randint(0, n, (4,), generator=g).tolist()):
            bad[int(torch.randint(0, Hk, (1,), generator=g)), t, int(torch.randint(0, D // 32, (1,), generator=g))] = True
        channels = bad.repeat_interleave(32, -1)
        slots = c.slots(i, n)
        v_new = torch.where(channels, math.nan, v).transpose(0, 1).float().to(DEV)
        c.cache.append(c.keys[i].transpose(0, 1).float().to(DEV).contiguous(), v_new.contiguous(), slots)
        k, back = c.cache.read(slots, torch.float32)
        assert torch.equal(k.double().cpu().transpose(0, 1), c.keys[i])
        assert torch.equal(back.isnan().cpu().transpose(0, 1), channels)
        values.append(torch.where(channels, 0.0, v))
        hit.append(channels.double())
    got = c.run(window)
    # a row is hit in a channel where a seen token is
    want = []
    for i, (n, m) in enumerate(zip(lengths, news)):
        last = n - m + torch.arange(m)[:, None]
        t = torch.arange(n)
        sees = (t <= last) & ((t > last - window) if window else torch.ones_like(t, dtype=torch.bool))
        want.append((sees.double() @ hit[i].repeat_interleave(Hq // Hk, 0) > 0).transpose(0, 1))
    want = torch.cat(want)
    assert torch.equal(got.isnan().cpu(), want)
    check(c, torch.where(want.to(DEV), 0.0, got), window, values, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("how", ["rising", "falling", "spikes"])
@pytest.mark.parametrize("lengths, news, D", [([700, 130], [1, 3], 128), ([700, 130], [300, 130], 128),
                                              ([400], [200], 64), ([300], [120], 256)])
def test_running_maxima_that_move(lengths, news, D, how, dtype):
    """Scores that climb a little each token, fall, or jump: a base of the exponents that is kept while the
    maximum is near it, and is raised where it is not."""
    c = Case(lengths, news, 8, 1, D, 32, dtype)
    direction = torch.where(torch.arange(D, device=DEV) % 2 == 0, 1.0, -1.0)
    for i, n in enumerate(lengths):
        t = torch.arange(n, device=DEV, dtype=torch.float32)
        by = {"rising": t * 0.06, "falling": -t * 0.06, "spikes": (t % 97 == 96) * (t * 0.05)}[how]
        k = (torch.randn(n, 1, D, device=DEV, generator=torch.Generator(device=DEV).manual_seed(i)) * 0.3
             + by[:, None, None] * direction / D ** 0.5)
        slots = c.slots(i, n)
        c.cache.append(k, c.values[i].transpose(0, 1).float().to(DEV).contiguous(), slots)
        c.keys[i] = c.cache.read(slots, torch.float32)[0].double().cpu().transpose(0, 1)
    # q k scale moves by about the step of `by` a token
    c.q = (c.q * 0.3 + direction).to(dtype)
    check(c, c.run())


@pytest.mark.parametrize("news", [3, 200])
@pytest.mark.parametrize("first, second", [(-2000.0, 300.0), (-30000.0, 5.0), (4000.0, 4002.0), (700.0, -900.0)])
def test_scores_far_from_zero(first, second, news):
    """Scores around one value in the first half and around another in the second.  Beside the reference's bound:
    a score's own error, the sum of |q k| 2^-21, is as large as some of these scores' differences, so a probability is
    off by no more than a factor of exp of twice it."""
    c = Case([400], [news], 8, 1, 128, 32)
    direction = torch.where(torch.arange(128, device=DEV) % 2 == 0, 1.0, -1.0)
    t = torch.arange(400, device=DEV)
    by = torch.where(t < 100, first, second)[:, None, None]
    k = torch.randn(400, 1, 128, device=DEV, generator=torch.Generator(device=DEV).manual_seed(2)) * by.abs() * 2.0 ** -10
    slots = c.slots(0, 400)
    c.cache.append(k + by * direction / 128 ** 0.5, c.values[0].transpose(0, 1).float().to(DEV).contiguous(), slots)
    c.keys[0] = c.cache.read(slots, torch.float32)[0].double().cpu().transpose(0, 1)
    c.q = direction.expand(news, 8, 128).contiguous().to(torch.bfloat16)
    got = c.run()
    want, mean, size = attend(c.q, c.keys, c.values, c.lengths, c.news, 128 ** -0.5)
    most = float(c.values[0].abs().max())
    off = torch.expm1(2 * size * 2.0 ** -21)
    bound = attend_bound(want, mean, 0 * size, got.dtype, 400) + (mean + want.abs()) * off + 400 * 2.0 ** -32 * most
    far = (got.double().cpu() - want).abs()
    assert (far <= bound).all(), (float((far - bound).max()), float((far / bound).max()))


@pytest.mark.parametrize("news", [1, 100])
def test_many_small_probabilities_beside_a_large_one(news):
    """One token, and 8000 that are 2^-22 of it each: together they are 0.2 % of the sum, and of the output."""
    c = Case([8001], [news], 4, 1, 128, 64)
    direction = torch.where(torch.arange(128, device=DEV) % 2 == 0, 1.0, -1.0)
    by = torch.full((8001, 1, 1), -8.0, device=DEV)
    by[5] = 8.0
    v = torch.ones(8001, 1, 128, device=DEV)
    v[5] = 0.5
    slots = c.slots(0, 8001)
    c.cache.append((by * direction).contiguous(), v, slots)
    c.keys[0], c.values[0] = (x.double().cpu().transpose(0, 1) for x in c.cache.read(slots, torch.float32))
    # a score is +-8 * 128 * size * 128^-0.5
    size = 22 * math.log(2) / 16 / 128 ** 0.5
    c.q = (direction * size).expand(news, 4, 128).contiguous().to(torch.float16)
    check(c, c.run())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("news", [1, 40])
def test_one_visible_token_is_copied(news, dtype):
    """A softmax over one token is one: the output is the value, which both types hold exactly."""
    c = Case([50], [news], 8, 2, 64, 16, dtype)
    got = c.run(window=1)
    want = c.values[0][:, 50 - news:].transpose(0, 1).repeat_interleave(4, 1)
    assert torch.equal(got.double().cpu(), want)


def test_more_sequences_than_a_wave_holds():
    g = torch.Generator().manual_seed(5)
    lengths = torch.randint(0, 200, (330,), generator=g).tolist()
    lengths[301] = 3000
    c = Case(lengths, [1] * 330, 4, 1, 64, 16)
    check(c, c.run())
    check(c, c.run(70), 70)


@pytest.mark.parametrize("heads", [1, 8])
def test_more_pieces_than_workgroups(heads):
    """Many sequences of several steps each: a workgroup takes piece after piece."""
    c = Case([900 + i for i in range(40)], [2] * 40, 2 * heads, heads, 64, 64)
    check(c, c.run())


@pytest.mark.parametrize("window", [0, 20])
def test_tiles_past_the_even_shares(window):
    """600 short prompts over two key heads: one workgroup for each tile and head."""
    c = Case([30 + i % 50 for i in range(600)], [20 + i % 31 for i in range(600)], 4, 2, 64, 16)
    check(c, c.run(window), window)


@pytest.mark.parametrize("D, page, window", [(64, 16, 0), (64, 256, 90), (128, 16, 33), (256, 16, 0), (256, 128, 65)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_prompts_of_uneven_lengths(D, page, window, dtype):
    lengths, news = [1, 513, 64, 200, 0, 95], [1, 130, 64, 7, 0, 95]
    c = Case(lengths, news, 12, 4, D, page, dtype)
    check(c, c.run(window), window)


def test_fewer_queries_than_a_prompt_has():
    """Tokens behind max_queries are not computed; the others are as if all were."""
    c = Case([400, 90], [300, 90], 2, 1)
    out = torch.full(c.q.shape, 5.0, dtype=c.q.dtype, device=DEV)
    c.cache.attend(c.q, c.table, c.seq_lens, None, c.starts, 70, 0, out)
    rows = list(range(70)) + list(range(300, 370))
    rest = [i for i in range(390) if i not in rows]
    assert bool((out[rest] == 5).all())
    whole = c.run()
    # (shares of the work begin elsewhere: two roundings of the output apart)
    torch.testing.assert_close(out[rows], whole[rows], rtol=2.0 ** -7, atol=2.0 ** -9)


@pytest.mark.parametrize("news", [1, 64])
def test_offsets_past_32_bits(news):
    """A cache of 4.7 GB whose last pages are used."""
    D, page, last = 128, 256, 135_000
    cache = tw.KVCache4(last, page, 1, D, DEV)
    n = 700
    slots = (last - 1 - torch.arange(n, device=DEV) // page) * page + torch.arange(n, device=DEV) % page
    assert int(slots.min()) // page * cache.pages.shape[-1] > 1 << 32
    g = torch.Generator(device=DEV).manual_seed(3)
    k, v = (torch.randn(n, 1, D, generator=g, device=DEV) for _ in range(2))
    cache.append(k, v, slots)
    k, v = (x.double().cpu().transpose(0, 1) for x in cache.read(slots, torch.float32))
    assert k.abs().amax() > 2 and v.abs().amax() > 2
    table = (last - 1 - torch.arange(3, device=DEV)).int()[None]
    q = torch.randn(news, 2, D, generator=g, device=DEV).bfloat16()
    lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    got = cache.attend(q, table, lens, None, torch.tensor([0, news], dtype=torch.int32, device=DEV), news)
    want, mean, size = attend(q, [k], [v], [n], [news], D ** -0.5)
    assert ((got.double().cpu() - want).abs() <= attend_bound(want, mean, size, got.dtype, n)).all()
