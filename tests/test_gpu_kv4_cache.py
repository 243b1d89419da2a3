"""The 4-bit cache's writer and reader: values, bytes, placement, rotation on the way."""
import pytest
import torch

import tokenweave_amd as tw
from kv4_reference import page_bytes, quantise
from tokenweave_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def tokens(T, H, D, dtype, seed=1, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [(torch.randn(T, H, D, generator=g, device=DEV) * std).to(dtype) for _ in range(2)]


def same(a, b):
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T, H, D, page", [(1, 1, 128, 64), (64, 1, 128, 16), (37, 4, 64, 32), (130, 2, 256, 128),
                                           (300, 3, 128, 256), (15, 12, 64, 16)])
def test_round_trip_gives_the_nearest_values(T, H, D, page, dtype):
    k, v = tokens(T, H, D, dtype)
    cache = tw.KVCache4(-(-T // page) + 2, page, H, D, DEV)
    cache.pages.fill_(0xA5)
    slots = torch.randperm(cache.num_pages * page, device=DEV)[:T]
    cache.append(k, v, slots)
    for got, x in zip(cache.read(slots, dtype), (k, v)):
        assert torch.equal(got.double().cpu(), quantise(x))


def test_every_value_of_16_bits():
    """All finite bf16 patterns and all fp16 ones: saturation, small blocks, ties, signs."""
    bits = torch.arange(65536, device=DEV, dtype=torch.int32).to(torch.int16)
    for dtype in (torch.bfloat16, torch.float16):
        x = bits.view(dtype)
        x = x[x.isfinite()]
        x = x[:x.numel() // 64 * 64].view(-1, 1, 64)
        mixed = x.flatten()[torch.randperm(x.numel(), device=DEV)].view_as(x)
        cache = tw.KVCache4(-(-x.shape[0] // 64), 64, 1, 64, DEV)
        slots = torch.arange(x.shape[0], device=DEV)
        cache.append(x, mixed, slots)
        k, v = cache.read(slots, torch.float32)
        assert torch.equal(k.double().cpu(), quantise(x)) and torch.equal(v.double().cpu(), quantise(mixed))


def test_ties_thresholds_and_extremes():
    row = torch.tensor([6.0, 7.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.2500001, 0.7499999, 1.2500001, 1.7499999,
                        2.5000002, 3.4999998, 5.0000005, -0.25, -0.75, -1.25, -1.75, -2.5, -3.5, -5.0, -6.5, 0.0, -0.0,
                        1e-30, -1e-30, 0.5, 1.0, 3.0, 4.0], device=DEV)
    rows = [row, row * 2.0 ** 11, row * 2.0 ** 13, row * 2.0 ** 40, row * 2.0 ** -23, row * 2.0 ** -30, row * 1e-38,
            torch.zeros(32, device=DEV)]
    rows += [torch.full((32,), f, device=DEV) for f in (7.0000005, 6.9999995, 14.0, 3.5, 3.4e38, 2.0 ** -25)]
    x = torch.stack(rows + rows).view(-1, 1, 64)
    cache = tw.KVCache4(2, 16, 1, 64, DEV)
    slots = torch.arange(x.shape[0], device=DEV)
    cache.append(x, x.flip(0), slots)
    k, v = cache.read(slots, torch.float32)
    assert torch.equal(k.double().cpu(), quantise(x)) and torch.equal(v.double().cpu(), quantise(x.flip(0)))


def test_infinity_and_nan_make_their_block_nan_and_no_other():
    k, v = tokens(6, 2, 128, torch.float16)
    k[0, 0, 5], k[1, 1, 127], k[2, 0, 64], v[3, 1, 31], v[4, 0, 32] = (float("inf"), float("nan"), -float("inf"),
                                                                      float("nan"), float("inf"))
    cache = tw.KVCache4(1, 16, 2, 128, DEV)
    slots = torch.arange(6, device=DEV)
    cache.append(k, v, slots)
    for got, x in zip(cache.read(slots, torch.float32), (k, v)):
        assert same(got.double().cpu(), quantise(x))
    assert int(cache.read(slots)[0].isnan().sum()) == 3 * 32


@pytest.mark.parametrize("D, page", [(64, 16), (128, 32), (256, 16)])
def test_bytes_are_where_the_layout_says(D, page):
    N, H = 2, 3
    g = torch.Generator().manual_seed(5)
    k, v = (quantise(torch.randn(N, H, page, D, generator=g)) for _ in range(2))
    want = page_bytes(k, v)
    cache = tw.KVCache4(N, page, H, D, DEV)
    slots = torch.arange(N * page, device=DEV)
    flat = [x.transpose(1, 2).reshape(N * page, H, D).float().to(DEV) for x in (k, v)]
    cache.pages.copy_(want)
    for got, x in zip(cache.read(slots, torch.float32), flat):
        assert torch.equal(got, x)
    cache.pages.fill_(0xFF)
    cache.append(*flat, slots)
    for got, x in zip(cache.read(slots, torch.float32), flat):
        assert torch.equal(got, x)
    # the writer's scale is the smallest with the block within 7, the oracle's the smallest with every value on
    # the grid: the same wherever a block holds a value above 3.5 scales
    differ = cache.pages.cpu() != want
    assert not differ[:, :, page * D:].any() or float(differ.double().mean()) < 0.05


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D, dim, Hq, Hk", [(128, 128, 8, 1), (64, 32, 28, 4), (256, 128, 4, 2), (128, 20, 3, 1)])
def test_rotation_on_the_way_is_the_rotation_before(D, dim, Hq, Hk, interleaved, dtype):
    """The same bits as `rotary_positions` followed by an append, for queries, keys and values."""
    T, page = 45, 16
    g = torch.Generator(device=DEV).manual_seed(3)
    qkv = torch.randn(T, (Hq + 2 * Hk) * D, generator=g, device=DEV).to(dtype)
    q, k, v = (x.view(T, -1, D) for x in qkv.split((Hq * D, Hk * D, Hk * D), 1))
    layer = tw.RotaryPositions(D, dim, 1000, interleaved=interleaved).to(DEV)
    positions, slots = torch.randint(0, 1000, (T,), device=DEV), torch.randperm(4 * page, device=DEV)[:T]
    slots[[3, 40]] = torch.tensor([-1, 4 * page], device=DEV)          # skipped
    one, two = (tw.KVCache4(4, page, Hk, D, DEV) for _ in range(2))
    one.pages.zero_(), two.pages.zero_()
    before = qkv.clone()
    q_out = torch.empty(T, Hq, D, dtype=dtype, device=DEV)
    one.append(k, v, slots, positions, layer, q, q_out)
    assert torch.equal(qkv, before)
    q1, k1 = torch.empty_like(q_out), torch.empty(T, Hk, D, dtype=dtype, device=DEV)
    layer(positions, q, k, q1, k1)
    two.append(k1, v, slots)
    assert torch.equal(q_out, q1) and torch.equal(one.pages, two.pages)
    one.append(k, v, slots, positions, layer, q)                       # queries in place
    assert torch.equal(q, q1) and torch.equal(k, before[:, Hq * D:(Hq + Hk) * D].view_as(k))
    got = one.read(slots, dtype)[0]
    assert not got[[3, 40]].any()


def test_skipped_and_untouched_places_keep_their_bytes():
    k, v = tokens(5, 2, 128, torch.bfloat16)
    cache = tw.KVCache4(3, 16, 2, 128, DEV)
    cache.pages.copy_(torch.randint(0, 256, cache.pages.shape, device=DEV, dtype=torch.uint8))
    old = cache.pages.clone()
    cache.append(k, v, torch.tensor([-1, 48, -5, 1 << 40, 17], device=DEV))
    changed = (cache.pages != old).any(-1)
    assert not changed[0].any() and not changed[2].any() and changed[1].all()
    # of one token in a page: 64 bytes of keys, 64 of values, 4 + 4 scales
    assert int((cache.pages != old).sum()) <= 2 * 136
    assert torch.equal(cache.read(torch.tensor([17], device=DEV))[0].double().cpu(), quantise(k[4:]))


def test_strides_and_alignment_give_the_same_bytes():
    k, v = tokens(33, 2, 128, torch.bfloat16)
    slots = torch.arange(33, device=DEV)
    layer = tw.RotaryPositions(128, 128, 100).to(DEV)
    pages = []
    for make in (lambda x: x, lambda x: torch.empty(x.numel() + 1, dtype=x.dtype, device=DEV)[1:].view_as(x).copy_(x),
                 lambda x: torch.empty(2, 33, 128, dtype=x.dtype, device=DEV).transpose(0, 1).copy_(x),
                 lambda x: torch.empty(33, 2, 131, dtype=x.dtype, device=DEV)[..., :128].copy_(x)):
        cache = tw.KVCache4(3, 16, 2, 128, DEV)
        cache.pages.zero_()
        cache.append(make(k), make(v), slots, slots, layer)
        pages.append(cache.pages)
        out = [make(torch.zeros_like(x)) for x in (k, v)]
        ops.kv4_read(*out, cache.pages, slots)
        want = cache.read(slots)
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    assert all(torch.equal(p, pages[0]) for p in pages)


def test_offsets_past_32_bits():
    """Slots whose bytes lie beyond 4 GiB."""
    page, H, D = 256, 8, 256
    per = tw.KVCache4.head_bytes(page, D) * H
    num = (9 << 29) // per + 2
    cache = tw.KVCache4(num, page, H, D, DEV)
    assert cache.pages.numel() > 1 << 32
    k, v = tokens(3, H, D, torch.bfloat16)
    slots = torch.tensor([num * page - 1, (num - 1) * page, 0], device=DEV)
    cache.append(k, v, slots)
    for got, x in zip(cache.read(slots), (k, v)):
        assert torch.equal(got.double().cpu(), quantise(x))


def test_direct_and_ctypes_routes_agree(monkeypatch):
    if ops._fast is None:
        pytest.skip("no compiled binding")
    k, v = tokens(9, 2, 64, torch.float16)
    slots = torch.arange(9, device=DEV)
    layer = tw.RotaryPositions(64, 64, 100).to(DEV)
    found = []
    for fast in (ops._fast, None):
        monkeypatch.setattr(ops, "_fast", fast)
        cache = tw.KVCache4(2, 16, 2, 64, DEV)
        cache.pages.zero_()
        q = k.clone()
        cache.append(k, v, slots, slots, layer, q)
        found.append((cache.pages, q, *cache.read(slots)))
    assert all(torch.equal(a, b) for a, b in zip(*found))


def test_no_tokens():
    cache = tw.KVCache4(1, 16, 2, 64, DEV)
    none = torch.empty(0, 2, 64, device=DEV)
    cache.append(none, none, torch.empty(0, dtype=torch.int64, device=DEV))
    assert cache.read(torch.empty(0, dtype=torch.int64, device=DEV))[0].shape == (0, 2, 64)


def test_refusals():
    k, v = tokens(4, 2, 64, torch.bfloat16)
    cache = tw.KVCache4(2, 16, 2, 64, DEV)
    slots, layer = torch.arange(4, device=DEV), tw.RotaryPositions(64, 64, 100).to(DEV)
    for bad, match in (((k, v[:3], slots), "v has shape"), ((k, v.half(), slots), "dtype"), ((k, v, slots.int()), "slots"),
                       ((k, v, slots[:3]), "slots holds 3"), ((k[:, :1], v[:, :1], slots), "pages has shape"),
                       ((k[..., :32], v[..., :32], slots), "head_size 64"),
                       ((k, v, slots, None, layer), "positions"), ((k, v, slots, slots, None, k), "cos_sin"),
                       ((k, v, slots, slots, layer, None, k), "q_out without q")):
        with pytest.raises(RuntimeError, match=match):
            cache.append(*bad)
    with pytest.raises(RuntimeError, match="pages"):
        ops.kv4_append(cache.pages[:, :, ::2], k, v, slots)
    with pytest.raises(NotImplementedError):
        cache.append(k.double(), v.double(), slots)
    for args in ((2, 16, 2, 96), (2, 24, 2, 64), (2, 8, 2, 64)):
        with pytest.raises(ValueError):
            tw.KVCache4(*args, DEV)
