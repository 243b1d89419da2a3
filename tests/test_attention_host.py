"""What needs no GPU of the rotation, the 4-bit cache and attention: frequencies, tables, batches, the
C entry points' refusals."""
import ctypes
import math

import pytest
import torch

import tokenweave_amd as tw
from kv4_reference import GRID, page_bytes, quantise
from tokenweave_amd import _lib

BUF = ctypes.create_string_buffer(4096 + 64)
AT = (ctypes.addressof(BUF) + 63) & ~63   # host memory: never dereferenced by these calls


def heads(n=2, data=AT, token=None, head=128):
    return ctypes.byref(_lib.Heads(data, n, n * 128 if token is None else token, head))


def test_frequencies_without_and_with_scaling():
    inv, factor = tw.rotary_frequencies(128, 500000.0)
    assert factor == 1.0 and inv.dtype == torch.float64 and inv.numel() == 64
    for j in (0, 1, 31, 63):
        assert math.isclose(float(inv[j]), 500000.0 ** (-2 * j / 128), rel_tol=1e-14)
    linear, _ = tw.rotary_frequencies(128, 500000.0, {"type": "linear", "factor": 4.0})
    assert torch.allclose(linear * 4, inv, rtol=1e-15)
    ntk, _ = tw.rotary_frequencies(128, 500000.0, {"type": "ntk", "factor": 4.0})
    assert float(ntk[0]) == 1.0 and math.isclose(float(ntk[-1]) * 4, float(inv[-1]), rel_tol=1e-12)
    bands, _ = tw.rotary_frequencies(128, 500000.0, {"type": "bands", "factor": 8.0, "original_max_position": 8192})
    wave = 2 * math.pi / inv
    assert torch.equal(bands[wave < 8192 / 4], inv[wave < 8192 / 4])
    assert torch.allclose(bands[wave > 8192] * 8, inv[wave > 8192], rtol=1e-15)
    between = (wave > 8192 / 4) & (wave < 8192)
    assert between.any() and (bands[between] < inv[between]).all() and (bands[between] > inv[between] / 8).all()
    yarn, grown = tw.rotary_frequencies(128, 500000.0, {"type": "yarn", "factor": 16.0, "original_max_position": 4096})
    assert math.isclose(grown, 0.1 * math.log(16.0) + 1)
    turns = 4096 * inv / (2 * math.pi)
    assert torch.equal(yarn[turns > 40], inv[turns > 40]) and torch.allclose(yarn[turns < 0.8] * 16, inv[turns < 0.8])
    assert tw.rotary_frequencies(128, 5e5, {"type": "yarn", "factor": 16.0, "original_max_position": 4096,
                                            "attention_factor": 1.5})[1] == 1.5


def test_table_is_the_64_bit_one_rounded():
    layer = tw.RotaryPositions(64, 32, 100000, scaling={"type": "linear", "factor": 2.0})
    assert layer.cos_sin.shape == (100000, 32) and layer.cos_sin.dtype == torch.float32
    for t, j in ((0, 0), (99999, 0), (99999, 15), (54321, 7)):
        angle = t * (10000.0 ** (-2 * j / 32) / 2)
        assert abs(float(layer.cos_sin[t, j]) - math.cos(angle)) < 2.0 ** -24 + 1e-10
        assert abs(float(layer.cos_sin[t, 16 + j]) - math.sin(angle)) < 2.0 ** -24 + 1e-10
    assert "cos_sin" not in layer.state_dict()


def test_host_refusals():
    for kind in ({"type": "other"}, {"type": "linear", "factor": 0.0},
                 {"type": "bands", "factor": 2.0, "original_max_position": 10, "low_freq_factor": 4.0, "high_freq_factor": 4.0}):
        with pytest.raises(ValueError):
            tw.rotary_frequencies(64, scaling=kind)
    for dim in (0, 3, 65):
        with pytest.raises(ValueError):
            tw.RotaryPositions(64, dim)
    with pytest.raises(ValueError):
        tw.RotaryPositions(64, 130)
    for args in ((2, 16, 2, 96), (2, 24, 2, 64), (2, 8, 2, 64), (2, 512, 2, 64)):
        with pytest.raises(ValueError):
            tw.KVCache4(*args, device="cpu")


def test_cpu_tensors_are_refused():
    q, pos = torch.randn(2, 1, 64), torch.arange(2)
    layer = tw.RotaryPositions(64, 64, 10)
    with pytest.raises(RuntimeError, match="GPU only"):
        layer(pos, q)
    cache = tw.KVCache4(1, 16, 1, 64, "cpu")
    with pytest.raises(RuntimeError, match="GPU only"):
        cache.append(q, q, pos)
    with pytest.raises(RuntimeError, match="GPU only"):
        cache.read(pos)
    with pytest.raises(RuntimeError, match="GPU only"):
        cache.attend(q.bfloat16(), torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32))


def test_cache_size():
    assert tw.KVCache4.head_bytes(64, 128) == 64 * (128 * 2 * 4.25 / 8)
    assert tw.KVCache4(3, 32, 2, 256, "cpu").pages.shape == (3, 2, 32 * 272)


def test_batch_split_keeps_every_token_and_its_position():
    starts = torch.tensor([0, 3, 4, 10, 12], dtype=torch.int32)
    lens = torch.tensor([30, 5, 6, 100], dtype=torch.int32)
    batch = tw.CachedBatch(torch.arange(12), torch.zeros(4, 2, dtype=torch.int32), lens, starts, 6)
    for at in range(0, 13):
        first, second = batch.split(at)
        assert first.slots.tolist() + second.slots.tolist() == list(range(12))
        where = []
        for part, base in ((first, 0), (second, at)):
            s, n = part.query_starts.tolist(), part.seq_lens.tolist()
            assert s[0] == 0 and s[-1] == part.slots.numel()
            for i in range(4):
                m = s[i + 1] - s[i]
                where += [(base + s[i] + j, i, n[i] - m + j) for j in range(m)]
        whole = [(int(starts[i]) + j, i, int(lens[i]) - int(starts[i + 1] - starts[i]) + j) for i in range(4)
                 for j in range(int(starts[i + 1] - starts[i]))]
        assert where == whole
    assert batch.split(5) is batch.split(5)
    even = tw.CachedBatch(torch.arange(6), torch.zeros(3, 2, dtype=torch.int32), lens[:3])
    assert even.split(3)[1].query_starts.tolist() == [0, 0, 1, 3]


def test_reference_quantiser_and_layout_agree():
    """The oracle's own two halves: what it rounds to is on the grid, and its bytes name each value once."""
    x = quantise(torch.randn(2, 1, 16, 64, generator=torch.Generator().manual_seed(1)))
    assert torch.equal(quantise(x), x)
    data = page_bytes(x, x.flip(0))
    assert data.shape == (2, 1, 16 * 68)
    assert {0.5, 1.0, 6.0} <= set(GRID.tolist())


def test_rotary_entry_point_checks_before_it_launches():
    L, ok = _lib.lib(), heads()
    base = (AT, AT, 100, 4, 128, 128, 0, 0, None)
    assert L.tw_rotary_positions(None, None, None, None, None, None, 0, 0, 128, 128, 0, 0, None) == _lib.TW_OK
    assert L.tw_rotary_positions(ok, None, None, None, *base) == _lib.TW_ERR_INVALID_ARGUMENT
    assert L.tw_rotary_positions(ok, ok, ok, None, *base) == _lib.TW_ERR_INVALID_ARGUMENT
    assert "both" in _lib.last_error()
    assert L.tw_rotary_positions(heads(3), ok, None, None, *base) == _lib.TW_ERR_INVALID_ARGUMENT
    assert L.tw_rotary_positions(ok, heads(2, None), None, None, *base) == _lib.TW_ERR_INVALID_ARGUMENT
    assert L.tw_rotary_positions(ok, heads(2, AT, -1), None, None, *base) == _lib.TW_ERR_INVALID_ARGUMENT
    for at, value in ((0, None), (1, None), (2, 0), (3, -1), (4, 0), (5, 130), (5, 3), (5, 0), (6, 4)):
        args = list(base)
        args[at] = value
        assert L.tw_rotary_positions(ok, ok, None, None, *args) == _lib.TW_ERR_INVALID_ARGUMENT, at
    assert L.tw_rotary_positions(ok, ok, None, None, *base[:7], 9, None) == _lib.TW_ERR_DTYPE
    assert L.tw_rotary_positions(ok, ok, None, None, AT, AT + 2, *base[2:]) == _lib.TW_ERR_ALIGNMENT


def test_cache_entry_points_check_before_they_launch():
    L, ok, bad = _lib.lib(), heads(), _lib.TW_ERR_INVALID_ARGUMENT
    def append(pages=AT, n=4, page=16, k=ok, v=ok, slots=AT, qo=None, q=None, pos=None, table=None, length=0, T=4, D=128,
               dim=0, flags=0, dtype=0):
        return L.tw_kv4_append(pages, n, page, k, v, slots, qo, q, pos, table, length, T, D, dim, flags, dtype, None)
    assert append(None, 0, 0, None, None, None, T=0) == _lib.TW_OK
    for kw in (dict(pages=None), dict(n=0), dict(page=24), dict(page=8), dict(page=512), dict(k=None), dict(v=heads(3)),
               dict(slots=None), dict(D=96), dict(T=-1), dict(q=ok, qo=ok), dict(q=ok), dict(qo=ok),
               dict(table=AT, length=10, dim=128), dict(table=AT, pos=AT, length=10, dim=129),
               dict(table=AT, pos=AT, length=0, dim=128), dict(table=AT, pos=AT, length=10, dim=128, q=heads(3), qo=ok)):
        assert append(**kw) == bad, kw
    assert append(pages=AT + 8) == _lib.TW_ERR_ALIGNMENT and append(dtype=7) == _lib.TW_ERR_DTYPE
    assert L.tw_kv4_read(ok, ok, None, 4, 16, AT, 4, 128, 0, None) == bad
    assert L.tw_kv4_read(ok, heads(1), AT, 4, 16, AT, 4, 128, 0, None) == bad
    assert L.tw_kv4_read(ok, ok, AT, 4, 16, None, 4, 128, 0, None) == bad
    assert L.tw_kv4_read(ok, ok, AT, 4, 16, AT, 0, 128, 0, None) == _lib.TW_OK


def test_attention_entry_point_checks_before_it_launches():
    L, bad = _lib.lib(), _lib.TW_ERR_INVALID_ARGUMENT
    def attend(out=heads(4), q=heads(4), pages=AT, n=4, page=16, kv=2, table=AT, stride=8, width=8, lens=AT, starts=None,
               B=2, T=2, most=1, D=128, scale=0.1, window=0, dtype=0, ws=AT, ws_bytes=1 << 40):
        return L.tw_kv4_attention(out, q, pages, n, page, kv, table, stride, width, lens, starts, B, T, most, D, scale,
                                  window, dtype, ws, ws_bytes, None)
    assert attend(T=0) == attend(B=0) == attend(most=0) == _lib.TW_OK
    for kw in (dict(out=None), dict(q=None), dict(q=heads(3)), dict(out=heads(2)), dict(kv=0), dict(kv=3), dict(page=20),
               dict(D=80), dict(table=None), dict(lens=None), dict(T=3), dict(T=-1), dict(window=-1), dict(B=-1),
               dict(width=-1), dict(width=1 << 40), dict(q=heads(4, AT, -2)), dict(pages=None)):
        assert attend(**kw) == bad, kw
    assert attend(dtype=_lib.TW_DTYPE_F32) == _lib.TW_ERR_DTYPE and attend(pages=AT + 4) == _lib.TW_ERR_ALIGNMENT
    need = L.tw_kv4_attention_workspace(4, 2, 128, 2, 2, 1, 8, 16)
    assert need >= 0
    if need:
        assert attend(ws=None) == bad and attend(ws_bytes=need - 1) == bad and attend(ws=AT + 4) == bad
