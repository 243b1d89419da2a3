"""Outputs whose rows share memory are refused before anything is launched: their rows are written by several threads.
Host memory stands for the tensors; a call that passes its checks ends with the launch, here without a GPU."""
import ctypes
import random

import pytest

from tokenweave_amd import _lib

BUF = ctypes.create_string_buffer(1 << 12)
AT = (ctypes.addressof(BUF) + 63) & ~63


def heads(n, token, head):
    return ctypes.byref(_lib.Heads(AT, n, token, head))


def overlap(T, H, D, token, head):
    """By every pair of rows."""
    starts = sorted(t * token + h * head for t in range(T) for h in range(H))
    return any(b - a < D for a, b in zip(starts, starts[1:]))


def calls(T, H, D, token, head):
    """(the call, its outputs' description) for each entry point with outputs of rows."""
    L, ok = _lib.lib(), heads(H, H * D, D)
    bad = heads(H, token, head)
    one = heads(1, D, D)
    yield lambda: L.tw_rotary_positions(bad, ok, None, None, AT, AT, 100, T, D, D, 0, 0, None), "q_out"
    yield lambda: L.tw_rotary_positions(one, one, bad, ok, AT, AT, 100, T, D, D, 0, 0, None), "k_out"
    yield lambda: L.tw_kv4_append(AT, 4, 16, ok, ok, AT, bad, ok, AT, AT, 100, T, D, D, 0, 0, None), "q_out"
    yield lambda: L.tw_kv4_read(bad, ok, AT, 4, 16, AT, T, D, 0, None), "k_out"
    yield lambda: L.tw_kv4_read(ok, bad, AT, 4, 16, AT, T, D, 0, None), "v_out"
    yield lambda: L.tw_kv4_attention(bad, ok, AT, 4, 16, 1, AT, 4, 4, AT, None, T, T, 1, D, 0.1, 0, 0, AT, 1 << 40, None), "out"


no_gpu = pytest.mark.skipif(_lib.lib().tw_num_compute_units() > 0, reason="calls that pass their checks would run")


def refused(call):
    rc = call()
    return rc == _lib.TW_ERR_INVALID_ARGUMENT and "share memory" in _lib.last_error()


@no_gpu
@pytest.mark.parametrize("T, H, token, head", [(4, 2, 0, 128), (4, 2, 256, 0), (2, 2, 0, 0), (3, 4, 256, 128), (5, 2, 127, 1000),
                                               (2, 3, 10000, 64), (4, 2, 128, 256), (1, 2, 512, 0), (2, 1, 0, 128)])
def test_rows_that_share_memory_are_refused(T, H, token, head):
    assert overlap(T, H, 128, token, head)
    for call, name in calls(T, H, 128, token, head):
        assert refused(call), name
        assert f" {name} " in _lib.last_error()


@no_gpu
@pytest.mark.parametrize("T, H, token, head", [(4, 2, 256, 128), (1, 2, 0, 128), (4, 1, 128, 0), (1, 1, 0, 0), (4, 2, 128, 512),
                                               (5, 3, 1000, 131), (2, 2, 384, 256), (3, 2, 256, 640)])
def test_rows_apart_are_taken_in_any_order(T, H, token, head):
    assert not overlap(T, H, 128, token, head)
    for call, name in calls(T, H, 128, token, head):
        assert not refused(call), name


@no_gpu
def test_drawn_strides():
    rng = random.Random(5)
    seen = set()
    for _ in range(400):
        T, H, D = rng.randint(1, 7), rng.randint(1, 6), rng.choice((64, 128))
        token, head = (rng.choice((rng.randint(0, 900), D * rng.randint(0, 8))) for _ in range(2))
        want = overlap(T, H, D, token, head)
        seen.add(want)
        for call, name in calls(T, H, D, token, head):
            assert refused(call) == want, (T, H, D, token, head, name)
    assert seen == {True, False}
