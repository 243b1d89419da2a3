"""Whatever the arrays on the device hold, a call touches the tokens of its tensors only, and the sequences that are in
order get their results."""
import pytest
import torch

from test_gpu_kv4_attention import DEV, Case
from tokenweave_amd import ops

pytestmark = pytest.mark.gpu
LOW, HIGH = -2 ** 31, 2 ** 31 - 1


@pytest.mark.parametrize("window", [0, 5])
@pytest.mark.parametrize("most", [4, 70])     # few rows and many
@pytest.mark.parametrize("starts, whole", [
    ([0, 20, LOW], [0]), ([0, 20, 40, LOW, 50], []), ([0, 20, HIGH], [0]), ([LOW, 20, 40], [1]), ([30, LOW, HIGH], []),
    ([50, 40, 30, 10], []), ([HIGH, LOW, HIGH], []), ([-5, LOW + 1, -7], [])])
def test_starts_outside_the_tokens(starts, whole, most, window):
    n, T, H, D, guard = len(starts) - 1, 60, 4, 128, 40
    c = Case([90] * n, [20] * n, H, 2, D, 16)
    q = torch.randn(T, H, D, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).bfloat16()
    wide = torch.full((T + 2 * guard, H, D), 7.0, dtype=q.dtype, device=DEV)
    out = wide[guard:guard + T]
    ops.kv4_attention(out, q, c.cache.pages, c.table, c.seq_lens, D ** -0.5, torch.tensor(starts, dtype=torch.int32, device=DEV),
                      most, window)
    torch.cuda.synchronize()
    assert bool((wide[:guard] == 7).all()) and bool((wide[guard + T:] == 7).all())
    for i in whole:
        rows = slice(starts[i], starts[i] + min(most, starts[i + 1] - starts[i]))
        want = ops_result(c, i, q[starts[i]:starts[i + 1]], most, window)
        torch.testing.assert_close(out[rows], want[:rows.stop - rows.start], rtol=2.0 ** -7, atol=2.0 ** -9)


def ops_result(c, i, q, most, window):
    """The sequence by itself."""
    return c.cache.attend(q, c.table[i:i + 1], c.seq_lens[i:i + 1], None,
                          torch.tensor([0, len(q)], dtype=torch.int32, device=DEV), most, window)


@pytest.mark.parametrize("most", [1, 40])
def test_lengths_outside_the_table(most):
    """A length below zero is no tokens, one past the table's places is all of them."""
    c = Case([64, 64], [1, 1], 4, 1, 128, 16)
    want = c.cache.attend(c.q, c.table, c.seq_lens, None, c.starts, most)
    c.seq_lens.copy_(torch.tensor([LOW, HIGH], dtype=torch.int32))
    got = c.cache.attend(c.q, c.table, c.seq_lens, None, c.starts, most)
    assert not got[0].any()
    torch.testing.assert_close(got[1], want[1], rtol=2.0 ** -7, atol=2.0 ** -9)
