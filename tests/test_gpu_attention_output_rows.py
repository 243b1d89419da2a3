"""Expanded outputs, whose rows share memory, are refused by the ops; outputs in any order of strides are not."""
import pytest
import torch

import tokenweave_amd as tw
from tokenweave_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("direct", [True, False])
def test_expanded_outputs_are_refused(direct, monkeypatch):
    if not direct:
        monkeypatch.setattr(ops, "_fast", None)
    T, H, D = 3, 2, 64
    q, k, v = (torch.randn(T, H, D, device=DEV).bfloat16() for _ in range(3))
    pos = torch.arange(T, device=DEV)
    rotary, cache = tw.RotaryPositions(D, D, 10).to(DEV), tw.KVCache4(1, 16, H, D, DEV)
    cache.append(k, v, pos)
    table, lens = torch.zeros(T, 1, dtype=torch.int32, device=DEV), torch.ones(T, dtype=torch.int32, device=DEV)
    for bad in (torch.zeros(1, H, D, device=DEV).bfloat16().expand(T, H, D), torch.zeros(T, 1, D, device=DEV).bfloat16().expand(T, H, D),
                torch.zeros(2 * T * D, device=DEV).bfloat16().as_strided((T, H, D), (D, D, 1))):
        for call in (lambda: rotary(pos, bad), lambda: rotary(pos, q, k, q.clone(), bad),
                     lambda: cache.append(k, v, pos, pos, rotary, q, bad), lambda: ops.kv4_read(q.clone(), bad, cache.pages, pos),
                     lambda: cache.attend(q, table, lens, out=bad)):
            with pytest.raises(RuntimeError, match="share memory"):
                call()
        assert not bad.any()
        cache.append(bad, bad, pos)      # inputs may be expanded
    by_head = torch.empty(H, T, D, dtype=q.dtype, device=DEV).transpose(0, 1)
    one = torch.empty(T, D, 1, dtype=q.dtype, device=DEV).transpose(1, 2)
    cache.append(k, v, pos)
    cache.attend(q, table, lens, out=by_head)
    assert torch.equal(by_head, cache.attend(q, table, lens))
    rotary(pos, q[:, :1], None, one)
    rotary(pos, q, None, by_head)
    assert torch.equal(one, by_head[:, :1])
