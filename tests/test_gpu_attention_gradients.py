"""The operators between the projections record no gradient: what would want one is refused."""
import pytest
import torch

import tokenweave_amd as tw
from tokenweave_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("direct", [True, False])
def test_tensors_that_want_gradients_are_refused(direct, monkeypatch):
    if not direct:
        monkeypatch.setattr(ops, "_fast", None)
    q, k, v = (torch.randn(3, 2, 64, device=DEV).bfloat16() for _ in range(3))
    leaf = q.clone().requires_grad_()
    grown = leaf * 2
    positions = torch.arange(3, device=DEV)
    rotary, cache = tw.RotaryPositions(64, 64, 10).to(DEV), tw.KVCache4(1, 16, 2, 64, DEV)
    cache.append(k, v, positions)
    table, lens = torch.zeros(3, 1, dtype=torch.int32, device=DEV), torch.ones(3, dtype=torch.int32, device=DEV)
    out = torch.full_like(q, 5.0)
    before, pages = grown.detach().clone(), cache.pages.clone()
    for call in (lambda x: rotary(positions, x), lambda x: rotary(positions, q, x, out, out.clone()),
                 lambda x: rotary(positions, q, None, x), lambda x: cache.append(x, v, positions),
                 lambda x: cache.append(k, x, positions), lambda x: cache.append(k, v, positions, positions, rotary, x, out),
                 lambda x: ops.kv4_read(x, out, cache.pages, positions), lambda x: cache.attend(x, table, lens, out=out),
                 lambda x: cache.attend(q, table, lens, out=x)):
        for x in (leaf, grown):
            with pytest.raises(RuntimeError, match="gradient"):
                call(x)
    assert torch.equal(grown, before) and torch.equal(cache.pages, pages) and bool((out == 5).all())
    # without gradients recorded they are data like any other
    with torch.no_grad():
        want = cache.attend(q, table, lens)
        assert torch.equal(cache.attend(leaf, table, lens), want)
        rotary(positions, leaf)
    rotary(positions, q)
    assert torch.equal(leaf.detach(), q)
