"""Bounded waits of the paged attention's tensor-core kernel: with the wait limit
at 0 every pipeline wait gives up, the call records ALTXS_ST_TIMEOUT, drains its
copies and products and returns; the next call, with the limit restored, is
right again."""

from __future__ import annotations

import pytest
import torch

from altxs_b200 import _lib, paged

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_waits_give_up_report_and_recover(dtype):
    L = _lib.lib()
    g = torch.Generator(device=DEV)
    g.manual_seed(1)
    cache = paged.PagedKV.empty(40, 16, 2, 64, dtype)
    cache.k.copy_(torch.randn(cache.k.shape, generator=g, device=DEV))
    cache.v.copy_(torch.randn(cache.v.shape, generator=g, device=DEV))
    alloc = paged.PageAllocator(2, 40, 16, 300, DEV)
    alloc.extend([100, 200])
    chunks = alloc.extend([40, 90])
    q = torch.randn(130, 4, 64, generator=g, device=DEV).to(dtype)
    want = cache.attend(chunks, q)
    cache.check_status()
    try:
        assert L.altxs_set_wait_limit(0) == 0
        cache.attend(chunks, q)
        torch.cuda.synchronize()
    finally:
        assert L.altxs_set_wait_limit(L.altxs_default_wait_limit()) == 0
    with pytest.raises(RuntimeError, match="status 0x10"):
        cache.check_status()
    for _ in range(2):
        assert torch.equal(cache.attend(chunks, q), want)
    cache.check_status()


def test_a_spoilt_workspace_is_reported_by_every_cache_that_shares_it():
    """A call that gave up may leave counters counting: until they are zeroed, calls of other caches in the same
    workspace report it too."""
    L = _lib.lib()
    g = torch.Generator(device=DEV)
    g.manual_seed(2)
    caches = [paged.PagedKV.empty(150, 16, 2, 64, torch.bfloat16) for _ in range(2)]
    for c in caches:
        c.k.copy_(torch.randn(c.k.shape, generator=g, device=DEV))
        c.v.copy_(torch.randn(c.v.shape, generator=g, device=DEV))
    alloc = paged.PageAllocator(1, 150, 16, 2400, DEV)
    alloc.extend([2300])
    chunks = alloc.extend([40])
    q = torch.randn(40, 4, 64, generator=g, device=DEV).bfloat16()
    want = [c.attend(chunks, q) for c in caches]
    assert [*caches[0]._ws.values()][0] is [*caches[1]._ws.values()][0]
    for c in caches:
        c.check_status()
    try:
        assert L.altxs_set_wait_limit(0) == 0
        caches[0].attend(chunks, q)
        torch.cuda.synchronize()
    finally:
        assert L.altxs_set_wait_limit(L.altxs_default_wait_limit()) == 0
    caches[1].attend(chunks, q)
    for c in caches:
        with pytest.raises(RuntimeError, match="status 0x10"):
            c.check_status()
    for _ in range(2):
        for c, w in zip(caches, want):
            assert torch.equal(c.attend(chunks, q), w)
    for c in caches:
        c.check_status()
