"""Collected weights that are read and written: in place, apart, or side by side in one buffer they give the same bits; what overlaps in any
other way is refused."""
from __future__ import annotations

import pytest
import torch

import w4a16
from test_gpu_kv4_layer import ints
from test_gpu_kv4_weights import F16, Case, gen
from w4a16 import KV4Cache, KV4Pages, kv4_evict, kv4_reserve

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_device_errors():
    yield
    assert w4a16.check_device_errors() == 0


@pytest.mark.parametrize("new", [[1, 3], [400, 350]])
def test_collected_weights(new):
    c = Case([700, 500], new, 8, 2, 64, 64, 16, F16, 90, 5)
    want = c.call(c.before, out=torch.zeros_like(c.before))
    B, KV, n = c.before.shape
    side = torch.zeros((B, KV, 2, n), device="cuda")
    side[:, :, 0] = c.before
    assert torch.equal(c.call(side[:, :, 0], out=side[:, :, 1]), want)
    assert torch.equal(side[:, :, 0].nan_to_num(nan=7.0), c.before.nan_to_num(nan=7.0))
    # contiguous, a float and a sequence on
    flat = torch.zeros(3 * B * KV * n, device="cuda")
    w = flat[:B * KV * n].view(B, KV, n)
    for by in (1, KV * n, B * KV * n - 1):
        for a, b in ((w, flat[by:by + B * KV * n].view(B, KV, n)), (flat[by:by + B * KV * n].view(B, KV, n), w)):
            with pytest.raises(AssertionError, match="share no memory"):
                c.call(a, out=b)
    assert not flat.any()
    for over in (flat.as_strided((B, KV, n), (KV * n, n - 1, 1)), flat.as_strided((B, KV, n), (n, n, 1))):
        with pytest.raises(AssertionError, match="share memory between"):
            c.call(over)


def test_eviction():
    L, R, KV, n = 2, 3, 2, 300

    def world():
        cache = KV4Cache(L, 100, KV, 64, page_size=16, pool=None)
        cache.pool.copy_(torch.randint(0, 255, cache.pool.shape, generator=gen(1), device="cuda", dtype=torch.uint8) & 0x3B)
        pages = KV4Pages.empty(cache, R, 20)
        assert kv4_reserve(pages, ints([0, 1, 2]), ints([300, 120, 211])).all()
        return cache, pages

    w = torch.rand((L, R, KV, n), generator=gen(2), device="cuda")
    kept = []
    for form in range(3):
        cache, pages = world()
        buf = torch.zeros((L, R, KV, 2, n), device="cuda")
        buf[..., 0, :] = w
        a = buf[..., 0, :] if form else w.clone()
        b = (a, buf[..., 1, :], torch.zeros_like(w))[form]
        pages, ok = kv4_evict(cache, pages, a, ints([0, 2, 1]), 100, sinks=3, recent=9, out_weights=b)
        assert ok.all()
        kept.append((b[..., :100].clone(), cache.pool.clone(), pages.block_table.clone()))
    assert all(torch.equal(x, y) for other in kept[1:] for x, y in zip(kept[0], other))
    cache, pages = world()
    before = cache.pool.clone()
    flat = torch.zeros(2 * w.numel(), device="cuda")
    with pytest.raises(AssertionError, match="share no memory"):
        kv4_evict(cache, pages, flat[:w.numel()].view_as(w), ints([0]), 100, out_weights=flat[n:n + w.numel()].view_as(w))
    with pytest.raises(AssertionError, match="share memory between"):
        kv4_evict(cache, pages, flat.as_strided(w.shape, (R * KV * n, KV * n, n - 1, 1)), ints([0]), 100)
    assert torch.equal(cache.pool, before) and not flat.any() and pages.kv_lens.tolist() == [300, 120, 211]
