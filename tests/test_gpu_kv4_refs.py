"""After every eviction the reference counts are what the tables hold: each page as often as it stands in a row, no page beyond what
the lengths need, none lost."""
from __future__ import annotations

import pytest
import torch

import w4a16
from test_gpu_kv4_layer import ints
from w4a16 import KV4Cache, KV4Pages, kv4_evict, kv4_fork, kv4_release, kv4_reserve

pytestmark = pytest.mark.gpu
DEV = "cuda"


def check(pages):
    table = pages.block_table
    held = table[table >= 0].long()
    assert torch.equal(pages.refs.long(), torch.bincount(held, minlength=pages.refs.shape[0]))
    need = (pages.kv_lens + pages.page_size - 1) // pages.page_size
    assert torch.equal((table >= 0).sum(1).int(), need)
    assert torch.equal(table >= 0, torch.arange(table.shape[1], device=DEV) < need[:, None])        # from the front on
    for row, n in zip(table, need.tolist()):
        assert row[:n].unique().numel() == n


@pytest.mark.parametrize("page,layers", [(16, 1), (32, 3), (128, 2)])
@pytest.mark.parametrize("in_place", [False, True])
def test_counts_follow_the_tables(page, layers, in_place):
    g = torch.Generator(device=DEV).manual_seed(page)
    rows, keep, cap = 8, 150, 700
    cache = KV4Cache(layers, 3 * rows * -(-cap // page) // 4 + 3, 2, 64, page_size=page)
    pages = KV4Pages.empty(cache, rows, -(-cap // page))
    weights = torch.rand((layers, rows, 2, cap), generator=g, device=DEV)
    evicted = 0
    for step in range(40):
        lens = pages.kv_lens.tolist()
        grow = [r for r in range(rows) if torch.rand((), generator=g, device=DEV) < 0.6]
        ends = [min(cap, lens[r] + int(torch.randint(1, 200, (), generator=g, device=DEV))) for r in grow]
        if step % 5 == 4 and grow:
            kv4_release(pages, ints(grow[:2]), out=pages)
            if grow[0] != rows - 1 and pages.kv_lens[rows - 1] > 0:
                pages = kv4_fork(cache, pages, ints([rows - 1]), ints([grow[0]]))[0]
        elif grow:
            kv4_reserve(pages, ints(grow), ints(ends))
        check(pages)
        asked = torch.randperm(rows, generator=g, device=DEV)[:1 + step % rows].int()
        before = pages.kv_lens.clone(), pages.block_table.clone()
        pages, ok = kv4_evict(cache, pages, weights, asked, keep, sinks=2, recent=30, out=pages if in_place else None)
        check(pages)
        over = before[0][asked.long()] > keep
        assert ok[~over].all()
        want = before[0].clone()
        want[asked[over & (ok == 1)].long()] = keep
        assert torch.equal(pages.kv_lens, want)
        same = pages.kv_lens == before[0]
        assert torch.equal(pages.block_table[same], before[1][same])
        evicted += int((over & (ok == 1)).sum())
    assert evicted >= 10
    kv4_release(pages, ints(list(range(rows))), out=pages)
    check(pages)
    assert not pages.refs.any() and w4a16.check_device_errors() == 0
