"""Pages of rows whose length was lowered (rejected drafts): none is lost, none is given away."""
from __future__ import annotations

import random

import pytest
import torch

import w4a16
from w4a16 import KV4Cache, KV4Pages, kv4_compact, kv4_fork, kv4_release, kv4_reserve

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.fixture(autouse=True)
def _no_device_errors():
    yield
    assert w4a16.check_device_errors() == 0


def test_a_lowered_row_grows_into_its_own_pages():
    cache = KV4Cache(1, 12, 1, 64, page_size=16)
    pages = KV4Pages.empty(cache, 3, 8)
    assert kv4_reserve(pages, ints([0, 1]), ints([100, 20])).tolist() == [1, 1]       # 7 and 2 pages
    row = pages.block_table[0].tolist()
    pages.kv_lens[0] = 33                                                            # 3 pages' worth
    assert kv4_reserve(pages, ints([0]), ints([90])).tolist() == [1]
    assert pages.block_table[0].tolist() == row and pages.refs.tolist() == [1] * 9 + [0] * 3
    pages.kv_lens[0] = 0
    assert kv4_reserve(pages, ints([2, 0]), ints([17, 128])).tolist() == [1, 1]       # 2 free ones, 7 of its own and one
    assert pages.block_table[0].tolist() == row[:7] + [11] and pages.block_table[2, :2].tolist() == [9, 10]
    assert kv4_reserve(pages, ints([1]), ints([33])).tolist() == [0]                  # none is left
    out = kv4_release(pages, ints([0, 1, 2]))
    assert (out.refs == 0).all() and (out.block_table == -1).all()


def test_no_page_is_lost_or_shared_by_mistake():
    r = random.Random(5)
    page, rows, width, n = 16, 10, 12, 70
    cache = KV4Cache(1, n, 1, 64, page_size=page)
    pages = KV4Pages.empty(cache, rows, width)
    low = [0] * rows                                  # what a row may be lowered to: what it shares
    for step in range(120):
        op = r.choice(["grow", "grow", "lower", "lower", "release", "fork", "compact"])
        lens = pages.kv_lens.tolist()
        if op == "grow":
            who = r.sample(range(rows), r.randint(1, rows))
            kv4_reserve(pages, ints(who), ints([lens[i] + r.randint(0, 60) for i in who]))
        elif op == "lower":
            i = r.randrange(rows)
            pages.kv_lens[i] = r.randint(min(low[i], lens[i]), lens[i])
        elif op == "release":
            who = r.sample(range(rows), 2)
            pages = kv4_release(pages, ints(who))
            for i in who:
                low[i] = 0
        elif op == "fork":
            table = pages.block_table.tolist()
            kids = [i for i in range(rows) if table[i][0] < 0]
            olds = [i for i in range(rows) if lens[i] > 0]
            if kids and olds:
                a, c = r.choice(olds), r.choice(kids)
                pages, ok = kv4_fork(cache, pages, ints([a]), ints([c]))
                if ok.item():
                    low[a] = max(low[a], lens[a] // page * page)
                    low[c] = lens[a] // page * page
        else:
            pages = kv4_compact(cache, pages)
        table, lens = pages.block_table.tolist(), pages.kv_lens.tolist()
        count = [0] * n
        for i, row in enumerate(table):
            held = [p for p in row if p >= 0]
            assert row == held + [-1] * (width - len(held)) and len(held) * page >= lens[i]
            for p in held:
                count[p] += 1
        assert pages.refs.tolist() == count
        for i in range(rows):                          # the page that a row writes next is its own
            at = lens[i] // page
            if lens[i] % page and lens[i] >= low[i]:
                assert count[table[i][at]] == 1
