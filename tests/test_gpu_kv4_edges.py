"""kv4_attention at the ends of its arguments' ranges."""
from __future__ import annotations

import pytest
import torch

import w4a16
from kv4_plain import PlainCache
from w4a16 import KV4Cache, kv4_attention

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


@pytest.fixture(autouse=True)
def _no_device_errors():
    yield
    assert w4a16.check_device_errors() == 0


def case(lens, new, H, KV, D, group, dtype, seed=0):
    g = gen(seed)
    c = PlainCache(lens, KV, D, group, 32, gen=g)
    cache = KV4Cache(1, c.num_pages, KV, D, page_size=32, group_size=group, pool=c.pool)
    q = torch.randn((sum(new), H, D), generator=g, device="cuda").to(dtype)
    cu = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
    return c, cache, q, dict(cu_q=cu, max_q=max(new), return_lse=True)


@pytest.mark.parametrize("lens,new,H,KV,D,group", [
    ([4, 200, 0], [9, 1, 3], 8, 2, 128, 128), ([50, 17], [70, 8], 6, 2, 64, 64), ([40, 300, 0], [130, 129, 70], 64, 8, 128, 64),
])
def test_windows_past_every_length_are_none(lens, new, H, KV, D, group):
    c, cache, q, kw = case(lens, new, H, KV, D, group, F16)
    want, want_lse = kv4_attention(q, cache, 0, c.table, c.kv_lens, **kw)
    for window in (max(lens), 2 ** 31 - 200, 2 ** 31 - 1, 2 ** 31, 2 ** 32, 2 ** 32 + 5, 2 ** 63):
        o, lse = kv4_attention(q, cache, 0, c.table, c.kv_lens, window=window, **kw)
        assert torch.equal(o, want) and torch.equal(lse, want_lse), window


@pytest.mark.parametrize("before,after", [(0, 5), (3, 0), (7, 200)])
@pytest.mark.parametrize("lens,new,H,KV,D,group", [
    ([100, 30], [1, 1], 8, 2, 128, 128), ([60, 70, 0], [5, 0, 2], 6, 2, 64, 64), ([300, 290], [130, 129], 64, 8, 128, 64),
])
def test_queries_of_no_sequence_give_zeros(before, after, lens, new, H, KV, D, group):
    c, cache, q, kw = case(lens, new, H, KV, D, group, BF16)
    want, want_lse = kv4_attention(q, cache, 0, c.table, c.kv_lens, **kw)
    T = before + q.shape[0] + after
    wide = torch.full((T, H, D), 7.0, device="cuda", dtype=BF16)
    wide[before:before + q.shape[0]] = q
    out = torch.full_like(wide, float("nan"))
    kw["cu_q"] = kw["cu_q"] + before
    o, lse = kv4_attention(wide, cache, 0, c.table, c.kv_lens, out=out, **kw)
    assert o is out
    rows = slice(before, before + q.shape[0])
    assert torch.equal(o[rows], want) and torch.equal(lse[rows], want_lse)
    none = torch.ones(T, dtype=torch.bool, device="cuda")
    none[rows] = False
    assert (o[none] == 0).all() and (lse[none] == -float("inf")).all()


def test_more_sequences_than_one_launch_takes():
    """5000 sequences in three launches, uniform and ragged, with queries before and after them."""
    n, KV, D = 5000, 2, 64
    g = gen(8)
    lens = [i * 7 % 19 for i in range(n)]
    pages = KV4Cache(1, 40, KV, D, page_size=16, pool=torch.randint(
        0, 40, (1, 40, KV, KV4Cache.bytes_per_page(D, 16, D)), generator=g, device="cuda", dtype=torch.uint8))
    table = torch.randint(0, 40, (n, 2), generator=g, device="cuda").int()
    kv_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = torch.randn((2 * n, 4, D), generator=g, device="cuda").half()
    o, lse = kv4_attention(q, pages, 0, table, kv_lens, return_lse=True)
    for lo in range(0, n, 1250):                                       # 1250 at a time: one launch each
        s = slice(lo, lo + 1250)
        part, part_lse = kv4_attention(q[2 * lo:2 * lo + 2500], pages, 0, table[s], kv_lens[s], return_lse=True)
        assert torch.equal(o[2 * lo:2 * lo + 2500], part) and torch.equal(lse[2 * lo:2 * lo + 2500], part_lse), lo
    new = torch.tensor([1 + i % 3 for i in range(n)], device="cuda")
    cu = torch.cat([torch.full((1,), 11, device="cuda"), 11 + new.cumsum(0)]).int()
    total = int(cu[-1])
    q = torch.randn((total + 9, 4, D), generator=g, device="cuda").half()
    o, lse = kv4_attention(q, pages, 0, table, kv_lens, cu_q=cu, max_q=3, return_lse=True,
                           out=torch.full_like(q, float("nan")))
    assert (o[:11] == 0).all() and (o[total:] == 0).all() and (lse[:11] == -float("inf")).all()
    for lo in range(0, n, 1250):
        a, b = int(cu[lo]), int(cu[lo + 1250])
        part, part_lse = kv4_attention(q[a:b], pages, 0, table[lo:lo + 1250], kv_lens[lo:lo + 1250],
                                       cu_q=cu[lo:lo + 1251] - a, max_q=3, return_lse=True)
        assert torch.equal(o[a:b], part) and torch.equal(lse[a:b], part_lse), lo


def test_ragged_calls_leave_nothing_behind():
    """The workspace does not depend on a call's sizes, and nothing is kept for each of them."""
    c, cache, q, _ = case([70, 40, 9, 30], [40, 40, 9, 30], 8, 2, 64, 64, F16)

    def kept():
        return sum(len(v) for v in vars(cache).values() if isinstance(v, dict))

    def call(new):
        cu = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
        kv4_attention(q[:sum(new)], cache, 0, c.table, c.kv_lens, cu_q=cu, max_q=max(new))

    call([1, 1, 1, 1])
    before, memory = kept(), None
    for i in range(1, 40):
        call([i, 1 + i % 7, 1, 1 + i % 3])
        torch.cuda.synchronize()
        memory = torch.cuda.memory_allocated() if memory is None else memory
        assert torch.cuda.memory_allocated() <= memory + 1024
    assert kept() == before


def test_a_larger_cache_on_the_same_stream():
    """The stream's workspace is replaced by a larger one between two calls of the smaller cache."""
    small, large = case([20000, 100], [1, 1], 8, 2, 64, 64, F16, 1), case([30000] + [200] * 79, [1] * 80, 32, 2, 128, 64, F16, 2)
    want = [kv4_attention(q, cache, 0, c.table, c.kv_lens, **kw) for c, cache, q, kw in (small, large)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for i in (0, 1, 0, 1):
            c, cache, q, kw = (small, large)[i]
            o, lse = kv4_attention(q, cache, 0, c.table, c.kv_lens, **kw)
            side.synchronize()
            assert torch.equal(o, want[i][0]) and torch.equal(lse, want[i][1])
