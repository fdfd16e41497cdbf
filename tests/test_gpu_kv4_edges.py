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
