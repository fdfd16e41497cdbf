"""Calls of the bounded cache's operators that are refused on the host, without a GPU: sizes and layouts that the kernels cannot
take."""
from __future__ import annotations

import ctypes

import pytest
import torch

from test_kv4_bounded_host import tables
from w4a16 import _lib, kv4_evict


class Cache:
    """What the checks look at, on the CPU."""
    _index, num_pages, page_size, num_layers, num_kv_heads = -1, 4, 16, 1, 2


class Pages:
    _index, page_size = -1, 16

    def __init__(self, rows, width):
        self._shape = (4, rows, width)


def test_an_eviction_asks_for_no_more_pages_than_32_bits_count():
    fn, ints = _lib.lib().w4a16_kv4_evict_scratch_ints, ctypes.c_int64(0)
    wide = tables(width=4096)
    for n, keep, status in ((1 << 19, 65536, -1), ((1 << 19) - 1, 65536, 0), (1 << 20, 65536, -1), (1 << 20, 2047 * 16, 0), (1 << 20, 2048 * 16, -1)):
        assert fn(wide, n, keep, ctypes.byref(ints)) == status, (n, keep)
        assert ints.value == (0 if status else n * (3 + keep // 16 + 4096) + 1 + 2)
    with pytest.raises(AssertionError, match="more than one call"):
        kv4_evict(Cache(), Pages(2, 4096), torch.zeros(1, 2, 2, 8), torch.zeros(1 << 19, dtype=torch.int32), 65536)
