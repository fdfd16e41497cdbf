"""Calls of the bounded cache's operators that are refused on the host, without a GPU: sizes and layouts that the kernels cannot
take."""
from __future__ import annotations

import ctypes

import pytest
import torch

from test_kv4_bounded_host import cache, tables
from w4a16 import _lib, kv4_evict, kv_cache


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


# Layouts of what is read and what is written, each a view of one buffer of floats, [1, 2, 2, 8] as [layers, rows, heads, tokens]: strides,
# and where they begin. The first ones are fine.
LAYOUTS = [
    (True, (32, 16, 8), 0, (32, 16, 8), 0),          # in place
    (True, (32, 16, 8), 0, (32, 16, 8), 32),         # one behind the other
    (True, (32, 16, 8), 32, (32, 16, 8), 0),
    (True, (64, 32, 16), 0, (64, 32, 16), 8),        # side by side, each with its neighbour between
    (True, (64, 32, 16), 8, (64, 32, 16), 0),
    (True, (64, 32, 8), 0, (64, 32, 8), 16),
    (True, (64, 8, 32), 0, (64, 8, 32), 16),         # heads before rows
    (True, (0, 0, 0), 0, (32, 16, 8), 8),            # one entry for all, read
    (True, (5, 16, 8), 0, (999, 16, 8), 0),          # (there is one layer)
    (False, (32, 16, 8), 0, (32, 16, 8), 1),         # a token on
    (False, (32, 16, 8), 8, (32, 16, 8), 0),         # a head on
    (False, (32, 16, 8), 0, (32, 16, 8), 31),
    (False, (64, 32, 16), 0, (64, 32, 16), 15),
    (True, (64, 32, 16), 0, (64, 32, 16), 40),       # a row and a head on, between
    (False, (64, 32, 16), 0, (64, 32, 16), 48),
    (False, (64, 32, 8), 0, (64, 32, 8), 15),
    (False, (64, 16, 8), 0, (64, 8, 16), 0),         # in place, rows for heads
    (False, (64, 16, 8), 0, (64, 32, 8), 8),         # other strides, the same memory
    (False, (0, 0, 0), 0, (32, 16, 8), 0),
    (False, (32, 16, 8), 100, (32, 16, 7), 0),       # written entries that share memory
    (False, (32, 16, 8), 100, (32, 15, 8), 0),
    (False, (32, 16, 8), 100, (32, 8, 8), 0),
    (False, (32, 16, 8), 100, (32, 0, 8), 0),
]


@pytest.mark.parametrize("good,read,read_at,written,written_at", LAYOUTS)
def test_weights_are_written_in_place_or_apart(good, read, read_at, written, written_at):
    """Blocks read and write in no order of each other but in place, so any other overlap would be a race."""
    # which floats each entry takes, to be sure of the table itself
    def floats(strides, at):
        r, h, t = torch.meshgrid(torch.arange(2), torch.arange(2), torch.arange(8), indexing="ij")
        return (at + r * strides[1] + h * strides[2] + t).flatten()

    a, b = floats(read, read_at), floats(written, written_at)
    assert good == (len(set(b.tolist())) == 32 and (torch.equal(a, b) or not set(a.tolist()) & set(b.tolist())))
    buf = torch.zeros(4096)
    w, out = (buf.as_strided((1, 2, 2, 8), (*strides, 1), at) for strides, at in ((read, read_at), (written, written_at)))
    if good:
        kv_cache._check_written(out, w)
    else:
        with pytest.raises(AssertionError, match="share"):
            kv_cache._check_written(out, w)
    # the same over the C entry points: what is fine comes as far as the device, which there is none of here
    lib, at = _lib.lib(), buf.data_ptr()
    if good and torch.cuda.is_available():
        return
    want = lib.w4a16_kv4_copy_pages(cache(), 256, 256, 0, None) if good else -1
    assert not good or want not in (0, -1)
    assert lib.w4a16_kv4_evict(cache(), tables(), tables(), at + 4 * read_at, *read, at + 4 * written_at, *written, 8, 256, 1, 33, 0, 0, 256, 256,
                               None) == want
    assert lib.w4a16_kv4_attention_weights(256, 0, 2, 8, 1024, 128, cache(), 0, 256, 1, 256, None, 2, 1, 1.0, 0, 0, 256, at + 4 * read_at, *read[1:],
                                           at + 4 * written_at, *written[1:], 8, 256, 1 << 20, None) == want


def test_weights_of_no_tokens_share_nothing():
    w = torch.zeros(2, 2, 0)
    kv_cache._check_written(w, w)
    kv_cache._check_written(torch.zeros(0, 2, 5).expand(0, 2, 5), torch.zeros(0, 2, 5))


def test_a_call_whose_result_overlaps_what_it_reads_is_refused():
    """The eviction's own checks come as far as that without a device."""
    buf = torch.zeros(1, 2, 2, 40)
    for kw in (dict(out_weights=buf[..., 1:33]), dict(out_weights=buf.transpose(1, 2)[..., :32])):
        with pytest.raises(AssertionError, match="share"):
            kv4_evict(Cache(), Pages(2, 4), buf[..., :32], torch.zeros(1, dtype=torch.int32), 5, **kw)


def test_capacities_below_zero_are_refused():
    lib = _lib.lib()
    for strides, apart in (((0, 0, 0), 256), ((400, 400, 0), 256), ((400, 0, 0), 0), ((1, 1, 1), 4)):
        assert lib.w4a16_kv4_evict(cache(layers=2), tables(), tables(), 4096, *strides, 4096 + apart, *strides, -5, 256, 1, 33, 0, 0, 256, 256, None) != 0
        assert lib.w4a16_kv4_attention_weights(256, 0, 2, 8, 1024, 128, cache(), 0, 256, 1, 256, None, 2, 1, 1.0, 0, 0, 256, 4096, *strides[1:],
                                               4096 + apart, *strides[1:], -5, 256, 1 << 20, None) != 0
