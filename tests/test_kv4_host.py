"""The 4-bit cache's host side, without a GPU: refusals, sizes and the C entry points' argument checks."""
from __future__ import annotations

import ctypes

import pytest
import torch

import w4a16
from w4a16 import KV4Cache, KV4Pages, _lib, kv4_attention, qk_norm_rope


@pytest.mark.parametrize("kw", [
    dict(head_dim=96), dict(page_size=24), dict(page_size=0), dict(page_size=8192), dict(group_size=32), dict(num_pages=0),
    dict(num_layers=0), dict(num_kv_heads=0), dict(group_size=96),
])
def test_cache_refuses_what_the_format_has_not(kw):
    with pytest.raises(ValueError):
        KV4Cache(**{**dict(num_layers=1, num_pages=4, num_kv_heads=2, head_dim=128), **kw})


def test_cpu_tensors_are_refused():
    with pytest.raises(AssertionError):
        KV4Cache(1, 4, 2, 128, pool=torch.zeros(1, 4, 2, 64 * 136, dtype=torch.uint8))
    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(AssertionError):
        KV4Pages(i, i.view(4, 1), i, 16)
    x = torch.zeros(1, 2, 128, dtype=torch.float16)
    with pytest.raises(AssertionError):
        qk_norm_rope(x, x, torch.zeros(1, dtype=torch.int64), torch.zeros(2, 128))


@pytest.mark.parametrize("D,page,group,want", [(128, 64, 128, 8704), (128, 16, 64, 2304), (64, 32, 64, 2304),
                                               (64, 16, 64, 1152)])
def test_page_bytes(D, page, group, want):
    out = ctypes.c_int64(0)
    assert _lib.lib().w4a16_kv4_page_bytes(D, page, group, ctypes.byref(out)) == 0 and out.value == want
    assert KV4Cache.bytes_per_page(D, page, group) == want
    for bad in ((96, page, 64), (D, page + 8, group), (D, page, 32), (D, 0, group)):
        assert _lib.lib().w4a16_kv4_page_bytes(*bad, ctypes.byref(out)) == -1


def test_entry_points_check_their_arguments_before_the_device():
    lib = _lib.lib()
    good = dict(pool=256, layers=1, pages=4, kv_heads=2, head_dim=128, page_size=64, group_size=128)
    for bad, status in ((dict(head_dim=96), -1), (dict(page_size=20), -1), (dict(group_size=16), -1), (dict(pages=0), -1),
                        (dict(pages=1 << 32), -1), (dict(pool=0), -1), (dict(pool=8), -2), (dict(kv_heads=0), -1)):
        c = _lib.KV4CacheStruct(**{**good, **bad})
        assert lib.w4a16_kv4_gather(ctypes.byref(c), 0, 256, 1, 256, 0, None) == status
        assert lib.w4a16_kv4_copy_pages(ctypes.byref(c), 256, 256, 1, None) == status
        assert lib.w4a16_kv4_attention(256, 0, 1, 8, 1024, 128, ctypes.byref(c), 0, 256, 1, 256, None, 1, 1, 1.0, 0, 256,
                                       None, None, 0, None) == status
    tables = dict(refs=256, block_table=256, kv_lens=256, pages=4, rows=2, width=3, page_size=16)
    for bad in (dict(refs=0), dict(rows=0), dict(width=0), dict(page_size=8), dict(width=1 << 28)):
        t = _lib.KV4TablesStruct(**{**tables, **bad})
        assert lib.w4a16_kv4_reserve(ctypes.byref(t), 256, 256, 1, 256, 256, None) == -1
        assert lib.w4a16_kv4_release(ctypes.byref(t), ctypes.byref(t), 256, 1, None) == -1


def test_names_are_public():
    for name in ("KV4Cache", "KV4Pages", "qk_norm_rope", "qk_norm_rope_append", "kv4_gather", "kv4_attention",
                 "kv4_reserve", "kv4_copy_pages", "kv4_fork", "kv4_release", "kv4_compact"):
        assert name in w4a16.__all__ and hasattr(w4a16, name)
    assert "out of range" in _lib.strerror(-8)
    assert kv4_attention.__doc__ and KV4Cache.__doc__
