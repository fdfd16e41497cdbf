"""The attention path between the W4A16 layers: a paged key/value cache held in 4 bits, the
preparation of queries and keys, attention over the cache, and the management of its pages.

No reference counterpart (the reference ends at the linear layers). Everything runs in the sm_100a
library on torch's current stream, allocates nothing on the host's way but its outputs, and never
synchronises: lengths, tables and reference counts live on the device.

A cached value is ``offset + scale * code`` with a 4-bit code and one fp16 (scale, offset) pair per
token, kv head and group of ``group_size`` channels (``include/w4a16_b200.h`` has the byte layout).
An index the device finds out of range (a position, slot, page or row) is skipped and raises
:class:`W4A16Error` from :func:`w4a16.check_device_errors`.
"""
from __future__ import annotations

import ctypes

import torch
from torch import Tensor

from . import _lib

__all__ = ["KV4Cache", "KV4Pages", "qk_norm_rope", "qk_norm_rope_append", "kv4_gather", "kv4_attention",
           "kv4_attention_weights", "kv4_reserve", "kv4_copy_pages", "kv4_fork", "kv4_release", "kv4_compact", "kv4_evict"]

_I32, _I64, _F32 = torch.int32, torch.int64, torch.float32
_CODES = {torch.float16: _lib.DTYPE_CODES[torch.float16], torch.bfloat16: _lib.DTYPE_CODES[torch.bfloat16]}
_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _lib.stream_of_index)
_CONTIGUOUS = torch.contiguous_format
_INT_MAX = 2 ** 31 - 1
_largest_workspace: dict[tuple[int, int, int], int] = {}


class KV4Cache:
    """The 4-bit pages of a model's keys and values, all layers in one buffer.

    Args:
        num_layers, num_pages: pages per layer; a page id means the same page of every layer.
        num_kv_heads: key/value heads (a rank's own, under tensor parallelism).
        head_dim: 64 or 128.
        page_size: tokens per page, a multiple of 16 (default 64).
        group_size: channels that share a scale and offset: 64, or ``head_dim`` (the default).
        device: a CUDA device (default: the current one).
        pool: optional uint8 ``[num_layers, num_pages, num_kv_heads, page_bytes]`` to use instead of a
            new (zeroed) buffer, e.g. pages received from another process.
    """

    def __init__(self, num_layers: int, num_pages: int, num_kv_heads: int, head_dim: int, *, page_size: int = 64,
                 group_size: int | None = None, device: torch.device | str | int | None = None,
                 pool: Tensor | None = None) -> None:
        group_size = head_dim if group_size is None else group_size
        if head_dim not in (64, 128):
            raise ValueError(f"head_dim={head_dim} must be 64 or 128")
        if page_size < 16 or page_size % 16 != 0 or page_size > 4096:
            raise ValueError(f"page_size={page_size} must be a multiple of 16, at most 4096")
        if group_size not in (64, head_dim):
            raise ValueError(f"group_size={group_size} must be 64 or head_dim={head_dim}")
        if min(num_layers, num_pages, num_kv_heads) < 1:
            raise ValueError("num_layers, num_pages and num_kv_heads must be positive")
        self.num_layers, self.num_pages, self.num_kv_heads = num_layers, num_pages, num_kv_heads
        self.head_dim, self.page_size, self.group_size = head_dim, page_size, group_size
        self.page_bytes = self.bytes_per_page(head_dim, page_size, group_size)
        shape = (num_layers, num_pages, num_kv_heads, self.page_bytes)
        if pool is None:
            pool = torch.zeros(shape, dtype=torch.uint8, device="cuda" if device is None else device)
        assert pool.is_cuda, "the pool must be on CUDA (a B200 / sm_100 device)"
        assert pool.dtype == torch.uint8 and pool.shape == shape and pool.is_contiguous(), (
            f"pool must be a contiguous uint8 {list(shape)} tensor")
        self.pool = pool
        self.device = pool.device
        self._index = pool.get_device()
        self._struct = _lib.KV4CacheStruct(pool.data_ptr(), num_layers, num_pages, num_kv_heads, head_dim, page_size,
                                           group_size)
        self._ref = ctypes.byref(self._struct)
        self._ws_bytes = 0
        self._collecting: tuple = (None, 0)        # kv4_attention_weights: the last call's sizes, and its workspace's

    @staticmethod
    def bytes_per_page(head_dim: int, page_size: int, group_size: int) -> int:
        """Bytes of a page of one layer and kv head."""
        return page_size * (head_dim + 8 * (head_dim // group_size))

    def _workspace_bytes(self) -> int:
        """What any attention over this cache needs: the largest it can be depends on the head's layout and the device
        only, and is reached with one warp to a team (many sequences), in the shapes of 8 and of 16 query rows."""
        key = (self._index, self.head_dim, self.group_size)
        if key not in _largest_workspace:
            size, most = ctypes.c_int64(0), 0
            with torch.cuda.device(self._index):
                for heads in (1, 16):
                    _lib.check(_lib.lib().w4a16_kv4_attention_workspace_size(
                        self._ref, 1 << 16, heads * self.num_kv_heads, 1 << 16, 1, ctypes.byref(size)),
                        "w4a16_kv4_attention_workspace_size")
                    most = max(most, size.value)
            _largest_workspace[key] = most
        self._ws_bytes = _largest_workspace[key]
        return self._ws_bytes

    def _check_layer(self, layer: int) -> None:
        assert 0 <= layer < self.num_layers, f"layer={layer} out of range for {self.num_layers} layers"


class KV4Pages:
    """Which sequence (row) holds which pages: ``refs`` int32 ``[num_pages]`` (rows that hold a page;
    0: free), ``block_table`` int32 ``[rows, pages per row]`` (-1: none), ``kv_lens`` int32 ``[rows]``.
    :meth:`empty` makes the tables of a pool nobody uses yet. The tensors may be written to, not replaced. An entry of
    ``kv_lens`` may be lowered (rejected drafts): the row keeps its pages, and grows into them first. Not below what
    it shares with other rows, though: new tokens would be written into their page."""

    def __init__(self, refs: Tensor, block_table: Tensor, kv_lens: Tensor, page_size: int) -> None:
        for name, t, dim in (("refs", refs, 1), ("block_table", block_table, 2), ("kv_lens", kv_lens, 1)):
            assert t.is_cuda and t.dtype == _I32 and t.dim() == dim and t.is_contiguous(), (
                f"{name} must be a contiguous {dim}-dimensional int32 CUDA tensor")
            assert t.device == refs.device, "the tables must be on one CUDA device"
        assert kv_lens.shape[0] == block_table.shape[0], "kv_lens needs one entry per row of block_table"
        assert page_size >= 16 and page_size % 16 == 0, f"page_size={page_size} must be a multiple of 16"
        self.refs, self.block_table, self.kv_lens, self.page_size = refs, block_table, kv_lens, page_size
        self._shape, self._index = (refs.shape[0], *block_table.shape), refs.get_device()
        self._struct = _lib.KV4TablesStruct(refs.data_ptr(), block_table.data_ptr(), kv_lens.data_ptr(), refs.shape[0],
                                            block_table.shape[0], block_table.shape[1], page_size)
        self._ref = ctypes.byref(self._struct)

    @classmethod
    def empty(cls, cache: KV4Cache, rows: int, pages_per_row: int) -> "KV4Pages":
        return cls(torch.zeros(cache.num_pages, dtype=_I32, device=cache.device),
                   torch.full((rows, pages_per_row), -1, dtype=_I32, device=cache.device),
                   torch.zeros(rows, dtype=_I32, device=cache.device), cache.page_size)

    def slots(self, rows: Tensor, positions: Tensor) -> Tensor:
        """Where tokens ``positions`` of sequences ``rows`` (int64 [T] each) lie, as int64 [T]: what
        :func:`qk_norm_rope_append` and :func:`kv4_gather` take. Their pages must be reserved."""
        return self.block_table[rows, positions // self.page_size].long() * self.page_size + positions % self.page_size

    def like(self) -> "KV4Pages":
        """Tables of the same shape, not initialised."""
        return self._like(0)[0]

    def _like(self, extra: int) -> tuple["KV4Pages", Tensor, int]:
        """:meth:`like`, in one allocation with ``extra`` ints behind the tables: (tables, buffer, the extra ints'
        address). The views are made when they are asked for: between two operations nobody does."""
        new = object.__new__(KV4Pages)
        P, R, W = new._shape = self._shape
        new._index, new.page_size = self._index, self.page_size
        new._buf = buf = torch.empty(R * W + P + R + extra, dtype=_I32, device=self._index)   # the table first: aligned
        at = buf.data_ptr()
        refs, lens = at + 4 * R * W, at + 4 * (R * W + P)
        new._struct = _lib.KV4TablesStruct(refs, at, lens, P, R, W, self.page_size)
        new._ref = ctypes.byref(new._struct)
        return new, buf, lens + 4 * R

    def __getattr__(self, name: str):
        if name not in ("refs", "block_table", "kv_lens") or "_buf" not in self.__dict__:
            raise AttributeError(name)
        P, R, W = self._shape
        table, self.refs, self.kv_lens, _ = self._buf.split_with_sizes((R * W, P, R, self._buf.shape[0] - R * W - P - R))
        self.block_table = table.view(R, W)
        return self.__dict__[name]


def _on(device_index: int, fn, *args) -> None:
    """Call a C entry point with ``device_index`` current and its stream as the last argument."""
    if device_index != _current_device():
        with torch.cuda.device(device_index):
            st = fn(*args, _raw_stream(device_index))
    else:
        st = fn(*args, _raw_stream(device_index))
    if st:
        _lib.check(st, fn.__name__)


def _check_heads(name: str, x: Tensor, like: Tensor | None = None) -> None:
    assert x.is_cuda, f"{name} must be on CUDA (a B200 / sm_100 device)"
    assert x.dtype in _CODES, f"{name} must be fp16 or bf16, got {x.dtype}"
    assert x.dim() == 3 and (x.stride(2) == 1 or x.numel() == 0), (
        f"{name} must be [tokens, heads, head_dim] with contiguous channels")
    if like is not None:
        assert x.dtype == like.dtype and x.get_device() == like.get_device(), f"{name} must match q in type and device"
        assert x.shape[0] == like.shape[0] and x.shape[2] == like.shape[2], (
            f"{name} must match q in tokens and head_dim: {tuple(x.shape)} and {tuple(like.shape)}")


def _rope_args(q: Tensor, k: Tensor, v: Tensor | None, positions: Tensor, cos_sin: Tensor, q_weight, k_weight, sections):
    """Checked (axes, end0, end1, weight code) of a rotation. The common case is one expression; anything
    else goes through the checks one by one, which say what is wrong."""
    d, dt, qs, ks, cs = q.get_device(), q.dtype, q.shape, k.shape, cos_sin.shape
    if sections is None:
        axes, end0, end1, shape, fits = 1, 0, 0, qs[:1], True
    else:
        axes, end0, end1, shape = 3, sum(sections[:1]), sum(sections[:2]), (3, *qs[:1])
        fits = len(sections) == 3 and min(sections) >= 0 and len(cs) == 2 and 2 * sum(sections) == cs[1]
    if (fits and d >= 0 and dt in _CODES and len(qs) == 3 and len(ks) == 3 and len(cs) == 2
            and k.dtype is dt and k.get_device() == d and ks[0] == qs[0] and ks[2] == qs[2] and qs[2] in (64, 128)
            and q.stride(2) == 1 and k.stride(2) == 1 and cos_sin.dtype is _F32 and cos_sin.is_contiguous()
            and cos_sin.get_device() == d and cs[1] % 8 == 0 and 0 < cs[1] <= qs[2] and cs[0] > 0
            and positions.dtype is _I64 and positions.shape == shape and positions.is_contiguous()
            and positions.get_device() == d
            and (v is None or (v.dtype is dt and v.shape == ks and v.get_device() == d and v.stride(2) == 1))
            and (q_weight is None or (q_weight.dtype is dt and q_weight.shape == qs[2:] and q_weight.get_device() == d
                                      and q_weight.is_contiguous()))
            and (k_weight is None or (k_weight.dtype is dt and k_weight.shape == qs[2:] and k_weight.get_device() == d
                                      and k_weight.is_contiguous()))):
        return axes, end0, end1, _CODES[dt]
    _check_heads("q", q)
    _check_heads("k", k, q)
    if v is not None:
        _check_heads("v", v, q)
    D, rot = q.shape[2], cos_sin.shape[-1]
    assert D in (64, 128), f"head_dim={D} must be 64 or 128"
    assert cos_sin.dtype is _F32 and cos_sin.dim() == 2 and cos_sin.is_contiguous() and cos_sin.get_device() == d, (
        "cos_sin must be a contiguous fp32 [positions, rotated channels] tensor on q's device")
    assert rot % 8 == 0 and 0 < rot <= D and cos_sin.shape[0] > 0, (
        f"rotated channels ({rot}) must be a multiple of 8, at most head_dim={D}")
    assert sections is None or (len(sections) == 3 and min(sections) >= 0 and sum(sections) == rot // 2), (
        f"sections={sections} must be three counts of frequencies that add up to {rot // 2}")
    assert positions.dtype is _I64 and positions.shape == shape and positions.is_contiguous() and (
        positions.get_device() == d), f"positions must be a contiguous int64 {list(shape)} tensor on q's device"
    code = _CODES[q.dtype]
    for w in (q_weight, k_weight):
        if w is not None:
            assert w.get_device() == d and w.shape == (D,) and w.is_contiguous() and w.dtype in (q.dtype, _F32), (
                f"norm weights must be contiguous [{D}] tensors of q's type or fp32 on its device")
            if w.dtype is _F32:
                code = 1
    if q_weight is not None and k_weight is not None:
        assert q_weight.dtype == k_weight.dtype, "both norm weights must have one type"
    return axes, end0, end1, code


def _ptr(t: Tensor | None):
    return None if t is None else t.data_ptr()


def _out_like(q: Tensor, out: Tensor | None, name: str = "out") -> Tensor:
    if out is None:
        return torch.empty_like(q, memory_format=_CONTIGUOUS)
    assert out.shape == q.shape and out.dtype == q.dtype and out.is_contiguous() and out.device == q.device, (
        f"{name} must be a contiguous {q.dtype} {list(q.shape)} tensor on q's device")
    return out


def qk_norm_rope(q: Tensor, k: Tensor, positions: Tensor, cos_sin: Tensor, q_weight: Tensor | None = None,
                 k_weight: Tensor | None = None, eps: float = 1e-6, *, sections: tuple[int, int, int] | None = None,
                 interleaved: bool = False, out: tuple[Tensor, Tensor] | None = None) -> tuple[Tensor, Tensor]:
    """RMS norm of each query and key head and their rotation by position, in one pass.

    Args:
        q: [T, heads, D] fp16 or bf16, channels contiguous (views of a fused projection's output will do).
        k: [T, kv_heads, D], likewise.
        positions: int64 [T], or [3, T] (time, height, width) with ``sections``.
        cos_sin: fp32 [max_position, rot]: the cosines of the rot/2 angles of a position, then their sines;
            the first ``rot`` channels of a head are rotated (a multiple of 8).
        q_weight, k_weight: norm weights [D] (q's type, or fp32); None: no norm.
        sections: how many of the rot/2 frequencies turn by each of three axes, in order.
        interleaved: pairs are channels (2i, 2i + 1) instead of (i, i + rot/2).
        out: optional (q, k) outputs.

    Returns:
        (q, k) dense, of q's type: fp32 arithmetic, rounded once.
    """
    axes, end0, end1, wcode = _rope_args(q, k, None, positions, cos_sin, q_weight, k_weight, sections)
    T, H, D = q.shape
    qo, ko = (_out_like(q, None), _out_like(k, None)) if out is None else (_out_like(q, out[0]), _out_like(k, out[1]))
    qs, ks = q.stride(), k.stride()
    _on(q.get_device(), _lib.lib().w4a16_qk_norm_rope, q.data_ptr(), k.data_ptr(), _CODES[q.dtype], T, H, k.shape[1], D,
        qs[0], qs[1], ks[0], ks[1], positions.data_ptr(), axes, end0, end1, cos_sin.data_ptr(), cos_sin.shape[0],
        cos_sin.shape[1], interleaved, _ptr(q_weight), _ptr(k_weight), wcode, eps, qo.data_ptr(), ko.data_ptr())
    return qo, ko


def qk_norm_rope_append(q: Tensor, k: Tensor, v: Tensor, cache: KV4Cache, layer: int, slots: Tensor, positions: Tensor,
                        cos_sin: Tensor, q_weight: Tensor | None = None, k_weight: Tensor | None = None,
                        eps: float = 1e-6, *, sections: tuple[int, int, int] | None = None, interleaved: bool = False,
                        out: Tensor | None = None) -> Tensor:
    """:func:`qk_norm_rope` whose keys, and the values ``v`` [T, kv_heads, D], go into the cache in 4 bits
    instead of memory in 16.

    ``slots`` int64 [T] says where: page * page_size + place in the page (negative: this token is not
    cached); no slot twice in one call. Returns the queries [T, heads, D]."""
    axes, end0, end1, wcode = _rope_args(q, k, v, positions, cos_sin, q_weight, k_weight, sections)
    T, H, D = q.shape
    d = q.get_device()
    assert 0 <= layer < cache.num_layers, f"layer={layer} out of range for {cache.num_layers} layers"
    assert k.shape[1] == cache.num_kv_heads and v.shape[1] == cache.num_kv_heads and D == cache.head_dim, (
        f"k and v must have the cache's {cache.num_kv_heads} heads of {cache.head_dim}")
    assert cache._index == d, "the cache must be on q's device"
    assert slots.dtype is _I64 and slots.shape == (T,) and slots.is_contiguous() and slots.get_device() == d, (
        f"slots must be a contiguous int64 [{T}] tensor on q's device")
    qo = _out_like(q, out)
    qs, ks, vs = q.stride(), k.stride(), v.stride()
    _on(d, _lib.lib().w4a16_qk_norm_rope_append, q.data_ptr(), k.data_ptr(), v.data_ptr(), _CODES[q.dtype], T, H, qs[0],
        qs[1], ks[0], ks[1], vs[0], vs[1], positions.data_ptr(), axes, end0, end1, cos_sin.data_ptr(), cos_sin.shape[0],
        cos_sin.shape[1], interleaved, _ptr(q_weight), _ptr(k_weight), wcode, eps, qo.data_ptr(), cache._ref, layer,
        slots.data_ptr())
    return qo


def kv4_gather(cache: KV4Cache, layer: int, slots: Tensor, dtype: torch.dtype = torch.float16) -> Tensor:
    """Cached tokens back in 16 bits: ``[2, n, kv_heads, D]`` (keys, then values) of the tokens in ``slots``
    int64 [n]; a negative slot gives zeros."""
    cache._check_layer(layer)
    assert dtype in _CODES, f"dtype must be fp16 or bf16, got {dtype}"
    assert slots.dtype is _I64 and slots.dim() == 1 and slots.is_contiguous() and slots.get_device() == cache._index, (
        "slots must be a contiguous int64 [n] tensor on the cache's device")
    n = slots.shape[0]
    out = cache.pool.new_empty((2, n, cache.num_kv_heads, cache.head_dim), dtype=dtype)
    _on(cache._index, _lib.lib().w4a16_kv4_gather, cache._ref, layer, slots.data_ptr(), n, out.data_ptr(), _CODES[dtype])
    return out


def kv4_attention(q: Tensor, cache: KV4Cache, layer: int, block_table: Tensor, kv_lens: Tensor, *,
                  cu_q: Tensor | None = None, max_q: int | None = None, scale: float | None = None, window: int = 0,
                  sinks: int = 0, out: Tensor | None = None, return_lse: bool = False) -> Tensor | tuple[Tensor, Tensor]:
    """Attention of new tokens over the cached ones, themselves among them.

    Args:
        q: [T, heads, D] fp16 or bf16; query head h reads kv head h // (heads // kv_heads). 16-byte aligned,
            strides multiples of 8 elements.
        block_table: int32 [sequences, pages]: each sequence's pages in order. What lies beyond a sequence's
            length is not read.
        kv_lens: int32 [sequences]: cached tokens, the new ones (already appended) included. 0: an unused
            place in the batch, whose queries give zeros.
        cu_q: int32 [sequences + 1]: the first query of each sequence; None: T / sequences each. A sequence's
            last query stands at position kv_lens - 1; each sees the tokens up to its own position. Queries before
            cu_q[0] and from cu_q[-1] on (padding) give zeros.
        max_q: the most queries a sequence has (with cu_q; default T).
        scale: of the scores; default 1 / sqrt(D).
        window: only the last ``window`` tokens up to a query's position; 0: all.
        sinks: with a window, a sequence's first ``sinks`` tokens stay visible (what lies between is not read).
        out: optional output.
        return_lse: also return the log-sum-exp of the scores, fp32 [T, heads] (-inf where nothing is seen).

    Returns:
        [T, heads, D] of q's type, or (that, lse).
    """
    # The common case in one expression; anything else goes through the checks one by one, which say
    # what is wrong.
    d, dt, qh, th = q.get_device(), q.dtype, q.shape, block_table.shape
    if not (d == cache._index and dt in _CODES and len(qh) == 3 and qh[2] == cache.head_dim and len(th) == 2
            and 0 <= layer < cache.num_layers and qh[1] > 0 and qh[1] % cache.num_kv_heads == 0
            and block_table.dtype is _I32 and block_table.get_device() == d and block_table.is_contiguous()
            and kv_lens.dtype is _I32 and kv_lens.get_device() == d and kv_lens.shape == th[:1] and kv_lens.is_contiguous()
            and window >= 0 and sinks >= 0):
        _check_attention(q, cache, layer, block_table, kv_lens, window, sinks)
    T, H, D = qh
    B, width = th
    qt, qs, qc = q.stride()
    assert qc == 1 or q.numel() == 0, "q must be [tokens, heads, head_dim] with contiguous channels"
    if cu_q is None:
        assert T == 0 or (B > 0 and T % B == 0), f"{T} queries do not divide into {B} sequences: cu_q is needed"
        max_q = T // B if B else 0
    else:
        assert cu_q.dtype is _I32 and cu_q.shape == (B + 1,) and cu_q.is_contiguous() and cu_q.get_device() == d, (
            f"cu_q must be a contiguous int32 [{B + 1}] tensor on q's device")
        max_q = T if max_q is None else max_q
        assert max_q >= 0, f"max_q={max_q} must not be negative"
    o = torch.empty_like(q, memory_format=_CONTIGUOUS) if out is None else _out_like(q, out)
    lse = q.new_empty((T, H), dtype=_F32) if return_lse else None
    ws = _lib.kv4_workspace(cache._ws_bytes or cache._workspace_bytes(), d, _raw_stream(d))
    _on(d, _lib.lib().w4a16_kv4_attention_sinks, q.data_ptr(), _CODES[dt], T, H, qt, qs, cache._ref, layer,
        block_table.data_ptr(), width, kv_lens.data_ptr(), None if cu_q is None else cu_q.data_ptr(), B, max_q,
        D ** -0.5 if scale is None else scale, min(window, _INT_MAX), min(sinks, _INT_MAX), o.data_ptr(),
        None if lse is None else lse.data_ptr(), ws.data_ptr(), ws.numel())
    return (o, lse) if return_lse else o


def _check_attention(q: Tensor, cache: KV4Cache, layer: int, block_table: Tensor, kv_lens: Tensor, window: int,
                     sinks: int) -> None:
    """kv4_attention's checks, one by one, so a bad call fails with the specific message."""
    _check_heads("q", q)
    _, H, D = q.shape
    d = q.get_device()
    cache._check_layer(layer)
    assert D == cache.head_dim and H > 0 and H % cache.num_kv_heads == 0, (
        f"q must have a multiple of the cache's {cache.num_kv_heads} kv heads, of {cache.head_dim} channels")
    assert cache._index == d, "the cache must be on q's device"
    assert block_table.dtype is _I32 and block_table.dim() == 2 and block_table.is_contiguous() and (
        block_table.get_device() == d), "block_table must be a contiguous int32 [sequences, pages] tensor on q's device"
    B = block_table.shape[0]
    assert kv_lens.dtype is _I32 and kv_lens.shape == (B,) and kv_lens.is_contiguous() and kv_lens.get_device() == d, (
        f"kv_lens must be a contiguous int32 [{B}] tensor on q's device")
    assert window >= 0, f"window={window} must not be negative"
    assert sinks >= 0, f"sinks={sinks} must not be negative"


def _check_weights(name: str, w: Tensor, shape: tuple, device_index: int) -> None:
    assert w.dtype is _F32 and w.get_device() == device_index and w.dim() == len(shape) + 1 and w.shape[:-1] == shape and (
        w.stride(-1) == 1 or w.shape[-1] <= 1), (
        f"{name} must be fp32 {[*shape, 'tokens']} on the cache's device, the last axis contiguous")


def _axes(w: Tensor) -> list[tuple[int, int]]:
    """(stride, entries) of all axes but the last, the largest stride first; those of one entry left out."""
    return sorted(((s, m) for m, s in zip(w.shape[:-1], w.stride()) if m != 1), reverse=True)


def _span(w: Tensor) -> int:
    """Floats from a non-empty tensor's first to behind its last."""
    return 1 + sum((m - 1) * s for m, s in zip(w.shape, w.stride()))


def _meet(axes: list[tuple[int, int]], tokens: int, by: int) -> bool:
    """Whether entries of nested axes, of two tensors that lie ``by`` floats apart, share some."""
    if not axes:
        return abs(by) < tokens
    (s, m), rest = axes[0], axes[1:]
    return any(abs(k) < m and _meet(rest, tokens, by - k * s) for k in (by // s, by // s + 1))


def _check_written(w: Tensor, read: Tensor) -> None:
    if w.numel() == 0:
        return
    axes, extent = _axes(w), w.shape[-1]
    for s, m in reversed(axes):
        assert s >= extent, "weights that are written must not share memory between their entries"
        extent += s * (m - 1)
    by = w.data_ptr() - read.data_ptr()
    if by >= 4 * _span(read) or by <= -4 * _span(w):
        return
    same = all(a == b or m == 1 for a, b, m in zip(w.stride(), read.stride(), w.shape))
    assert same if by == 0 else axes == _axes(read) and by % 4 == 0 and not _meet(axes, w.shape[-1], by // 4), (
        "weights that are written must be those that are read, or share no memory with them")


def kv4_attention_weights(q: Tensor, cache: KV4Cache, layer: int, block_table: Tensor, kv_lens: Tensor, lse: Tensor,
                          weights: Tensor, *, cu_q: Tensor | None = None, max_q: int | None = None,
                          scale: float | None = None, window: int = 0, sinks: int = 0, out: Tensor | None = None) -> Tensor:
    """The attention weight that cached tokens collect, what :func:`kv4_evict` goes by: to each token's weight of a kv
    head the sum, over the queries that see it and the heads of its group, of ``exp(score - lse)`` is added.

    Args:
        q ... kv_lens, cu_q ... sinks: as in the :func:`kv4_attention` call whose weights are meant.
        lse: fp32 [T, heads], what that call returned with ``return_lse`` (a query of -inf gives nothing).
        weights: fp32 [sequences, kv_heads, tokens], what earlier calls collected; any strides but the last. Tokens that are
            new in this call (the queries' own) start from nothing, whatever it holds, so neither new rows nor
            places of rejected drafts have to be cleared.
        out: where the sums go, all tokens of every sequence; shares no memory with ``weights``, or is it. Default:
            ``weights``, where only those that a query sees change. What lies behind a sequence's length is not written.

    Every query counts, those of drafts that are rejected later too: their own places start from nothing again, but what
    they gave to older tokens stays. To collect from the drafts that stand alone, call this behind
    :func:`w4a16.verify_drafts` with the lengths that the attention had (lower them afterwards), and with ``lse`` -inf
    in the rows of the rejected drafts. With K drafts to a sequence: ``gone = torch.arange(K + 1, device=lse.device) >
    accepted[:, None]; lse.unflatten(0, (-1, K + 1)).masked_fill_(gone[..., None], -math.inf)``.

    Returns ``out``, or ``weights``. A sequence longer than the weights is left out, with the error of an index out of
    range. fp32 throughout; two calls on the same inputs give the same bits.
    """
    # The common case in one expression; anything else goes through the checks one by one, which say what is wrong.
    d, qh = q.get_device(), q.shape
    assert d >= 0, "q must be on CUDA (a B200 / sm_100 device)"
    th, wh, after = block_table.shape, weights.shape, weights if out is None else out
    if not (d == cache._index and q.dtype in _CODES and len(qh) == 3 and qh[2] == cache.head_dim and len(th) == 2
            and 0 <= layer < cache.num_layers and qh[1] > 0 and qh[1] % cache.num_kv_heads == 0 and q.stride(2) == 1
            and block_table.dtype is _I32 and block_table.get_device() == d and block_table.is_contiguous()
            and kv_lens.dtype is _I32 and kv_lens.get_device() == d and kv_lens.shape == th[:1] and kv_lens.is_contiguous()
            and window >= 0 and sinks >= 0 and lse.dtype is _F32 and lse.shape == qh[:2] and lse.get_device() == d and lse.is_contiguous()
            and len(wh) == 3 and wh[0] == th[0] and wh[1] == cache.num_kv_heads and weights.dtype is _F32
            and weights.get_device() == d and weights.stride(2) == 1 and after.is_contiguous() and after.shape == wh
            and after.dtype is _F32 and after.get_device() == d
            and cu_q is not None and cu_q.dtype is _I32 and cu_q.shape == (th[0] + 1,) and cu_q.is_contiguous() and cu_q.get_device() == d
            and (max_q is None or max_q >= 0)):
        _check_collecting(q, cache, layer, block_table, kv_lens, lse, weights, cu_q, max_q, window, sinks, out)
    T, H, _ = qh
    B, width = th
    if cu_q is None:
        max_q = T // B if B else 0
    elif max_q is None:
        max_q = T
    if B == 0:
        return after
    # (the sizes of the last call are likely those of this one)
    sizes = (T, H, B, max_q, wh[2])
    known, nbytes = cache._collecting
    if known != sizes:
        need = ctypes.c_int64(0)
        with torch.cuda.device(d):
            _lib.check(_lib.lib().w4a16_kv4_attention_weights_workspace_size(cache._ref, *sizes, ctypes.byref(need)),
                       "w4a16_kv4_attention_weights_workspace_size")
        nbytes = need.value
        cache._collecting = sizes, nbytes
    ws = torch.empty(nbytes, dtype=torch.uint8, device=d)
    qt, qs, _ = q.stride()
    ws0, ws1, _ = weights.stride()
    as0, as1, _ = after.stride()
    try:
        _on(d, _lib.lib().w4a16_kv4_attention_weights, q.data_ptr(), _CODES[q.dtype], T, H, qt, qs, cache._ref, layer,
            block_table.data_ptr(), width, kv_lens.data_ptr(), _ptr(cu_q), B, max_q, q.shape[2] ** -0.5 if scale is None else scale,
            min(window, _INT_MAX), min(sinks, _INT_MAX), lse.data_ptr(), weights.data_ptr(), ws0, ws1, after.data_ptr(), as0, as1,
            wh[2], ws.data_ptr(), nbytes)
    except _lib.W4A16Error:
        _check_written(after, weights)         # (the common case leaves it to the library to find an overlap)
        raise
    return after


def _check_collecting(q: Tensor, cache: KV4Cache, layer: int, block_table: Tensor, kv_lens: Tensor, lse: Tensor, weights: Tensor,
                      cu_q: Tensor | None, max_q: int | None, window: int, sinks: int, out: Tensor | None) -> None:
    """kv4_attention_weights' checks, one by one, so a bad call fails with the specific message."""
    _check_attention(q, cache, layer, block_table, kv_lens, window, sinks)
    T, H, _ = q.shape
    B = block_table.shape[0]
    d = cache._index
    assert lse.dtype is _F32 and lse.shape == (T, H) and lse.is_contiguous() and lse.get_device() == d, (
        f"lse must be a contiguous fp32 [{T}, {H}] tensor on q's device")
    if cu_q is None:
        assert T == 0 or (B > 0 and T % B == 0), f"{T} queries do not divide into {B} sequences: cu_q is needed"
    else:
        assert cu_q.dtype is _I32 and cu_q.shape == (B + 1,) and cu_q.is_contiguous() and cu_q.get_device() == d, (
            f"cu_q must be a contiguous int32 [{B + 1}] tensor on q's device")
        assert max_q is None or max_q >= 0, f"max_q={max_q} must not be negative"
    shape = (B, cache.num_kv_heads)
    _check_weights("weights", weights, shape, d)
    if out is not None:
        _check_weights("out", out, shape, d)
        assert out.shape == weights.shape, "out must have the shape of weights"
    _check_written(weights if out is None else out, weights)


def _ints(name: str, t: Tensor, n: int, device_index: int) -> None:
    assert t.dtype is _I32 and t.shape == (n,) and t.is_contiguous() and t.get_device() == device_index, (
        f"{name} must be a contiguous int32 [{n}] tensor on the cache's device")


def _check_pages(cache: KV4Cache, pages: KV4Pages) -> None:
    assert pages._index == cache._index, "the tables must be on the cache's device"
    assert pages._shape[0] == cache.num_pages and pages.page_size == cache.page_size, (
        "the tables must be of the cache's pages")


def _tables_out(pages: KV4Pages, out: KV4Pages | None, extra: int = 0) -> tuple[KV4Pages, Tensor | None, int | None]:
    """(tables to write, a buffer that ends with ``extra`` ints, their address)."""
    if out is None:
        return pages._like(extra)
    assert out._shape == pages._shape and out.page_size == pages.page_size and out._index == pages._index, (
        "out must be tables of the same shape")
    buf = torch.empty(extra, dtype=_I32, device=pages._index) if extra else None
    return out, buf, None if buf is None else buf.data_ptr()


def kv4_copy_pages(cache: KV4Cache, src: Tensor, dst: Tensor) -> None:
    """Copy page ``src[i]`` to page ``dst[i]`` in every layer (int32 [n] each; a pair with a negative entry is
    skipped). A page that is some pair's dst must be no other pair's src or dst."""
    n = src.shape[0] if src.dim() == 1 else -1
    _ints("src", src, n, cache._index)
    _ints("dst", dst, n, cache._index)
    _on(cache._index, _lib.lib().w4a16_kv4_copy_pages, cache._ref, src.data_ptr(), dst.data_ptr(), n)


def kv4_reserve(pages: KV4Pages, rows: Tensor, lens: Tensor) -> Tensor:
    """Let row ``rows[i]`` hold ``lens[i]`` tokens (int32 [n] each, no row twice): it gets the free pages with the
    lowest ids, in the order of the requests, and its ``kv_lens`` becomes ``lens[i]``. Returns int32 [n]: 1, or
    0 (row unchanged) where the free pages do not reach that far down the list, the table is too narrow, or
    the row holds more than ``lens[i]`` already. Pages that a row has beyond its length (its ``kv_lens`` was lowered)
    are used before free ones. Changes ``pages`` in place."""
    d = pages._index
    n = rows.shape[0] if rows.dim() == 1 else -1
    _ints("rows", rows, n, d)
    _ints("lens", lens, n, d)
    buf = torch.empty(2 * n + 1, dtype=_I32, device=d)
    _on(d, _lib.lib().w4a16_kv4_reserve, pages._ref, rows.data_ptr(), lens.data_ptr(), n, buf.data_ptr(),
        buf.data_ptr() + 4 * n)
    return buf[:n]


def kv4_fork(cache: KV4Cache, pages: KV4Pages, parents: Tensor, children: Tensor, *,
             out: KV4Pages | None = None) -> tuple[KV4Pages, Tensor]:
    """Row ``children[i]`` becomes a copy of sequence ``parents[i]`` (int32 [n] each): full pages are shared, a partly
    filled last page is copied, in every layer, into the lowest free page. Children hold no pages before, appear
    once, and are no parents. Returns the tables (new ones, or ``out``, which may be ``pages``) and int32 [n]:
    1, or 0 (and an empty child) where no page was free."""
    _check_pages(cache, pages)
    n = parents.shape[0] if parents.dim() == 1 else -1
    _ints("parents", parents, n, cache._index)
    _ints("children", children, n, cache._index)
    out, buf, at = _tables_out(pages, out, 3 * n)      # ok, and 2 n of scratch
    _on(cache._index, _lib.lib().w4a16_kv4_fork, cache._ref, pages._ref, out._ref, parents.data_ptr(), children.data_ptr(),
        n, at, at and at + 4 * n)
    return out, parents.new_empty(0) if buf is None else buf.narrow(0, buf.shape[0] - 3 * n, n)


def kv4_release(pages: KV4Pages, rows: Tensor, *, out: KV4Pages | None = None) -> KV4Pages:
    """The rows (int32 [n]) give their pages back and are empty. Returns the tables (new ones, or ``out``, which
    may be ``pages``)."""
    d = pages._index
    n = rows.shape[0] if rows.dim() == 1 else -1
    _ints("rows", rows, n, d)
    out = _tables_out(pages, out)[0]
    _on(d, _lib.lib().w4a16_kv4_release, pages._ref, out._ref, rows.data_ptr(), n)
    return out


def kv4_compact(cache: KV4Cache, pages: KV4Pages, *, out: KV4Pages | None = None) -> KV4Pages:
    """Make the pool dense: with c pages in use, the i-th page in use with an id >= c moves to the i-th free page
    with an id < c, in every layer, and the tables follow. The pages from c on are then free. Returns the tables
    (new ones, or ``out``, which may be ``pages``)."""
    _check_pages(cache, pages)
    out, buf, at = _tables_out(pages, out, 2 * cache.num_pages + 1)
    _on(cache._index, _lib.lib().w4a16_kv4_compact, cache._ref, pages._ref, out._ref, at)
    return out


def kv4_evict(cache: KV4Cache, pages: KV4Pages, weights: Tensor, rows: Tensor, keep: int, *, sinks: int = 0,
              recent: int = 0, out: KV4Pages | None = None, out_weights: Tensor | None = None) -> tuple[KV4Pages, Tensor]:
    """Rows that hold more than ``keep`` tokens keep ``keep`` of them, in every layer and kv head on its own: the
    first ``sinks``, the last ``recent``, and of the others those with the largest weights (equal ones: the
    lowest positions; NaN: below every number), in their order.

    Args:
        weights: fp32 [layers, rows of the tables, kv_heads, tokens], what :func:`kv4_attention_weights` collects; any
            strides but the last.
        rows: int32 [n], the rows to look at; one of at most ``keep`` tokens stays as it is.
        out: where the new tables go; default: new ones. May be ``pages``.
        out_weights: where the kept tokens' weights go ([..., :keep] of the rows evicted from); default: ``weights``. Another
            tensor shares no memory with it.

    What is kept moves into fresh pages (the lowest free ids, in the order of the requests), so pages that other rows
    share stay as they are, and the row's old ones are given back: a row needs ``ceil(keep / page_size)`` free pages
    for the time of the call. Keys keep the rotation of the position they were appended at; the next token is appended
    at place ``keep``, with the position it has in the text.

    Returns the tables and int32 [n]: 1, or 0 (row unchanged) where the free pages do not reach that far down the
    list, or the row was named before. A row out of range, or longer than the weights, gives 0 and the error of an index
    out of range.
    """
    _check_pages(cache, pages)
    d = cache._index
    n = rows.shape[0] if rows.dim() == 1 else -1
    _ints("rows", rows, n, d)
    kept = weights if out_weights is None else out_weights
    shape = (cache.num_layers, pages._shape[1], cache.num_kv_heads, *weights.shape[3:])
    if not (len(shape) == 4 and weights.shape == shape and weights.dtype is _F32 and weights.get_device() == d and weights.stride(3) == 1
            and kept.shape == shape and kept.dtype is _F32 and kept.get_device() == d and kept.is_contiguous()):
        _check_weights("weights", weights, shape[:3], d)
        if out_weights is not None:
            _check_weights("out_weights", out_weights, shape[:3], d)
            assert out_weights.shape == weights.shape, "out_weights must have the shape of weights"
        _check_written(kept, weights)
    assert sinks >= 0 and recent >= 0 and 1 <= keep <= _INT_MAX and sinks + recent <= keep, (
        f"keep={keep} must be positive, and hold sinks={sinks} and recent={recent}")
    _, R, W = pages._shape
    need = min(-(-keep // cache.page_size), W)
    assert n * need <= _INT_MAX, f"{n} rows of {need} pages are more than one call can ask for"
    out, buf, at = _tables_out(pages, out, n * (4 + need + W) + 1 + R)
    ws, ks = weights.stride(), kept.stride()
    try:
        _on(d, _lib.lib().w4a16_kv4_evict, cache._ref, pages._ref, out._ref, weights.data_ptr(), ws[0], ws[1], ws[2],
            kept.data_ptr(), ks[0], ks[1], ks[2], weights.shape[3], rows.data_ptr(), n, keep, sinks, recent, at, at and at + 4 * n)
    except _lib.W4A16Error:
        _check_written(kept, weights)          # (the common case leaves it to the library to find an overlap)
        raise
    return out, buf.narrow(0, (at - buf.data_ptr()) // 4, n)
