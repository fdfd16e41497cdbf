"""The end of a step of drafted tokens: their verification against the target's probabilities.

No reference counterpart (the reference ends at the linear layers). The step appends a sequence's last token and
its drafts to the cache, attends them together (:func:`w4a16.kv4_attention`), and takes the target's
probabilities behind each; :func:`verify_drafts` says how many drafts stand, draws the next token, and lowers the
cache's lengths by what was rejected. It runs in the sm_100a library on torch's current stream and never
synchronises.
"""
from __future__ import annotations

import torch
from torch import Tensor

from . import _lib
from .kv_cache import _on, _ptr

__all__ = ["verify_drafts"]

_I32, _I64, _F32 = torch.int32, torch.int64, torch.float32
_TYPES = _lib.DTYPE_CODES


def _check_probabilities(name: str, x: Tensor, shape: tuple, like: Tensor | None) -> None:
    assert x.is_cuda, f"{name} must be on CUDA (a B200 / sm_100 device)"
    assert x.dtype in _TYPES, f"{name} must be fp32, fp16 or bf16, got {x.dtype}"
    assert x.dim() == 3 and x.shape == shape and (x.stride(2) == 1 or x.shape[2] == 1), (
        f"{name} must be {list(shape)} probabilities, the last axis contiguous")
    if like is not None:
        assert x.dtype == like.dtype and x.get_device() == like.get_device(), f"{name} must match target in type and device"


def _check(target: Tensor, draft: Tensor | None, tokens: Tensor, uniforms: Tensor, counts: Tensor | None, kv_lens: Tensor | None,
           rows: Tensor | None) -> None:
    """verify_drafts' checks, one by one, so a bad call fails with the specific message."""
    assert target.dim() == 3 and target.shape[1] > 0 and target.shape[2] > 0, "target must be [sequences, drafts + 1, vocabulary]"
    B, K1, V = target.shape
    K = K1 - 1
    d = target.get_device()
    _check_probabilities("target", target, (B, K1, V), None)
    if draft is not None:
        _check_probabilities("draft", draft, (B, K, V), target)
    assert tokens.dtype is _I64 and tokens.shape == (B, K) and tokens.is_contiguous() and tokens.get_device() == d, (
        f"tokens must be a contiguous int64 [{B}, {K}] tensor on target's device")
    assert uniforms.dtype is _F32 and uniforms.shape == (B, K1) and uniforms.is_contiguous() and uniforms.get_device() == d, (
        f"uniforms must be a contiguous fp32 [{B}, {K1}] tensor on target's device")
    for name, t in (("counts", counts), ("rows", rows)):
        assert t is None or (t.dtype is _I32 and t.shape == (B,) and t.is_contiguous() and t.get_device() == d), (
            f"{name} must be a contiguous int32 [{B}] tensor on target's device")
    assert kv_lens is None or (kv_lens.dtype is _I32 and kv_lens.dim() == 1 and kv_lens.is_contiguous()
                               and kv_lens.get_device() == d), "kv_lens must be a contiguous int32 tensor on target's device"
    assert rows is None or kv_lens is not None, "rows say which entries of kv_lens are meant"
    assert kv_lens is None or rows is not None or kv_lens.shape[0] >= B, f"kv_lens must have an entry for each of {B} sequences"


def verify_drafts(target: Tensor, draft: Tensor | None, tokens: Tensor, uniforms: Tensor, *, counts: Tensor | None = None,
                  kv_lens: Tensor | None = None, rows: Tensor | None = None) -> tuple[Tensor, Tensor]:
    """Accept the drafts that the target's probabilities bear out, and draw the token behind them.

    Draft i of a sequence is accepted while ``uniforms[i] * q < p``: p and q are what the target and the draft
    model give it at its place. The token behind the a accepted ones is drawn by the last of ``uniforms`` from
    max(target[a] - draft[a], 0), or from target[a] itself where all were accepted (or nothing is left): the first
    whose running sum exceeds that number times the whole. The sums are within 2^-45 + V 2^-64 of the
    whole, however large the batch.

    Args:
        target: [B, K + 1, V] probabilities (fp32, fp16 or bf16; they need not add up to 1, any strides but the
            last) behind each sequence's last token and its K drafts.
        draft: [B, K, V] probabilities that the drafts were drawn from; None: they were not drawn (looked up in the
            text, say), which is a probability of 1 each.
        tokens: int64 [B, K], the drafts.
        uniforms: fp32 [B, K + 1] random numbers in [0, 1): one for each draft, and the last one for the draw.
        counts: int32 [B]: a sequence has only the first ``counts[b]`` drafts; None: K each.
        kv_lens: int32, lowered in place by the number of each sequence's rejected drafts (``KV4Pages.kv_lens``).
        rows: int32 [B]: which entry of ``kv_lens`` is a sequence's; None: the first B in order.

    Returns:
        (tokens int64 [B, K + 1], accepted int32 [B]): the accepted drafts, the token drawn behind them, and -1 from
        there on. A row without any probability has nothing to draw: its token is -1. A value whose difference is
        negative or not finite counts as none.
    """
    # The common case in one expression; anything else goes through the checks one by one, which say what is wrong.
    d, dt, shape = target.get_device(), target.dtype, target.shape
    if not (d >= 0 and dt in _TYPES and len(shape) == 3 and shape[1] > 0 and shape[2] > 0 and target.stride(2) == 1
            and (draft is None or (draft.dtype is dt and draft.get_device() == d and draft.shape == (shape[0], shape[1] - 1, shape[2])
                                   and draft.stride(2) == 1))
            and tokens.dtype is _I64 and tokens.shape == (shape[0], shape[1] - 1) and tokens.is_contiguous()
            and tokens.get_device() == d and uniforms.dtype is _F32 and uniforms.shape == shape[:2] and uniforms.is_contiguous()
            and uniforms.get_device() == d and kv_lens is None and rows is None
            and (counts is None or (counts.dtype is _I32 and counts.shape == shape[:1] and counts.is_contiguous()
                                    and counts.get_device() == d))):
        _check(target, draft, tokens, uniforms, counts, kv_lens, rows)
    B, K1, V = shape
    K = K1 - 1
    out, accepted = tokens.new_empty((B, K1)), tokens.new_empty((B,), dtype=_I32)
    ts, ds = target.stride(), (0, 0) if draft is None else draft.stride()
    _on(d, _lib.lib().w4a16_verify_drafts, target.data_ptr(), ts[0], ts[1],
        _ptr(draft), ds[0], ds[1],
        _TYPES[dt], B, K, V, tokens.data_ptr(), uniforms.data_ptr(), _ptr(counts), _ptr(kv_lens),
        _ptr(rows), 0 if kv_lens is None else kv_lens.shape[0], out.data_ptr(), accepted.data_ptr())
    return out, accepted
