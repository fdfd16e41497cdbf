"""``W4A16Attention`` -- an attention layer between two W4A16 projections, over the 4-bit paged cache.

No reference counterpart (the reference ends at the linear layers). It runs what a serving step runs:

    qkv projection        W4A16Linear                      (fused dequant-GEMM)
    norm, rotation, cache qk_norm_rope_append              (one kernel)
    attention             kv4_attention                    (prompts, drafts and single tokens in one call)
    output projection     W4A16Linear

Sequences live in a :class:`KV4Cache` shared by all layers and a :class:`KV4Pages` that says which pages are
whose; ``kv4_reserve`` makes room before a step, ``kv4_fork``, ``kv4_release`` and ``kv4_compact`` manage them
between steps.
"""
from __future__ import annotations

import torch
from torch import Tensor, nn

from .kv_cache import KV4Cache, KV4Pages, kv4_attention, qk_norm_rope_append
from .linear import W4A16Linear

__all__ = ["W4A16Attention"]


class W4A16Attention(nn.Module):
    """Attention of ``heads`` query heads over ``kv_heads`` cached heads of ``head_dim`` channels, fp16.

    Args:
        hidden: features of the layer's input and output.
        heads, kv_heads, head_dim: head layout; ``heads`` a multiple of ``kv_heads``, ``head_dim`` 64 or 128.
        group_size: quantisation group of the two projections.
        bias: whether the projections have one.
        qk_norm: RMS norm of every query and key head (weights ``q_norm`` and ``k_norm``, ones until loaded).
        eps: of that norm.
        interleaved: rotation pairs (2i, 2i + 1) instead of (i, i + rot/2).
        window: a query sees the last ``window`` tokens; 0: all.

    The projections are ``qkv`` (query heads, then key heads, then value heads) and ``out``.
    """

    def __init__(self, hidden: int, heads: int, kv_heads: int, head_dim: int, *, group_size: int = 128,
                 bias: bool = False, qk_norm: bool = True, eps: float = 1e-6, interleaved: bool = False, window: int = 0,
                 device: torch.device | str | None = None) -> None:
        super().__init__()
        if head_dim not in (64, 128):
            raise ValueError(f"head_dim={head_dim} must be 64 or 128")
        if kv_heads < 1 or heads < 1 or heads % kv_heads != 0:
            raise ValueError(f"heads={heads} must be a multiple of kv_heads={kv_heads}")
        if window < 0:
            raise ValueError(f"window={window} must not be negative")
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.eps, self.interleaved, self.window = eps, interleaved, window
        self.qkv = W4A16Linear(hidden, (heads + 2 * kv_heads) * head_dim, group_size, bias, device)
        self.out = W4A16Linear(heads * head_dim, hidden, group_size, bias, device)
        for name in ("q_norm", "k_norm"):
            self.register_buffer(name, torch.ones(head_dim, dtype=torch.float16, device=device) if qk_norm else None)

    def forward(self, x: Tensor, cache: KV4Cache, layer: int, pages: KV4Pages, slots: Tensor, positions: Tensor,
                cos_sin: Tensor, *, cu_q: Tensor | None = None, max_q: int | None = None,
                sections: tuple[int, int, int] | None = None) -> Tensor:
        """``x`` [T, hidden] fp16, the new tokens of all rows of ``pages`` one after another; ``pages.kv_lens``
        counts them already. ``slots`` (``pages.slots``), ``positions``, ``cos_sin`` and ``sections`` as in
        :func:`qk_norm_rope_append`, ``cu_q`` and ``max_q`` as in :func:`kv4_attention`."""
        assert x.dim() == 2, f"x must be [tokens, hidden], got {tuple(x.shape)}"
        H, KV = self.heads, self.kv_heads
        qkv = self.qkv(x).view(x.shape[0], H + 2 * KV, self.head_dim)
        q = qk_norm_rope_append(qkv[:, :H], qkv[:, H:H + KV], qkv[:, H + KV:], cache, layer, slots, positions, cos_sin,
                                self.q_norm, self.k_norm, self.eps, sections=sections, interleaved=self.interleaved)
        o = kv4_attention(q, cache, layer, pages.block_table, pages.kv_lens, cu_q=cu_q, max_q=max_q, window=self.window)
        return self.out(o.flatten(1))

    def extra_repr(self) -> str:
        return f"heads={self.heads}, kv_heads={self.kv_heads}, head_dim={self.head_dim}, window={self.window}"
