"""Plain float64 forms of the 4-bit cache's operators, for the tests: the cached value's definition
(offset + scale * code per token, head and group), norm and rotation, attention. Written from the
formulas on whole tensors; the byte layout is built and read here on its own, one block at a time."""
from __future__ import annotations

import math

import torch

F64 = torch.float64


def quantise(x, group):
    """x [..., D] -> (codes int64 [..., D], scale, offset float64 [..., D / group])."""
    y = x.double().unflatten(-1, (-1, group)).clamp(-65504.0, 65504.0)
    offset = y.amin(-1).half().double()
    scale = ((y.amax(-1) - offset) / 15.0).half().double()
    scale = torch.where(scale > 0, scale, torch.ones_like(scale))
    codes = torch.round((y - offset[..., None]) / scale[..., None]).clamp(0, 15).long()
    return codes.flatten(-2), scale, offset


def value(codes, scale, offset):
    group = codes.shape[-1] // scale.shape[-1]
    return codes.double() * scale.repeat_interleave(group, -1) + offset.repeat_interleave(group, -1)


class PlainCache:
    """Keys and values [sequences][tokens, kv_heads, D] as codes and pairs, and their bytes in pages."""

    def __init__(self, lens, kv_heads, D, group, page_size, *, gen, v_scale=1.0, spare=3, device="cuda"):
        self.lens, self.kv, self.D, self.group, self.page_size = lens, kv_heads, D, group, page_size
        need = [-(-n // page_size) for n in lens]
        self.num_pages = sum(need) + spare
        order = torch.randperm(self.num_pages, generator=torch.Generator().manual_seed(7)).tolist()
        width = max(need + [1]) + 1
        table = torch.full((len(lens), width), 1 << 30, dtype=torch.int32)   # entries past a length are not read
        blk = 16 * (D + 8 * (D // group))
        pool = torch.full((self.num_pages, kv_heads, page_size // 16, blk), 0xFF, dtype=torch.uint8, device=device)
        self.k, self.v = [], []
        for b, n in enumerate(lens):
            pages = [order.pop() for _ in range(need[b])]
            table[b, :need[b]] = torch.tensor(pages, dtype=torch.int32)
            kk = torch.randn((n, kv_heads, D), generator=gen, device=device) * 1.5
            vv = (torch.randn((n, kv_heads, D), generator=gen, device=device) + 0.5) * v_scale
            for which, (x, keep) in enumerate(((kk, self.k), (vv, self.v))):
                codes, scale, offset = quantise(x, group)
                keep.append(value(codes, scale, offset))
                packed = (codes[..., 0::2] | (codes[..., 1::2] << 4)).to(torch.uint8)
                pairs = torch.stack([scale, offset], -1).half().flatten(-2).contiguous().view(torch.uint8)
                for t0 in range(0, n, 16):   # a block of 16 tokens (the last one partly written)
                    m = min(16, n - t0)
                    page, blk_at = pages[t0 // page_size], t0 % page_size // 16
                    at = which * 8 * D
                    pool[page, :, blk_at, at:at + m * D // 2] = packed[t0:t0 + m].transpose(0, 1).flatten(1)
                    at = 16 * D + which * 64 * (D // group)
                    size = 4 * (D // group)
                    pool[page, :, blk_at, at:at + m * size] = pairs[t0:t0 + m].transpose(0, 1).flatten(1)
        self.table = table.to(device)
        self.pool = pool.flatten(-2)[None].contiguous()
        self.kv_lens = torch.tensor(lens, dtype=torch.int32, device=device)

    def slots(self, b, first, n):
        t = torch.arange(first, first + n, device=self.table.device)
        return self.table[b, t // self.page_size].long() * self.page_size + t % self.page_size


def attend(q, k, v, share, scale, window):
    """One sequence: q [m, heads, D], k and v [n, kv, D] -> o [m, heads, D], lse [m, heads], float64."""
    m, H, D = q.shape
    n = k.shape[0]
    pos = torch.arange(n - m, n, device=q.device)[:, None]
    t = torch.arange(n, device=q.device)[None]
    see = t <= pos
    if window:
        see &= t > pos - window
    kk, vv = k.repeat_interleave(share, 1), v.repeat_interleave(share, 1)
    s = torch.einsum("mhd,nhd->hmn", q.double(), kk) * scale
    s = s.masked_fill(~see, -math.inf)
    lse = torch.logsumexp(s, -1) if n else torch.full((H, m), -math.inf, dtype=F64, device=q.device)
    p = torch.where(lse[..., None] > -math.inf, torch.exp(s - lse[..., None]), torch.zeros_like(s))
    return torch.einsum("hmn,nhd->mhd", p, vv), lse.T


def norm_rope(x, w, positions, cos_sin, sections, interleaved, eps):
    """x [T, heads, D] -> float64."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
    rot = cos_sin.shape[1]
    half = rot // 2
    freq = torch.arange(half, device=x.device)
    if sections is None:
        pos = positions[:, None].expand(-1, half)
    else:
        axis = (freq >= sections[0]).long() + (freq >= sections[0] + sections[1]).long()
        pos = positions[axis].T
    cos, sin = cos_sin.double()[pos, freq][:, None], cos_sin.double()[pos, half + freq][:, None]
    ia, ib = (2 * freq, 2 * freq + 1) if interleaved else (freq, half + freq)
    out = x.clone()
    out[..., ia] = x[..., ia] * cos - x[..., ib] * sin
    out[..., ib] = x[..., ib] * cos + x[..., ia] * sin
    return out


def cos_sin_table(n, rot, device="cuda", base=10000.0):
    f = base ** (-torch.arange(0, rot, 2, dtype=F64) / rot)
    a = torch.arange(n, dtype=F64)[:, None] * f
    return torch.cat([a.cos(), a.sin()], -1).float().to(device)
