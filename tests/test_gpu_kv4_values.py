"""kv4_attention on values of every size: small ones, sizes that differ from token to token, groups without spread.

Tolerance of a result: half a unit in the last place of the output; probabilities times value scales (or values and
probabilities) rounded to fp16, 2^-11 of the largest value the row may see; scores in fp32, within 2e-5 of the row's
own bound |q| max |k| scale, which moves the mean by at most that times the largest value. All but the first are
proportional to the values: nothing absolute is lost below fp16's own 2^-25."""
from __future__ import annotations

import math

import pytest
import torch

import w4a16
from kv4_plain import PlainCache, attend, cos_sin_table, value
from w4a16 import KV4Cache, kv4_attention, qk_norm_rope_append

pytestmark = pytest.mark.gpu

HALF_ULP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
F16, BF16 = torch.float16, torch.bfloat16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


@pytest.fixture(autouse=True)
def _no_device_errors():
    yield
    assert w4a16.check_device_errors() == 0


def compare(q, k, v, o, lse, share, window=0):
    """One sequence's rows against float64, each kv head by its own largest value."""
    D = q.shape[2]
    want, wl = attend(q, k, v, share, 1 / math.sqrt(D), window)
    top = (q.double().norm(dim=-1) * k.norm(dim=-1).amax() / math.sqrt(D))[..., None]
    vmax = v.abs().amax((0, 2)).repeat_interleave(share)[:, None]
    tol = HALF_ULP[q.dtype] * want.abs() + (2.0 ** -11 + 2e-5 * (1 + top)) * vmax + (2.0 ** -25 if q.dtype is F16 else 0)
    err = (o.double() - want).abs()
    assert (err <= tol).all(), ((err - tol) / vmax).max().item()
    assert ((lse.double() - wl).abs() <= 2e-5 * (1 + top[..., 0])).all()


@pytest.mark.parametrize("v_scale", [1e-1, 1e-2, 1e-3, 2e-4])
@pytest.mark.parametrize("lens,new,H,KV,D,group", [
    ([8000, 777], [1, 1], 16, 2, 128, 128), ([3000, 90], [1, 1], 8, 2, 128, 64), ([500, 333], [3, 2], 16, 2, 128, 64),
    ([3001], [5], 6, 2, 64, 64), ([400, 150], [130, 70], 64, 8, 128, 128),
])
def test_small_values(v_scale, lens, new, H, KV, D, group):
    for dtype in (F16, BF16):
        g = gen(len(lens) + D)
        c = PlainCache(lens, KV, D, group, 32, gen=g, v_scale=v_scale)
        cache = KV4Cache(1, c.num_pages, KV, D, page_size=32, group_size=group, pool=c.pool)
        heat = 4.0 ** torch.rand((1, H, 1), generator=g, device="cuda")        # flat and peaked heads
        q = (torch.randn((sum(new), H, D), generator=g, device="cuda") * heat).to(dtype)
        cu = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
        o, lse = kv4_attention(q, cache, 0, c.table, c.kv_lens, cu_q=cu, max_q=max(new), return_lse=True)
        first = 0
        for b, m in enumerate(new):
            r = slice(first, first + m)
            compare(q[r], c.k[b], c.v[b], o[r], lse[r], H // KV)
            first += m


def held(cache, n):
    """Keys and values float64 [n, kv, D] of the first n slots, from the pool's bytes."""
    D, G = cache.head_dim, cache.head_dim // cache.group_size
    b = cache.pool[0].unflatten(-1, (-1, 16 * (D + 8 * G)))                   # [pages, kv, blocks, bytes]
    out = []
    for which in (0, 1):
        codes = b[..., which * 8 * D:(which + 1) * 8 * D].unflatten(-1, (16, D // 2))
        codes = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).permute(0, 2, 3, 1, 4).flatten(0, 2)
        at = 16 * D + which * 64 * G
        pairs = b[..., at:at + 64 * G].contiguous().view(torch.float16).unflatten(-1, (16, G, 2))
        pairs = pairs.permute(0, 2, 3, 1, 4, 5).flatten(0, 2).double()
        out.append(value(codes, pairs[..., 0], pairs[..., 1])[:n])
    return out


def appended(k, v, group, fill=0, page=16):
    """A cache of one sequence that holds k and v [n, kv, D], and what it holds in float64."""
    n, KV, D = k.shape
    cache = KV4Cache(1, -(-n // page) + 1, KV, D, page_size=page, group_size=group)
    cache.pool.fill_(fill)
    slots = torch.arange(n, device="cuda")
    qk_norm_rope_append(k.new_empty(n, 0, D), k, v, cache, 0, slots, torch.zeros(n, dtype=torch.int64, device="cuda"),
                        cos_sin_table(1, 8))
    table = torch.arange(cache.num_pages, dtype=torch.int32, device="cuda")[None]
    return cache, table, torch.tensor([n], dtype=torch.int32, device="cuda"), *held(cache, n)


@pytest.mark.parametrize("D,group", [(128, 128), (128, 64), (64, 64)])
@pytest.mark.parametrize("order", ["rising", "falling", "one"])
def test_values_whose_size_changes_along_the_sequence(D, group, order):
    """Small values keep their bits for rows that see no others (a window, or a draft's earlier rows)."""
    g = gen(D)
    n, KV, share = 900, 2, 4
    size = torch.ones(n, device="cuda") * 1e-3
    if order == "one":
        size[n - 1] = 3000.0
    else:
        size = 10.0 ** torch.linspace(-4, 3, n, device="cuda")
        if order == "falling":
            size = size.flip(0)
    k = torch.randn((n, KV, D), generator=g, device="cuda").half()
    v = (torch.randn((n, KV, D), generator=g, device="cuda") * size[:, None, None]).half()
    cache, table, lens, kd, vd = appended(k, v, group)
    q = torch.randn((2, KV * share, D), generator=g, device="cuda").half()
    cu = torch.tensor([0, 2], dtype=torch.int32, device="cuda")
    for window in (0, 50):
        o, lse = kv4_attention(q, cache, 0, table, lens, cu_q=cu, max_q=2, window=window, return_lse=True)
        for i in (0, 1):
            to = n - 1 + i
            lo = max(0, to - window) if window else 0
            compare(q[i:i + 1], kd[lo:to], vd[lo:to], o[i:i + 1], lse[i:i + 1], share)


def test_what_lies_beside_the_tokens_changes_nothing():
    g = gen(3)
    for D, group in ((128, 128), (128, 64), (64, 64)):
        for n in (1, 21, 50):
            k = torch.randn((n, 2, D), generator=g, device="cuda").half()
            v = (torch.randn((n, 2, D), generator=g, device="cuda") * 1e-3).half()
            q = torch.randn((1, 8, D), generator=g, device="cuda").half()
            outs = []
            for fill in (0, 0x3C, 0x7B, 0xFB, 0xFF):      # scales of 0, 1.06, 61e3, -61e3 and NaN
                cache, table, lens, _, _ = appended(k, v, group, fill, page=64)
                outs.append(kv4_attention(q, cache, 0, table, lens, return_lse=True))
            for o, lse in outs[1:]:
                assert torch.equal(o, outs[0][0]) and torch.equal(lse, outs[0][1])


@pytest.mark.parametrize("v_scale", [2e-5, 1e-4, 1e-3, 1e-2, 1.0, 100.0, 3000.0])
@pytest.mark.parametrize("n,new,H,KV,D,group", [
    (8000, 1, 16, 2, 128, 128), (3000, 1, 8, 2, 128, 64), (2000, 3, 16, 2, 128, 64), (3001, 5, 6, 2, 64, 64),
    (900, 130, 64, 8, 128, 128),
])
def test_values_of_all_sizes_are_equally_exact(v_scale, n, new, H, KV, D, group):
    """A row's error in the root mean square of its channels: the roundings of its tokens are independent, so they add up
    as squares. Each token's p v is off by less than 2^-11 of p times the largest value in that mean (two roundings of
    2^-11 / sqrt(12)), and p by 2e-6 of it for a unit of |q| max |k| scale; then bf16's half unit."""
    g = gen(n + D)
    k = torch.randn((n, KV, D), generator=g, device="cuda").bfloat16()
    v = (torch.randn((n, KV, D), generator=g, device="cuda") * v_scale).bfloat16()
    cache, table, lens, kd, vd = appended(k, v, group, page=64)
    q = (torch.randn((new, H, D), generator=g, device="cuda") * 1.5).bfloat16()
    got = kv4_attention(q, cache, 0, table, lens).double()
    want, lse = attend(q, kd, vd, H // KV, 1 / math.sqrt(D), 0)
    _, twice = attend(q, kd, vd, H // KV, 2 / math.sqrt(D), 0)      # of p^2: the same keys at twice the scale
    spread = torch.exp(0.5 * twice - lse)
    top = q.double().norm(dim=-1) * kd.norm(dim=-1).amax() / math.sqrt(D)
    rms = (got - want).square().mean(-1).sqrt()
    tol = (2.0 ** -11 + 2e-6 * (1 + top)) * spread * vd.abs().amax() + 2.0 ** -8 * want.square().mean(-1).sqrt()
    assert (rms <= tol).all(), (rms / tol).max().item()


@pytest.mark.parametrize("D,group", [(128, 128), (128, 64), (64, 64)])
@pytest.mark.parametrize("new,share", [(1, 4), (3, 4), (70, 8)])
def test_groups_without_spread(D, group, new, share):
    """Values that are one number each group: zero, small, large, and one per token; beside them ordinary ones."""
    g = gen(D + new)
    n, KV = 517, 16
    k = torch.randn((n, KV, D), generator=g, device="cuda").half()
    v = torch.randn((n, KV, D), generator=g, device="cuda").half()
    v[:, 0] = 0
    v[:, 1] = 1e-3
    v[:, 2] = 300.0
    v[:, 3] = (torch.randn((n, 1), generator=g, device="cuda") * 1e-2).half()
    v[:, 4, :64] = 0
    v[::3, 5] = 0                                   # some tokens
    v[:, 6] = (v[:, 6].float() * 1e-3).half()
    v[::3, 6] = 1e-3                                # among small ones
    cache, table, lens, kd, vd = appended(k, v, group)
    q = (torch.randn((new, KV * share, D), generator=g, device="cuda") * 2).half()
    o, lse = kv4_attention(q, cache, 0, table, lens, return_lse=True)
    compare(q, kd, vd, o, lse, share)
    o = o.unflatten(1, (KV, share)).double()
    assert (o[:, 0] == 0).all()
    if group == 64:
        assert (o[:, 4, :, :64] == 0).all()
    for head in (1, 2):                             # a mean of one number: fp32's and the output's roundings
        assert ((o[:, head] - vd[0, head, 0]).abs() <= (2.0 ** -11 + 1e-5) * vd[0, head, 0]).all()


@pytest.mark.parametrize("token", [3, 40, 66])
@pytest.mark.parametrize("new,share", [(1, 4), (2, 6), (70, 8)])
def test_a_nan_of_vanishing_weight_is_still_one(token, new, share):
    """The weight 2^-350 of a NaN value is zero in fp32, in a whole tile as in one that the sequence ends in."""
    n, KV, D = 70, 16, 64
    g = gen(token)
    k = torch.randn((n, KV, D), generator=g, device="cuda").half()
    v = torch.randn((n, KV, D), generator=g, device="cuda").half()
    k[token], v[token] = -10, float("nan")
    cache, table, lens, _, _ = appended(k, v, 64)
    q = torch.full((new, KV * share, D), 3.0, device="cuda", dtype=F16)
    o = kv4_attention(q, cache, 0, table, lens)
    sees = torch.arange(n - new, n, device="cuda") >= token
    assert o[sees].isnan().all() and o[~sees].isfinite().all()
