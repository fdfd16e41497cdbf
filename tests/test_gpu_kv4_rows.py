"""kv4_attention computes each query row as if it were alone: a row of another magnitude, or with an infinity
or NaN in it, beside rows of ordinary ones, in every kernel and tile.

Tolerance of a row, from its own numbers: half a unit in the last place of the output; probabilities (times value
scales, or values beside them) rounded to fp16: 2^-11 of the largest value; scores in fp32, and the query's
channels kept to 2^-24 of the row's largest: within 2e-5 of the row's own bound on its scores, |q| max |k| scale,
which moves the mean by at most that times the spread of the values."""
from __future__ import annotations

import math

import pytest
import torch

import w4a16
from kv4_plain import PlainCache, attend
from w4a16 import KV4Cache, kv4_attention

pytestmark = pytest.mark.gpu

HALF_ULP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
F16, BF16 = torch.float16, torch.bfloat16
FACTORS = [1e-6, 1e-3, 2.0 ** 10, 2.0 ** 14, 6e4, 1e8, 1e30, math.inf, -math.inf, math.nan]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def check_rows(c, q, new, o, lse, skip=None, scale=None, window=0):
    """Each row of q [T, heads, D] against the float64 form within the tolerance of its own scores; rows marked in
    `skip` [T, heads] are left out."""
    T, H, D = q.shape
    sc = 1 / math.sqrt(D) if scale is None else scale
    first = 0
    for b, (n, m) in enumerate(zip(c.lens, new)):
        if m == 0 or n == 0:
            first += m
            continue
        rows = slice(first, first + m)
        first += m
        qq = q[rows].double()
        keep = torch.ones((m, H), dtype=torch.bool, device="cuda") if skip is None else ~skip[rows]
        want, wl = attend(torch.where(keep[..., None], qq, torch.zeros_like(qq)), c.k[b], c.v[b], H // c.kv, sc, window)
        top = qq.norm(dim=-1) * c.k[b].norm(dim=-1).amax() * abs(sc)
        vmax = c.v[b].abs().amax()
        tol = HALF_ULP[q.dtype] * want.abs() + (2.0 ** -11 * vmax + 2e-5 * (1 + top) * vmax)[..., None]
        err = (o[rows].double() - want).abs()
        assert ((err <= tol) | ~keep[..., None]).all(), (b, (err / tol)[keep].max().item())
        seen = keep & (wl > -math.inf)
        assert ((lse[rows].double() - wl).abs() <= 2e-5 * (1 + top))[seen].all(), (b, (lse[rows].double() - wl)[seen].abs().max())


def attend_with_one_row(factor, lens, new, H, KV, D, group, dtype, token, head):
    """One row's largest channel (or, for a finite factor, the whole row) set apart."""
    g = gen(H + D)
    c = PlainCache(lens, KV, D, group, 32, gen=g)
    cache = KV4Cache(1, c.num_pages, KV, D, page_size=32, group_size=group, pool=c.pool)
    q = torch.randn((sum(new), H, D), generator=g, device="cuda").clamp(-1, 1).to(dtype)
    if math.isfinite(factor):
        q[token, head] *= factor
    else:
        q[token, head, 5] = factor
    cu = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
    o, lse = kv4_attention(q, cache, 0, c.table, c.kv_lens, cu_q=cu, max_q=max(new), return_lse=True)
    skip = torch.zeros(q.shape[:2], dtype=torch.bool, device="cuda")
    skip[token, head] = not math.isfinite(factor)
    check_rows(c, q, new, o, lse, skip)
    if math.isnan(factor):
        assert o[token, head].isnan().all()
    assert w4a16.check_device_errors() == 0


@pytest.mark.parametrize("factor", FACTORS)
@pytest.mark.parametrize("lens,new,H,KV,D,group", [
    ([777, 60], [1, 1], 16, 2, 128, 128),         # tiles of eight rows
    ([300, 777], [3, 2], 16, 2, 128, 64),         # of sixteen
    ([150, 40], [4, 9], 6, 2, 64, 64),
])
def test_single_and_drafted_tokens(factor, lens, new, H, KV, D, group):
    if abs(factor) <= 65504 or not math.isfinite(factor):
        attend_with_one_row(factor, lens, new, H, KV, D, group, F16, 0, 3)
    attend_with_one_row(factor, lens, new, H, KV, D, group, BF16, sum(new) - 1, H - 1)


@pytest.mark.parametrize("magnitude", [1e5, 1e8, 1e12, 1e30])
@pytest.mark.parametrize("lens,new,H,KV,D,group", [
    ([400, 150], [130, 70], 64, 8, 128, 128), ([300, 140], [140, 66], 64, 8, 128, 64), ([290, 290], [131, 100], 64, 8, 64, 64),
    ([777, 60], [1, 1], 16, 2, 128, 128),
])
def test_queries_whose_scores_pass_the_resolution_of_fp32(magnitude, lens, new, H, KV, D, group):
    """A result is then some mean of the values of the tokens whose scores are largest up to that resolution, and
    finite: 2^-11 of the values apart (each rounded to fp16), and half a unit of bf16."""
    g = gen(7)
    c = PlainCache(lens, KV, D, group, 32, gen=g)
    cache = KV4Cache(1, c.num_pages, KV, D, page_size=32, group_size=group, pool=c.pool)
    q = (torch.randn((sum(new), H, D), generator=g, device="cuda") * magnitude).bfloat16()
    cu = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
    o, lse = kv4_attention(q, cache, 0, c.table, c.kv_lens, cu_q=cu, max_q=max(new), return_lse=True)
    assert o.isfinite().all() and lse.isfinite().all()
    first = 0
    for b, (n, m) in enumerate(zip(lens, new)):
        qq = q[first:first + m].double()
        vmax = c.v[b].abs().amax()
        got = o[first:first + m].double()
        assert (got.abs() <= vmax * (1 + 2.0 ** -8 + 2.0 ** -11)).all()
        _, wl = attend(qq, c.k[b], c.v[b], H // KV, 1 / math.sqrt(D), 0)
        top = qq.norm(dim=-1) * c.k[b].norm(dim=-1).amax() / math.sqrt(D)
        assert ((lse[first:first + m].double() - wl).abs() <= 2e-5 * (1 + top)).all()
        first += m
    assert w4a16.check_device_errors() == 0


@pytest.mark.parametrize("factor", FACTORS)
@pytest.mark.parametrize("lens,new,H,KV,D,group", [
    ([400, 150], [130, 70], 64, 8, 128, 128),     # more than 8192 rows x kv heads x sequences, and than 64 rows
    ([300, 140], [140, 66], 64, 8, 128, 64),
    ([290, 290], [131, 100], 64, 8, 64, 64),
])
def test_prompts(factor, lens, new, H, KV, D, group):
    assert max(new) * (H // KV) * KV * len(new) > 8192
    if abs(factor) <= 65504 or not math.isfinite(factor):
        attend_with_one_row(factor, lens, new, H, KV, D, group, F16, 37, 3)
    attend_with_one_row(factor, lens, new, H, KV, D, group, BF16, sum(new) - 1, H - 1)
    attend_with_one_row(factor, lens, new, H, KV, D, group, BF16, 0, 9)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_rows_of_all_magnitudes_in_one_prompt(dtype):
    """Every row of its own magnitude, rows of zeros among them, windows and a last tile of few rows."""
    g = gen(4)
    new, H, KV, D = [150, 35], 64, 8, 128
    c = PlainCache([333, 35], KV, D, D, 32, gen=g)
    cache = KV4Cache(1, c.num_pages, KV, D, page_size=32, pool=c.pool)
    span = 14 if dtype is F16 else 40
    q = torch.randn((sum(new), H, D), generator=g, device="cuda").clamp(-1, 1)
    q *= 2.0 ** torch.randint(-span, span + 1, (sum(new), H, 1), generator=g, device="cuda").float()
    q[::7, ::3] = 0
    q = q.to(dtype)
    cu = torch.tensor([0, 150, 185], dtype=torch.int32, device="cuda")
    for window in (0, 40):
        o, lse = kv4_attention(q, cache, 0, c.table, c.kv_lens, cu_q=cu, max_q=150, window=window, return_lse=True)
        check_rows(c, q, new, o, lse, window=window)
    assert w4a16.check_device_errors() == 0
