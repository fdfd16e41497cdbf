"""The 4-bit paged cache on the GPU: query/key preparation, quantised append and read-back, attention
and page management against plain float64 forms (kv4_plain.py).

Tolerances, from the arithmetic: a result rounded once to T is within half a unit in the last place,
HALF_ULP[T] * |y|; fp32 sums of at most 128 products add less than 2e-5 of the head's largest value.
Attention rounds each probability times its value scale s to fp16 (2^-11 relative, 2^-25 absolute
below 2^-14) against codes centred on 7.5: at most (2^-11 * s + n * 2^-25) * 7.5 in the weighted mean
over n tokens; its fp32 scores are within 2e-5 of the largest, which moves the mean by at most that
times the spread of the values. (Prompts round probabilities and values instead, each to within 2^-11
of a value, in either direction: the same bound, met in the mean.)"""
from __future__ import annotations

import math

import pytest
import torch

import w4a16
from kv4_plain import PlainCache, attend, cos_sin_table, norm_rope, quantise, value
from w4a16 import (KV4Cache, KV4Pages, W4A16Error, kv4_attention, kv4_compact, kv4_copy_pages, kv4_fork, kv4_gather,
                   kv4_release, kv4_reserve, qk_norm_rope, qk_norm_rope_append)

pytestmark = pytest.mark.gpu

HALF_ULP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
F16, BF16 = torch.float16, torch.bfloat16


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(g, *shape, dtype=F16, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


@pytest.fixture(autouse=True)
def _no_device_errors():
    yield
    assert w4a16.check_device_errors() == 0


# ------------------------------------------------------------------------- norm and rotation
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("T,H,KV,D,rot,axes,pairs,norm,layout", [
    (1, 32, 8, 128, 128, 1, False, True, "fused"),
    (3, 28, 4, 128, 96, 3, True, True, "fused"),
    (33, 5, 1, 64, 64, 1, False, True, "dense"),
    (7, 16, 16, 64, 16, 3, False, False, "heads first"),
    (130, 8, 2, 128, 8, 1, True, True, "odd"),
    (2, 1, 1, 128, 120, 1, False, True, "odd"),
    (5, 0, 3, 64, 32, 1, False, True, "dense"),
    (0, 8, 2, 64, 64, 1, False, True, "dense"),
])
def test_qk_norm_rope(T, H, KV, D, rot, axes, pairs, norm, layout, dtype):
    g = gen(T + D)
    if layout == "fused":
        x = rand(g, T, H + 2 * KV, D, dtype=dtype, scale=3.0)
        q, k = x[:, :H], x[:, H:H + KV]
    elif layout == "heads first":
        q, k = rand(g, H, T, D, dtype=dtype).transpose(0, 1), rand(g, KV, T, D, dtype=dtype).transpose(0, 1)
    elif layout == "odd":     # rows that start on any 2-byte boundary
        x = rand(g, T, (H + KV) * D + 1, dtype=dtype)
        q, k = x[:, 1:1 + H * D].unflatten(1, (H, D)), x[:, 1 + H * D:].unflatten(1, (KV, D))
    else:
        q, k = rand(g, T, H, D, dtype=dtype), rand(g, T, KV, D, dtype=dtype)
    wq = rand(g, D, dtype=dtype if T != 33 else torch.float32) + 1 if norm else None
    wk = rand(g, D, dtype=dtype if T != 33 else torch.float32) + 1 if norm else None
    third = rot // 6
    sections = None if axes == 1 else (rot // 2 - 2 * third, third, third)
    pos = torch.randint(0, 500, (T,) if axes == 1 else (3, T), generator=g, device="cuda")
    cs = cos_sin_table(500, rot)
    qo, ko = qk_norm_rope(q, k, pos, cs, wq, wk, 1e-5, sections=sections, interleaved=pairs)
    for x, w, got in ((q, wq, qo), (k, wk, ko)):
        assert got.dtype == dtype and got.shape == x.shape and got.is_contiguous()
        want = norm_rope(x, w, pos, cs, sections, pairs, 1e-5)
        if want.numel():
            tol = HALF_ULP[dtype] * want.abs() + 2e-5 * want.abs().amax() + 2.0 ** -24
            assert ((got.double() - want).abs() <= tol).all()


def test_qk_norm_rope_infinite_and_nan_stay_in_their_head():
    g = gen(1)
    q, k = rand(g, 4, 4, 128), rand(g, 4, 2, 128)
    pos, cs = torch.arange(4, device="cuda"), cos_sin_table(8, 64)
    w = torch.ones(128, device="cuda", dtype=F16)
    clean = qk_norm_rope(q, k, pos, cs, w, w)
    q[1, 2, 5], k[3, 1, 100] = float("nan"), float("inf")
    dirty = qk_norm_rope(q, k, pos, cs, w, w)
    keep = torch.ones(4, 4, dtype=torch.bool, device="cuda")
    keep[1, 2] = False
    assert torch.equal(clean[0][keep], dirty[0][keep]) and dirty[0][1, 2].isnan().all()
    keep = torch.ones(4, 2, dtype=torch.bool, device="cuda")
    keep[3, 1] = False
    assert torch.equal(clean[1][keep], dirty[1][keep]) and dirty[1][3, 1].isnan().any()


# -------------------------------------------------------------------------- append and gather
def close_to_cached(got, want, group, dtype):
    """`got` (as read back) against what 64 bits say the cache holds for `want`. A code may differ by one where the
    exact value lies within 1e-3 steps of the middle between two codes (fp32 arithmetic); the pair may differ by
    one fp16 rounding where the exact minimum or maximum lies that near to one."""
    codes, scale, offset = quantise(want, group)
    held = value(codes, scale, offset)
    steps = (want.double().clamp(-65504, 65504) - offset.repeat_interleave(group, -1)) / scale.repeat_interleave(group, -1)
    tie = ((steps - torch.floor(steps)) - 0.5).abs() < 1e-3
    err = (got.double() - held).abs()
    s = scale.repeat_interleave(group, -1)
    pair = 2.0 ** -10 * (16 * s + offset.abs().repeat_interleave(group, -1))     # one unit of scale and of offset
    tol = HALF_ULP[dtype] * held.abs() + 2.0 ** -24
    ok = (err <= tol) | (err <= tol + pair) & (err > tol)
    assert (ok | tie & (err <= s + tol + pair)).all()
    if err.numel():
        assert (err <= tol).double().mean() > 0.98     # other roundings are rare


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("T,H,KV,D,group,page,rot", [
    (1, 32, 8, 128, 128, 64, 128), (2, 32, 8, 128, 128, 64, 128), (37, 28, 4, 128, 64, 16, 96), (100, 6, 3, 64, 64, 48, 64), (130, 0, 1, 64, 64, 128, 32),
    (64, 8, 1, 128, 128, 32, 64),
])
def test_append_then_gather(T, H, KV, D, group, page, rot, dtype):
    g = gen(T)
    x = rand(g, T, H + 2 * KV, D, dtype=dtype, scale=2.0)
    q, k, v = x[:, :H], x[:, H:H + KV], x[:, H + KV:]
    wq, wk = rand(g, D, dtype=dtype) * 0.1 + 1, rand(g, D, dtype=dtype) * 0.1 + 1
    pages = -(-T // page) + 4
    cache = KV4Cache(2, pages, KV, D, page_size=page, group_size=group)
    cache.pool.fill_(0xA5)
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:T]
    slots[::5] = -1
    cs = cos_sin_table(700, rot)
    pos = torch.randint(0, 700, (T,), generator=g, device="cuda")
    qo = qk_norm_rope_append(q, k, v, cache, 1, slots, pos, cs, wq, wk)
    assert torch.equal(qo, qk_norm_rope(q, k, pos, cs, wq, wk)[0])
    assert (cache.pool[0] == 0xA5).all()                      # the other layer
    keep = slots >= 0
    for out_dtype in (F16, BF16):
        kv = kv4_gather(cache, 1, slots, out_dtype)
        assert (kv[:, ~keep] == 0).all()
        close_to_cached(kv[0][keep], norm_rope(k, wk, pos, cs, None, False, 1e-6)[keep], group, out_dtype)
        close_to_cached(kv[1][keep], v.double()[keep], group, out_dtype)
    # bytes of tokens that were not written stay: each token has its own nibbles and pairs
    written = int(keep.sum())
    per_token = D + 8 * (D // group)
    assert (cache.pool[1] != 0xA5).sum() <= written * KV * per_token


def test_append_extremes():
    """Constant groups, groups with an infinity or NaN, values past fp16's range."""
    T, KV, D = 8, 1, 64
    k = torch.zeros(T, KV, D, device="cuda", dtype=BF16)
    v = torch.randn(T, KV, D, generator=gen(3), device="cuda").to(BF16)
    k[1], k[2] = 3.0, -1e-9
    v[3, 0, 7], v[4, 0, 63], v[5, 0, 0] = float("nan"), float("-inf"), 1e30
    v[6] *= 1e-12
    cache = KV4Cache(1, 2, KV, D, page_size=16)
    slots = torch.arange(T, device="cuda") + 3
    cs = cos_sin_table(4, 8)
    qk_norm_rope_append(torch.empty(T, 0, D, device="cuda", dtype=BF16), k, v, cache, 0, slots,
                        torch.zeros(T, dtype=torch.int64, device="cuda"), cs)
    kv = kv4_gather(cache, 0, slots, F16).double()
    assert (kv[0, 0] == 0).all() and (kv[0, 1] == 3).all() and (kv[0, 2].abs() <= 2.0 ** -24).all()
    assert kv[1, 3].isnan().all() and kv[1, 4].isnan().all() and kv[1, [0, 1, 2, 5, 6, 7]].isfinite().all()
    assert abs(kv[1, 5].max() - 65504) <= 2.0 ** -10 * 65504 and (kv[1, 6].abs() <= 2.0 ** -24).all()


# --------------------------------------------------------------------------------- attention
def check_attention(lens, new, H, KV, D, group, page, dtype, window=0, *, q_scale=1.0, v_scale=1.0, seed=0, scale=None,
                    strided=False, uniform=False, max_q=None):
    g = gen(seed)
    c = PlainCache(lens, KV, D, group, page, gen=g, v_scale=v_scale)
    cache = KV4Cache(1, c.num_pages, KV, D, page_size=page, group_size=group, pool=c.pool)
    T = sum(new)
    heat = 4.0 ** torch.rand((1, H, 1), generator=g, device="cuda")
    if strided:
        q = rand(g, H, T, D + 8, dtype=dtype, scale=q_scale).transpose(0, 1)[..., :D]
    else:
        q = rand(g, T, H, D, dtype=dtype, scale=q_scale)
    q = q.mul_(heat.to(dtype))
    cu = torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int32, device="cuda")
    kw = {} if uniform else {"cu_q": cu, "max_q": max(new) if max_q is None else max_q}
    o, lse = kv4_attention(q, cache, 0, c.table, c.kv_lens, scale=scale, window=window, return_lse=True, **kw)
    again, lse2 = kv4_attention(q, cache, 0, c.table, c.kv_lens, scale=scale, window=window, return_lse=True, **kw)
    assert torch.equal(o, again) and torch.equal(lse, lse2), "two calls on the same inputs differ"
    assert o.dtype == dtype and o.shape == (T, H, D) and lse.dtype == torch.float32
    sc = 1 / math.sqrt(D) if scale is None else scale
    first = 0
    for b, (n, m) in enumerate(zip(lens, new)):
        if m == 0:
            continue
        qq = q[first:first + m]
        want, wl = attend(qq, c.k[b], c.v[b], H // KV, sc, window)
        got, gl = o[first:first + m].double(), lse[first:first + m].double()
        first += m
        empty = wl == -math.inf
        assert torch.equal(gl == -math.inf, empty) and (got[empty] == 0).all()
        if n == 0:
            continue
        top = (qq.double().norm(dim=-1).amax() * c.k[b].norm(dim=-1).amax() * abs(sc)).item()   # bounds the scores
        vmax = c.v[b].abs().amax().item()
        s_max = 2 * vmax / 15
        tol = HALF_ULP[dtype] * want.abs() + (2.0 ** -11 * s_max + n * 2.0 ** -25) * 7.5 + 2e-5 * (1 + top) * vmax
        assert got.isfinite().all()
        worst = ((got - want).abs() - tol).max().item()
        assert worst <= 0, f"sequence {b}: {worst} over the tolerance {tol.max().item()}"
        assert ((gl - wl)[~empty].abs() <= 2e-5 * (1 + top)).all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D,group", [(128, 128), (128, 64), (64, 64)])
@pytest.mark.parametrize("page", [16, 48, 64, 128])
def test_attention_single_tokens(D, group, page, dtype):
    check_attention([1, 15, 16, 17, 0, 63, 64, 65, 200, 777], [1] * 10, 8, 2, D, group, page, dtype, uniform=True)


@pytest.mark.parametrize("H,KV", [(1, 1), (7, 1), (28, 4), (16, 16), (32, 1), (12, 4), (48, 1), (6, 3)])
def test_attention_head_layouts(H, KV):
    check_attention([300, 33], [1, 1], H, KV, 128, 128, 64, F16, seed=H)
    check_attention([300, 33, 5], [3, 1, 5], H, KV, 64, 64, 32, BF16, seed=H)


@pytest.mark.parametrize("new", [[2, 1, 4], [5, 5, 5], [1, 40, 7], [130, 1, 0], [33, 300, 129], [0, 257, 1]])
@pytest.mark.parametrize("window", [0, 1, 30, 5000])
def test_attention_several_new_tokens(new, window):
    check_attention([150, 300, 129], new, 8, 2, 128, 128, 64, F16, window, seed=sum(new))
    check_attention([130, 1301, 700], new, 4, 2, 64, 64, 16, BF16, window, seed=sum(new))


@pytest.mark.parametrize("new", [[6, 200], [1, 1], [40, 9]])
def test_attention_more_new_tokens_than_cached(new):
    """Queries before the sequence's first cached token, and a sequence with none, see nothing."""
    check_attention([4, 0], new, 8, 4, 128, 64, 32, F16)
    check_attention([0, 17], new, 8, 8, 64, 64, 16, BF16)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_attention_long(dtype):
    check_attention([20011, 3], [1, 1], 8, 1, 128, 128, 64, dtype, uniform=True)
    check_attention([9001, 12000], [1, 4], 32, 4, 128, 64, 16, dtype)
    check_attention([9001], [1], 16, 16, 64, 64, 32, dtype, window=4097)


def test_attention_many_sequences():
    lens = [(37 * i * i + 11 * i) % 400 for i in range(150)]
    check_attention(lens, [1] * 150, 8, 2, 128, 128, 32, F16, uniform=True)
    check_attention(lens, [1 + i % 3 for i in range(150)], 4, 4, 64, 64, 16, BF16)


def test_attention_prompt_lengths():
    for n in (127, 128, 129, 255, 257, 640):
        check_attention([n], [n], 8, 2, 128, 128, 64, F16, seed=n)
    check_attention([1500, 900], [700, 513], 16, 2, 128, 64, 128, BF16)
    check_attention([1500, 900], [700, 513], 7, 7, 64, 64, 16, F16, window=100)


def test_attention_value_and_query_ranges():
    """Queries beyond fp16's range (bf16), tiny and huge values, scores that grow along the sequence."""
    check_attention([300, 70], [1, 1], 8, 2, 128, 128, 64, BF16, q_scale=3e5, scale=1e-6)
    check_attention([300, 70], [1, 60], 8, 2, 128, 128, 64, BF16, q_scale=3e5, scale=1e-6)
    check_attention([300, 70], [1, 60], 8, 2, 128, 64, 64, F16, q_scale=1e-3, scale=30.0)
    check_attention([300, 70], [1, 1], 8, 2, 64, 64, 64, F16, v_scale=2000.0)
    check_attention([300, 200], [1, 90], 8, 2, 128, 128, 64, BF16, v_scale=9000.0)


def test_attention_strides_streams_and_out():
    check_attention([100, 300], [1, 70], 8, 2, 128, 128, 64, F16, strided=True)
    check_attention([100, 300], [2, 3], 8, 2, 64, 64, 64, BF16, strided=True, max_q=90)
    g = gen(5)
    c = PlainCache([400, 90], 2, 128, 128, 64, gen=g)
    cache = KV4Cache(1, c.num_pages, 2, 128, pool=c.pool)
    q = rand(g, 2, 8, 128)
    want = kv4_attention(q, cache, 0, c.table, c.kv_lens)
    out = torch.empty_like(want)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        assert kv4_attention(q, cache, 0, c.table, c.kv_lens, out=out) is out
    side.synchronize()
    assert torch.equal(out, want)
    # a captured call replays on new lengths and queries
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv4_attention(q, cache, 0, c.table, c.kv_lens, out=out)
    q.copy_(rand(g, 2, 8, 128))
    c.kv_lens.copy_(torch.tensor([123, 0], device="cuda"))
    graph.replay()
    assert torch.equal(out, kv4_attention(q, cache, 0, c.table, c.kv_lens)) and (out[1] == 0).all()


def test_attention_sees_a_nan_it_attends_to_and_no_other():
    g = gen(9)
    c = PlainCache([40, 40], 1, 64, 64, 16, gen=g)
    cache = KV4Cache(1, c.num_pages, 1, 64, page_size=16, pool=c.pool)
    k = torch.full((1, 1, 64), float("nan"), device="cuda", dtype=F16)
    qk_norm_rope_append(torch.empty(1, 0, 64, device="cuda", dtype=F16), k, k, cache, 0, c.slots(0, 20, 1),
                        torch.zeros(1, dtype=torch.int64, device="cuda"), cos_sin_table(1, 8))
    q = rand(g, 2, 2, 64)
    o = kv4_attention(q, cache, 0, c.table, c.kv_lens)
    assert o[0].isnan().all() and o[1].isfinite().all()
    o = kv4_attention(q, cache, 0, c.table, c.kv_lens, window=19)
    assert o.isfinite().all()


def test_decode_step_by_step_is_the_prompt_at_once():
    """Appending and attending token by token gives the prompt's attention (to the roundings of P)."""
    g = gen(11)
    T, H, KV, D = 70, 8, 2, 128
    x = rand(g, T, H + 2 * KV, D)
    q, k, v = x[:, :H], x[:, H:H + KV], x[:, H + KV:]
    w = torch.ones(D, device="cuda", dtype=F16)
    cs, pos = cos_sin_table(T, D), torch.arange(T, device="cuda")
    cache = KV4Cache(1, 8, KV, D, page_size=16)
    pages = KV4Pages.empty(cache, 1, 8)
    row = torch.zeros(1, dtype=torch.int32, device="cuda")
    steps = []
    for t in range(T):
        assert int(kv4_reserve(pages, row, torch.tensor([t + 1], dtype=torch.int32, device="cuda"))) == 1
        slot = pages.block_table[0, t // 16].long()[None] * 16 + t % 16
        qo = qk_norm_rope_append(q[t:t + 1], k[t:t + 1], v[t:t + 1], cache, 0, slot, pos[t:t + 1], cs, w, w)
        steps.append(kv4_attention(qo, cache, 0, pages.block_table, pages.kv_lens))
    qo, _ = qk_norm_rope(q, k, pos, cs, w, w)
    whole = kv4_attention(qo, cache, 0, pages.block_table, pages.kv_lens)
    assert torch.allclose(torch.cat(steps).float(), whole.float(), rtol=2.0 ** -9, atol=2.0 ** -9)


# ------------------------------------------------------------------------------ page management
class Model:
    """Reference counts, tables and page contents in Python."""

    def __init__(self, pages, rows, width, page_size):
        self.refs, self.ps, self.width = [0] * pages, page_size, width
        self.table, self.lens = [[-1] * width for _ in range(rows)], [0] * rows
        self.data = list(range(1000, 1000 + pages))     # what a page holds

    def free(self):
        return [i for i, r in enumerate(self.refs) if r == 0]

    def held(self, n):
        return -(-n // self.ps)

    def reserve(self, rows, lens):
        free, asked, ok = self.free(), 0, []
        for r, n in zip(rows, lens):
            have, want = self.held(self.lens[r]), self.held(n)
            if n < self.lens[r] or want > self.width:
                ok.append(0)
                continue
            start, asked = asked, asked + want - have
            if want > have and asked > len(free):
                ok.append(0)
                continue
            for c in range(have, want):
                page = free[start + c - have]
                self.table[r][c], self.refs[page] = page, 1
            self.lens[r] = n
            ok.append(1)
        return ok

    def fork(self, parents, children):
        free, asked, ok, copies = self.free(), 0, [], []
        for a, c in zip(parents, children):
            n = self.lens[a]
            row = self.table[a][:self.held(n)]
            good = 1
            if n % self.ps:
                if asked < len(free):
                    copies.append((row[-1], free[asked]))
                    row[-1] = free[asked]
                else:
                    good = 0
                asked += 1
            ok.append(good)
            row = row if good else []
            for p in row:
                self.refs[p] += 1
            self.table[c] = row + [-1] * (self.width - len(row))
            self.lens[c] = n if good else 0
        for s, d in copies:
            self.data[d] = self.data[s]
        return ok

    def release(self, rows):
        for r in rows:
            for p in self.table[r]:
                if p >= 0:
                    self.refs[p] -= 1
            self.table[r], self.lens[r] = [-1] * self.width, 0

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        holes = [i for i in range(live) if self.refs[i] == 0]
        movers = [i for i in range(live, len(self.refs)) if self.refs[i] > 0]
        to = dict(zip(movers, holes))
        for s, d in to.items():
            self.refs[d], self.refs[s], self.data[d] = self.refs[s], 0, self.data[s]
        self.table = [[to.get(p, p) for p in row] for row in self.table]

    def check(self, pages, cache):
        assert pages.refs.tolist() == self.refs
        assert pages.block_table.tolist() == self.table
        assert pages.kv_lens.tolist() == self.lens
        for p in {p for row in self.table for p in row if p >= 0}:
            for layer in range(cache.num_layers):
                page = cache.pool[layer, p]
                want = stamp(self.data[p], layer, page)
                assert torch.equal(page, want), (p, layer)


def stamp(what, layer, like):
    n = like.numel()
    return ((torch.arange(n, device="cuda") * 7 + what * 31 + layer * 13 + (torch.arange(n, device="cuda") >> 8)) % 251
            ).to(torch.uint8).view(like.shape)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("num_pages,rows,width,page,layers,kv,D", [
    (40, 12, 9, 16, 3, 2, 64), (1500, 30, 80, 32, 2, 1, 128), (2100, 9, 300, 16, 1, 1, 64), (7, 5, 4, 48, 2, 3, 64),
])
def test_pages_against_a_model(num_pages, rows, width, page, layers, kv, D):
    import random
    r = random.Random(num_pages)
    cache = KV4Cache(layers, num_pages, kv, D, page_size=page)
    m = Model(num_pages, rows, width, page)
    for p in range(num_pages):
        for layer in range(layers):
            cache.pool[layer, p] = stamp(m.data[p], layer, cache.pool[layer, p])
    pages = KV4Pages.empty(cache, rows, width)
    refused = 0
    for step in range(40):
        op = r.choice(["reserve", "reserve", "fork", "release", "compact"])
        if op == "reserve":
            who = r.sample(range(rows), r.randint(1, rows))
            want = [max(0, m.lens[x] + r.choice([0, 1, r.randint(0, page * 3), r.randint(0, page * width), -1])) for x in who]
            got = kv4_reserve(pages, ints(who), ints(want))
            expect = m.reserve(who, want)
            assert got.tolist() == expect
            refused += expect.count(0)
        elif op == "fork":
            kids = [x for x in range(rows) if m.lens[x] == 0]
            old = [x for x in range(rows) if m.lens[x] > 0]
            if not kids or not old:
                continue
            kids = r.sample(kids, r.randint(1, len(kids)))
            old = [r.choice(old) for _ in kids]
            pages, ok = kv4_fork(cache, pages, ints(old), ints(kids), out=pages if step % 2 else None)
            assert ok.tolist() == m.fork(old, kids)
        elif op == "release":
            who = r.sample(range(rows), r.randint(1, max(1, rows // 3)))
            pages = kv4_release(pages, ints(who + who[:1]), out=pages if step % 2 else None)
            m.release(who)
        else:
            pages = kv4_compact(cache, pages, out=pages if step % 2 else None)
            m.compact()
        m.check(pages, cache)
    assert refused > 0


def test_copy_pages():
    cache = KV4Cache(3, 50, 2, 128, page_size=16, group_size=64)
    cache.pool.copy_(torch.randint(0, 256, cache.pool.shape, device="cuda", dtype=torch.uint8))
    want = cache.pool.clone()
    src, dst = ints([3, 4, -1, 7, 7]), ints([49, 0, 8, -1, 20])
    want[:, [49, 0, 20]] = want[:, [3, 4, 7]]
    kv4_copy_pages(cache, src, dst)
    assert torch.equal(cache.pool, want)
    kv4_copy_pages(cache, src[:0], dst[:0])
    assert torch.equal(cache.pool, want)


def test_pages_of_a_pool_past_32_bits():
    """Offsets in a pool of more than 4 GiB."""
    cache = KV4Cache(2, 40000, 8, 128, page_size=64)
    assert cache.pool.numel() > 1 << 32
    cache.pool[1, 39999] = stamp(5, 1, cache.pool[1, 39999])
    cache.pool[0, 3] = 7
    kv4_copy_pages(cache, ints([39999]), ints([2]))
    assert torch.equal(cache.pool[1, 2], cache.pool[1, 39999])
    g = gen(2)
    c = PlainCache([130], 8, 128, 128, 64, gen=g)
    new = torch.tensor([39000, 3, 39998], device="cuda")
    cache.pool[1, new] = c.pool[0, c.table[0, :3].long()]
    q = rand(g, 1, 32, 128)
    got = kv4_attention(q, cache, 1, new.int()[None], c.kv_lens)
    want = kv4_attention(q, KV4Cache(1, c.num_pages, 8, 128, pool=c.pool), 0, c.table, c.kv_lens)
    assert torch.equal(got, want)
    x = rand(g, 1, 24, 128)
    slot = torch.tensor([39999 * 64 + 63], device="cuda")
    pos, cs = torch.zeros(1, dtype=torch.int64, device="cuda"), cos_sin_table(1, 128)
    qk_norm_rope_append(x[:, :8], x[:, 8:16], x[:, 16:], cache, 1, slot, pos, cs)
    close_to_cached(kv4_gather(cache, 1, slot)[1], x[:, 16:].double(), 128, F16)


# ------------------------------------------------------------------------------------ refusals
def test_refusals():
    cache = KV4Cache(2, 8, 2, 64, page_size=16)
    q, k = rand(gen(0), 2, 4, 64), rand(gen(0), 2, 2, 64)
    pos, cs = torch.zeros(2, dtype=torch.int64, device="cuda"), cos_sin_table(4, 64)
    slots = torch.tensor([0, 1], device="cuda")
    table, lens = ints([[0], [1]]), ints([1, 1])
    for bad in (dict(positions=pos.int()), dict(positions=pos[:1]), dict(q=q.float()), dict(q=q[..., ::2]), dict(k=k[:1]),
                dict(cos_sin=cs.half()), dict(cos_sin=cs[:, :60]), dict(sections=(16, 8, 4)), dict(q_weight=pos),
                dict(sections=(16, 8, 8)), dict(k=k.bfloat16()), dict(q=q.cpu())):
        with pytest.raises(AssertionError):
            qk_norm_rope(**{**dict(q=q, k=k, positions=pos, cos_sin=cs), **bad})
    for bad in (dict(slots=slots.int()), dict(layer=2), dict(layer=-1), dict(v=k[:, :1]), dict(slots=slots[:1])):
        with pytest.raises(AssertionError):
            qk_norm_rope_append(**{**dict(q=q, k=k, v=k, cache=cache, layer=0, slots=slots, positions=pos, cos_sin=cs), **bad})
    for bad in (dict(q=q[:, :3]), dict(block_table=table.long()), dict(kv_lens=lens[:1]), dict(window=-1), dict(layer=7),
                dict(cu_q=ints([0, 2])), dict(q=torch.cat([q, q[:1]])), dict(out=q.float()), dict(block_table=table[0])):
        with pytest.raises(AssertionError):
            kv4_attention(**{**dict(q=q, cache=cache, layer=0, block_table=table, kv_lens=lens), **bad})
    with pytest.raises(W4A16Error):       # queries that no 16-byte load reaches
        kv4_attention(rand(gen(0), 2, 4 * 64 + 4)[:, 4:].unflatten(1, (4, 64)), cache, 0, table, lens)
    pages = KV4Pages.empty(cache, 4, 2)
    with pytest.raises(AssertionError):
        kv4_fork(KV4Cache(1, 9, 2, 64, page_size=16), pages, ints([0]), ints([1]))
    with pytest.raises(AssertionError):
        kv4_reserve(pages, ints([0]).long(), ints([1]))
    with pytest.raises(AssertionError):
        kv4_copy_pages(cache, ints([0]), ints([0, 1]))


def test_indices_out_of_range_are_flagged_and_skipped():
    cache = KV4Cache(1, 4, 1, 64, page_size=16)
    x = rand(gen(0), 2, 1, 64)
    cs = cos_sin_table(4, 64)
    good = torch.tensor([0, 1], device="cuda")

    def flagged():
        with pytest.raises(W4A16Error) as e:
            w4a16.check_device_errors()
        assert e.value.status == -8 and w4a16.check_device_errors() == 0

    qk_norm_rope(x, x, torch.tensor([0, 4], device="cuda"), cs)
    flagged()
    qk_norm_rope(x, x, torch.tensor([-1, 0], device="cuda"), cs)
    flagged()
    before = cache.pool.clone()
    qk_norm_rope_append(x, x, x, cache, 0, torch.tensor([64, 1 << 40], device="cuda"), good, cs)
    flagged()
    assert torch.equal(cache.pool, before)
    assert (kv4_gather(cache, 0, torch.tensor([64], device="cuda")) == 0).all()
    flagged()
    qk_norm_rope_append(x, x, x, cache, 0, good, good, cs)
    for page in (4, -1, 1 << 30):
        o = kv4_attention(x, cache, 0, ints([[0], [page]]), ints([2, 2]))
        flagged()
        assert torch.equal(o[0], kv4_attention(x[:1], cache, 0, ints([[0]]), ints([2]))[0]) and (o[1] == 0).all()
    kv4_copy_pages(cache, ints([4]), ints([0]))
    flagged()
    pages = KV4Pages.empty(cache, 2, 3)
    assert kv4_reserve(pages, ints([2, 0]), ints([5, 5])).tolist() == [0, 1]
    flagged()
    kv4_release(pages, ints([-1]), out=pages)
    flagged()
    _, ok = kv4_fork(cache, pages, ints([0, 9]), ints([1, 0]), out=pages)
    flagged()
    assert ok.tolist() == [1, 0]
