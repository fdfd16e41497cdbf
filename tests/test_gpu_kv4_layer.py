"""W4A16Attention: prompts, drafts, single tokens and page management as a serving loop runs them."""
import math

import pytest
import torch

from kv4_plain import PlainCache, attend, cos_sin_table
from test_gpu_kv4 import check_attention, gen
from w4a16 import (KV4Cache, KV4Pages, W4A16Attention, check_device_errors, kv4_attention, kv4_compact, kv4_fork, kv4_gather,
                   kv4_release, kv4_reserve, qk_norm_rope, qk_norm_rope_append)

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
DEV = "cuda"


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def make_layer(hidden, H, KV, D, **kw):
    g = gen(3)
    layer = W4A16Attention(hidden, H, KV, D, device=DEV, **kw)
    for lin in (layer.qkv, layer.out):
        w = torch.randn((lin.in_features, lin.out_features), generator=g, device=DEV) / math.sqrt(lin.in_features)
        lin.quantize_from_dense(w)
    if layer.q_norm is not None:
        layer.q_norm.copy_(1 + 0.1 * torch.randn(D, generator=g, device=DEV))
    return layer


class Loop:
    """The rows' new tokens through the layer, one step at a time."""

    def __init__(self, layer, cache, rows, width):
        self.layer, self.cache, self.pages = layer, cache, KV4Pages.empty(cache, rows, width)
        self.lens = [0] * rows
        self.cs = cos_sin_table(4096, layer.head_dim)
        layer.out.register_forward_pre_hook(lambda mod, args: setattr(self, "seen", args[0]))

    def step(self, xs):
        """xs: the new tokens [n, hidden] of each row (n may be 0)."""
        lay, new = self.layer, [x.shape[0] for x in xs]
        grow = [r for r, n in enumerate(new) if n]
        ends = [a + n for a, n in zip(self.lens, new)]
        assert kv4_reserve(self.pages, ints(grow), ints([ends[r] for r in grow])).all()
        row = torch.cat([torch.full((n,), r, device=DEV) for r, n in enumerate(new)])
        pos = torch.cat([torch.arange(a, b, device=DEV) for a, b in zip(self.lens, ends)])
        cu = ints([0] + torch.tensor(new).cumsum(0).tolist())
        x = torch.cat(xs)
        y = lay(x, self.cache, 0, self.pages, self.pages.slots(row, pos), pos, self.cs, cu_q=cu, max_q=max(new))
        qkv = lay.qkv(x).view(x.shape[0], -1, lay.head_dim)
        self.q = qk_norm_rope(qkv[:, :lay.heads], qkv[:, lay.heads:lay.heads + lay.kv_heads], pos, self.cs, lay.q_norm,
                              lay.k_norm, lay.eps)[0].split(new)
        self.o = self.seen.view(x.shape[0], lay.heads, lay.head_dim).split(new)
        self.lens = ends
        return y.split(new)

    def stored(self, r):
        pos = torch.arange(self.lens[r], device=DEV)
        return kv4_gather(self.cache, 0, self.pages.slots(torch.full_like(pos, r), pos)).double()


def rows_of(g, hidden, *new):
    return [torch.randn((n, hidden), generator=g, device=DEV).half() for n in new]


@pytest.mark.parametrize("H,KV,D,page,group,window,norm", [(8, 2, 128, 32, 128, 0, True), (6, 3, 64, 16, 64, 50, True),
                                                           (4, 4, 128, 64, 64, 0, False)])
def test_layer_serves_prompts_drafts_and_tokens(H, KV, D, page, group, window, norm):
    layer = make_layer(256, H, KV, D, window=window, qk_norm=norm)
    loop = Loop(layer, KV4Cache(1, 80, KV, D, page_size=page, group_size=group), 4, 20)
    g = gen(11)
    for new in ([130, 9, 0, 1], [1, 1, 0, 1], [5, 0, 70, 3], [1, 1, 1, 1]):
        ys = loop.step(rows_of(g, 256, *new))
        for r, n in enumerate(new):
            assert ys[r].shape == (n, 256) and ys[r].isfinite().all()
            if n == 0:
                continue
            # against the cached keys and values rounded to fp16: with half an ulp of every key a score moves by at
            # most 2^-11 of the bound `top`, a result by twice that of vmax; half an ulp each of the values, here
            # and in the kernel, and of the probabilities; then the output's own and fp32's
            k, v = loop.stored(r)
            want, _ = attend(loop.q[r], k, v, H // KV, 1 / math.sqrt(D), window)
            top = (loop.q[r].double().norm(dim=-1).amax() * k.norm(dim=-1).amax() / math.sqrt(D)).item()
            vmax = v.abs().amax().item()
            tol = 2.0 ** -11 * want.abs() + (2 * top + 3) * 2.0 ** -11 * vmax + 2e-5 * (1 + top) * vmax
            assert ((loop.o[r].double() - want).abs() <= tol).all()
    check_device_errors()


def test_fork_release_and_compact_between_steps():
    layer = make_layer(256, 8, 2, 128)
    cache = KV4Cache(1, 40, 2, 128, page_size=16)
    loop = Loop(layer, cache, 4, 12)
    g = gen(12)
    loop.step(rows_of(g, 256, 37, 100, 0, 0))
    pages, ok = kv4_fork(cache, loop.pages, ints([1, 1]), ints([2, 3]))
    assert ok.tolist() == [1, 1] and pages.kv_lens.tolist() == [37, 100, 100, 100]
    loop.pages, loop.lens = pages, [37, 100, 100, 100]
    xs = rows_of(g, 256, 1, 1, 0, 1)
    ys = loop.step([xs[0], xs[1], xs[1], xs[2].new_zeros(0, 256)])   # row 2 goes on as its parent does, row 3 waits
    assert torch.equal(loop.q[1], loop.q[2])
    vmax = loop.stored(1)[1].abs().amax().item()
    assert (loop.o[1].double() - loop.o[2].double()).abs().amax() <= 2.0 ** -10 * 2 * vmax   # roundings of two orders of sums
    assert (loop.stored(1) == loop.stored(2)).all() and ys[3].shape == (0, 256)
    # the parent goes; the pool is made dense; what is left reads the same
    q = torch.randn((4, 8, 128), generator=g, device=DEV).half()
    loop.pages = kv4_release(loop.pages, ints([1]))
    before = kv4_attention(q, cache, 0, loop.pages.block_table, loop.pages.kv_lens)
    loop.pages = kv4_compact(cache, loop.pages)
    used = int((loop.pages.refs > 0).sum())
    assert (loop.pages.refs[:used] > 0).all() and (loop.pages.refs[used:] == 0).all()
    after = kv4_attention(q, cache, 0, loop.pages.block_table, loop.pages.kv_lens)
    assert torch.equal(before, after) and (after[1] == 0).all() and after.isfinite().all()
    check_device_errors()


@pytest.mark.parametrize("H,KV,D,group", [(8, 1, 128, 128), (8, 1, 128, 64), (16, 1, 64, 64)])
def test_small_prompts_step_and_tile_edges(H, KV, D, group):
    """Prompts of small batches: lengths around the tokens of a step, rows around one and two row tiles, and a window
    that begins inside a step."""
    for n in (1, 31, 33, 63, 64, 65, 127, 128, 129, 193, 257):
        check_attention([n, 3], [9, 1], H, KV, D, group, 16, F16, seed=n)            # 72 or 144 rows
        check_attention([max(n, 40)], [33], H, KV, D, group, 16, BF16, seed=n)       # a last tile of few rows
        check_attention([300 + n], [40], H, KV, D, group, 16, F16, window=n, seed=n)


def test_small_prompt_sees_a_nan_value_it_attends_to_and_no_other():
    """A NaN value makes its group NaN for the queries that see it, not for earlier ones or other groups."""
    g = gen(10)
    for group, token in ((64, 70), (128, 70), (64, 129)):
        c = PlainCache([130], 1, 128, group, 16, gen=g)
        cache = KV4Cache(1, c.num_pages, 1, 128, page_size=16, group_size=group, pool=c.pool)
        v = torch.zeros((1, 1, 128), device=DEV, dtype=F16)
        v[..., 100] = float("nan")
        k = torch.randn((1, 1, 128), device=DEV, generator=g).half()
        qk_norm_rope_append(torch.empty(1, 0, 128, device=DEV, dtype=F16), k, v, cache, 0, c.slots(0, token, 1),
                            torch.zeros(1, dtype=torch.int64, device=DEV), cos_sin_table(1, 8))
        q = torch.randn((100, 2, 128), device=DEV, generator=g).half()
        for window in (0, 20):
            o, lse = kv4_attention(q, cache, 0, c.table, c.kv_lens, window=window, return_lse=True)
            at = torch.arange(30, 130, device=DEV)
            sees = (at >= token) & ((at < token + window) if window else True)
            half = 0 if group == 128 else 64
            assert o[sees][..., half:].isnan().all() and o[~sees].isfinite().all() and o[..., :half].isfinite().all()
            assert lse.isfinite().all()


@pytest.mark.parametrize("H,KV,D,group", [(64, 8, 128, 128), (64, 8, 128, 64), (48, 16, 64, 64)])
def test_large_prompts_step_and_tile_edges(H, KV, D, group):
    """As above with enough rows, kv heads and sequences for the kernel that takes long prompts: lengths around the
    tokens of a step, one and two row tiles, tiles of few rows, short sequences in the same batch."""
    share = H // KV
    for i, n in enumerate((1, 31, 33, 63, 64, 65, 127, 128, 129, 193)):
        new = [n + 8192 // (3 * KV * share) + 1, 256 // share + 1, 1 + i % 3]
        assert max(new) * share * KV * 3 > 8192 and max(new) * share > 64
        check_attention([max(n, new[0]), new[1] + i, n], new[:2] + [min(n, new[2])], H, KV, D, group, 16, F16, seed=n)
        check_attention([new[0] + n, 7, 300], [new[0], 0, 130 // share], H, KV, D, group, 32, BF16, window=1 + n, seed=n)


def test_large_prompt_sees_a_nan_value_it_attends_to_and_no_other():
    g = gen(10)
    for group, token in ((64, 70), (128, 70), (64, 129)):
        c = PlainCache([130], 32, 128, group, 16, gen=g)
        cache = KV4Cache(1, c.num_pages, 32, 128, page_size=16, group_size=group, pool=c.pool)
        v = torch.zeros((1, 32, 128), device=DEV, dtype=F16)
        v[:, 5, 100] = float("nan")
        k = torch.randn((1, 32, 128), device=DEV, generator=g).half()
        qk_norm_rope_append(torch.empty(1, 0, 128, device=DEV, dtype=F16), k, v, cache, 0, c.slots(0, token, 1),
                            torch.zeros(1, dtype=torch.int64, device=DEV), cos_sin_table(1, 8))
        q = torch.randn((100, 96, 128), device=DEV, generator=g).half()
        for window in (0, 20):
            o, lse = kv4_attention(q, cache, 0, c.table, c.kv_lens, window=window, return_lse=True)
            at = torch.arange(30, 130, device=DEV)
            sees = (at >= token) & ((at < token + window) if window else True)
            half = 0 if group == 128 else 64
            hit, rest = o[:, 15:18], torch.cat([o[:, :15], o[:, 18:]], 1)
            assert hit[sees][..., half:].isnan().all() and hit[~sees].isfinite().all() and hit[..., :half].isfinite().all()
            assert rest.isfinite().all() and lse.isfinite().all()


def test_large_prompts_of_large_values():
    """Values near fp16's end in the kernel that rounds them to fp16: finite, and within its bound."""
    check_attention([200, 90, 160], [180, 90, 100], 16, 16, 128, 128, 32, F16, v_scale=14000.0, seed=1)
