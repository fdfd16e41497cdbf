"""Workspaces under CUDA graphs: graphs replayed in another order than they were captured in, graphs that share memory
with others, and calls outside a graph on the stream it was captured on."""
from __future__ import annotations

import pytest
import torch

import w4a16
from kv4_plain import PlainCache
from w4a16 import KV4Cache, kv4_attention

pytestmark = pytest.mark.gpu


class Dirt:
    """A graph whose replay fills the free memory of a graph pool (and stream) with one 64-bit word."""

    def __init__(self, pool, nbytes, stream=None, word=-1):
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph, pool=pool, stream=stream):
            x = torch.empty(nbytes // 8, dtype=torch.int64, device="cuda")
            x.fill_(word)
            del x

    def spread(self):
        self.graph.replay()
        torch.cuda.synchronize()


def sequences(lens, seed):
    c = PlainCache(lens, 2, 128, 128, 64, gen=torch.Generator(device="cuda").manual_seed(seed))
    cache = KV4Cache(1, c.num_pages, 2, 128, pool=c.pool)
    q = torch.randn((len(lens), 16, 128), generator=torch.Generator(device="cuda").manual_seed(seed + 1), device="cuda").half()
    want = kv4_attention(q, cache, 0, c.table, c.kv_lens)
    return c, cache, q, want, torch.full((2, *want.shape), float("nan"), device="cuda", dtype=want.dtype)


def test_graphs_replayed_in_another_order():
    pool = torch.cuda.graph_pool_handle()
    dirt = Dirt(pool, 64 << 20)
    cases = [sequences([9000], 1), sequences([7000, 20000], 2), sequences([5000], 3)]       # split over many teams
    graphs = []
    for c, cache, q, want, out in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            for o in out:
                kv4_attention(q, cache, 0, c.table, c.kv_lens, out=o)
        graphs.append(g)
    for order in ((1, 0, 2), (2, 2, 1), (0, 1, 2)):
        dirt.spread()
        for i in order:
            graphs[i].replay()
            torch.cuda.synchronize()
            want, out = cases[i][3:]
            assert torch.equal(out[0], want) and torch.equal(out[1], want), (order, i)
            out.fill_(float("nan"))
    assert w4a16.check_device_errors() == 0


def test_calls_outside_a_graph_on_its_stream():
    side, pool = torch.cuda.Stream(), torch.cuda.graph_pool_handle()
    dirt = Dirt(pool, 64 << 20, side)
    small, large = sequences([300], 4), sequences([30000] + [200] * 79, 5)     # more teams, long parts
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kv4_attention(small[2], small[1], 0, small[0].table, small[0].kv_lens, out=small[4][0])
    side.synchronize()
    dirt.spread()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, pool=pool, stream=side):
        kv4_attention(large[2], large[1], 0, large[0].table, large[0].kv_lens, out=large[4][0])
    with torch.cuda.stream(side):
        for _ in range(2):
            o = kv4_attention(large[2], large[1], 0, large[0].table, large[0].kv_lens, out=torch.full_like(large[3], float("nan")))
            side.synchronize()
            assert torch.equal(o, large[3])
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(large[4][0], large[3]) and torch.equal(small[4][0], small[3])
    assert w4a16.check_device_errors() == 0


def test_gemm_graphs_replayed_in_another_order():
    """The GEMMs' workspace holds pieces of column strips (few rows) and counters of K splits (many rows)."""
    g = torch.Generator(device="cuda").manual_seed(6)
    K, N, G = 4096, 2048, 128
    w = w4a16.quantize_weight((torch.randn((K, N), generator=g, device="cuda") * 0.02).half(), G)
    pool = torch.cuda.graph_pool_handle()
    dirt = Dirt(pool, 128 << 20, word=1 << 32)       # as a piece of a strip that has arrived looks, and odd counters of one
    xs = [torch.randn((m, K), generator=g, device="cuda").half() for m in (1, 40, 8, 100)]
    assert all(w4a16._lib.gemm_workspace_bytes(x.shape[0], N, K, G, x.device) > 0 for x in xs)
    want = [w4a16.w4a16_matmul(x, *w, G) for x in xs]
    outs = [torch.full((2, *y.shape), float("nan"), device="cuda", dtype=y.dtype) for y in want]
    graphs = []
    for x, out in zip(xs, outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            for o in out:
                w4a16.w4a16_matmul(x, *w, G, out=o)
        graphs.append(graph)
    for order in ((2, 0, 3, 1), (1, 3), (0, 1, 2, 3)):
        dirt.spread()
        for i in order:
            graphs[i].replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[i][0], want[i]) and torch.equal(outs[i][1], want[i]), (order, i)
            outs[i].fill_(float("nan"))
    assert w4a16.check_device_errors() == 0
