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
    """A graph whose replay fills the free memory of a graph pool (and stream) with 0xFF."""

    def __init__(self, pool, nbytes, stream=None):
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph, pool=pool, stream=stream):
            x = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
            x.fill_(255)
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
