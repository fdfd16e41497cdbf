"""Weights collected from the drafts that stand alone: behind the verification, with a log-sum-exp of -inf where a query's draft
was rejected, before the lengths are lowered. Against the float64 form over the accepted queries and the lowered lengths; tolerance
as in test_gpu_kv4_weights.py."""
from __future__ import annotations

import math

import pytest
import torch

import w4a16
from kv4_bounded_plain import collect
from test_gpu_kv4_weights import BF16, F16, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 4), (3, 1)])
@pytest.mark.parametrize("H,KV,D,dtype", [(8, 2, 128, F16), (12, 4, 64, BF16), (72, 2, 128, F16)])
def test_rejected_drafts_give_nothing(H, KV, D, dtype, window, sinks):
    B, K = 5, 4
    c = Case([700, 333, 5, 64, 1200], [K + 1] * B, H, KV, D, 64, 16, dtype, window, sinks)
    accepted = torch.tensor([4, 0, 2, 1, 3], dtype=torch.int32, device="cuda")
    full = c.call(c.before.clone())
    lse = c.lse.clone()
    gone = torch.arange(K + 1, device="cuda") > accepted[:, None]            # queries of rejected drafts
    c.lse.unflatten(0, (-1, K + 1)).masked_fill_(gone[..., None], -math.inf)
    assert (c.lse == -math.inf).sum() == 10 * H
    w = c.call(c.before.clone(), cu_q=None, max_q=None)
    c.c.kv_lens -= K - accepted
    for b in range(B):
        a, n = int(accepted[b]), c.lens[b] - K + int(accepted[b])
        rows = slice(b * (K + 1), b * (K + 1) + a + 1)
        want = collect(c.q[rows], c.c.k[b][:n], lse[rows], c.before[b], c.share, c.scale, window, sinks)
        had = c.before[b, :, :n].double().nan_to_num(nan=0.0)
        had[:, n - a - 1:] = 0.0
        top = (c.q[rows].double().norm(dim=-1).amax() * c.c.k[b][:n].norm(dim=-1).amax() * c.scale).item()
        tol = (want - had) * (2e-6 * (1 + top) + 2.0 ** -20) + 2.0 ** -23 * want + 1e-30
        assert ((w[b, :, :n].double() - want).abs() <= tol).all()
        assert (w[b, :, n:c.lens[b]] == 0).all()                             # the rejected tokens' own places
        # collected before the verification they count
        assert a == K or (full[b, :, :n].double().sum() > want.sum() + 0.5)
    assert w4a16.check_device_errors() == 0
