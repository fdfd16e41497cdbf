"""The draw of verify_drafts where the running sums come near the border: ranges that hold nothing, numbers at the end of
their range."""
from __future__ import annotations

from fractions import Fraction

import numpy as np
import pytest
import torch

import w4a16
from w4a16 import verify_drafts

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_device_errors():
    yield
    assert w4a16.check_device_errors() == 0


def draw(r, u):
    """The token by exact arithmetic."""
    at = np.nonzero(r)[0]
    r = [Fraction(float(r[v])) for v in at]
    border, total = Fraction(float(u)) * sum(r), Fraction(0)
    for v, x in zip(at, r):
        total += x
        if total > border:
            return int(v)
    return int(at[-1])


def drawn(row, u, batch=1):
    """The token drawn from row [V] by u, in `batch` sequences alike."""
    row = torch.as_tensor(row, dtype=torch.float32, device="cuda")
    out, accepted = verify_drafts(row.expand(batch, 1, -1), None, torch.empty((batch, 0), dtype=torch.int64, device="cuda"),
                                  torch.full((batch, 1), u, device="cuda"))
    assert (accepted == 0).all() and (out == out[0]).all()
    return int(out[0, 0])


def test_a_range_of_nothing_has_no_border():
    """The sums before two neighbouring ranges differ by a rounding although the second is empty, and the border lies between."""
    row = np.zeros(16384, np.float32)
    for at, x in ((6, "0x1.b4b0fcp-34"), (57, "0x1.b4b0fcp-34"), (10, "0x1.9791b4p-4"), (53, "0x1.9791b4p-4"), (11, "0x1.1ed662p-34"),
                  (52, "0x1.1ed662p-34")):
        row[256 * at] = float.fromhex(x)
    assert draw(row, 0.5) == 13312
    assert drawn(row, 0.5) == 13312


@pytest.mark.parametrize("V", [16384, 16385, 131072])
def test_numbers_beyond_the_range_take_the_last_token(V):
    """Sharp distributions with nothing in the tail, numbers of 1 and more."""
    rng = np.random.default_rng(V)
    rows = np.zeros((400, V), np.float32)
    last = rng.integers(V // 8, V // 2, 400)
    for row, n in zip(rows, last):
        row[:n + 1] = np.exp(rng.normal(size=n + 1) * 8.0 - 20.0)
    target = torch.from_numpy(rows).cuda()
    for u in (1.0, 1.5, float("inf")):
        out, _ = verify_drafts(target[:, None], None, torch.empty((400, 0), dtype=torch.int64, device="cuda"), torch.full((400, 1), u, device="cuda"))
        assert out[:, 0].tolist() == last.tolist()
