"""The draw of verify_drafts where the running sums come near the border: ranges that hold nothing, numbers at the end of
their range, and sums of many values of very different sizes."""
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


def mirrored(V, seed, sharp):
    """Values that read the same from both ends, and what the first half has more than the second: nothing yet."""
    rng = np.random.default_rng(seed)
    half = np.exp(rng.normal(size=V // 2) * sharp).astype(np.float32)
    half /= 2 * half.sum(dtype=np.float64)
    half[0], half[-1] = 0.0, 2.0 ** -20
    return np.concatenate([half, half[::-1]])


# The kernel's sums are within 2^-45 of themselves and 2^-53 more for each fp64 addition of a thread, 1024 of them here: within
# 2^-42.7 of the whole together. A half that has 2^-41 of the whole more than the other moves the edge by 2^-42 from where half
# of the whole lies, so the token is decided, whatever the order of the sums.
MORE = 2.0 ** -41


@pytest.mark.parametrize("batch", [1, 40, 300])
@pytest.mark.parametrize("V", [20000, 1 << 17, (1 << 17) + 2, 1 << 22])
def test_the_token_does_not_depend_on_the_batch(V, batch):
    for seed in range(8):
        row = mirrored(V, seed, sharp=1.0 + seed)
        assert drawn(row + np.float32(MORE) * (np.arange(V) == 0), 0.5, batch) == V // 2 - 1, seed
        assert drawn(row + np.float32(MORE) * (np.arange(V) == V - 1), 0.5, batch) == V // 2, seed


@pytest.mark.parametrize("batch", [1, 40, 300])
@pytest.mark.parametrize("V", [20000, 1 << 17, (1 << 17) + 2, 1 << 22])
def test_the_token_does_not_depend_on_the_batch_with_a_draft(V, batch):
    """The same for what a target has over a draft."""
    for seed in range(8):
        p = mirrored(V, seed, sharp=1.0 + seed)
        part = np.random.default_rng(100 + seed).random(V // 2, dtype=np.float32)
        q = p * np.concatenate([part, part[::-1]])
        q[V // 2 - 1:V // 2 + 1] = 0.0
        q[[5, V - 6]] = 4 * p[[5, V - 6]]                 # token 5 is not accepted
        whole = (p.astype(np.float64) - np.minimum(p, q)).sum()
        assert whole > 0.2                                # (so MORE is no less of it)
        for at, want in ((0, V // 2 - 1), (V - 1, V // 2)):
            target = torch.from_numpy(p + np.float32(MORE) * (np.arange(V) == at)).cuda()
            draft = torch.from_numpy(q).cuda()
            out, accepted = verify_drafts(target.expand(batch, 2, V), draft.expand(batch, 1, V), torch.full((batch, 1), 5, device="cuda"),
                                          torch.tensor([[0.9, 0.5]], device="cuda").expand(batch, 2).contiguous())
            assert (accepted == 0).all() and (out[:, 0] == want).all(), (seed, out[:, 0])
