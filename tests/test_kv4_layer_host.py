"""W4A16Attention's host side, without a GPU: its buffers and its refusals."""
from __future__ import annotations

import pytest
import torch

from w4a16 import W4A16Attention


def test_buffers():
    layer = W4A16Attention(256, 6, 2, 64, bias=True)
    assert {k: tuple(v.shape) for k, v in layer.state_dict().items()} == {
        "q_norm": (64,), "k_norm": (64,),
        "qkv.qweight": (32, 640), "qkv.scales": (2, 640), "qkv.zeros": (2, 640), "qkv.bias": (640,),
        "out.qweight": (48, 256), "out.scales": (3, 256), "out.zeros": (3, 256), "out.bias": (256,)}
    assert W4A16Attention(256, 6, 2, 64, qk_norm=False).q_norm is None


@pytest.mark.parametrize("args,kw", [((256, 6, 4, 64), {}), ((256, 6, 2, 96), {}), ((256, 0, 1, 64), {}), ((256, 6, 2, 64), {"window": -1}),
                                     ((200, 6, 2, 64), {})])
def test_refusals(args, kw):
    with pytest.raises(ValueError):
        W4A16Attention(*args, **kw)


def test_a_wrong_input_is_refused_before_anything_runs():
    layer = W4A16Attention(256, 6, 2, 64)
    with pytest.raises(AssertionError):
        layer(torch.zeros(2, 3, 256, dtype=torch.float16), None, 0, None, None, None, None)
