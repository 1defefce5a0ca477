"""Scales and caps that the kernels' 32 bits do not hold are refused, not turned into others."""
import math

import pytest
import torch

from rumus_b200.ops import functional as F
from rumus_b200.ops.span import span_decode


def _calls(**kw):
    q = torch.randn(1, 3, 2, 8)
    pages = torch.randn(1, 4, 2, 8)
    yield lambda: F.span_attention(q, q, q, **kw)
    yield lambda: span_decode(q[:, 0], pages, pages, torch.zeros(1, 1, dtype=torch.int32), torch.tensor([3], dtype=torch.int32), 3, **kw)


@pytest.mark.parametrize("kw", [dict(cap=1e300), dict(cap=3e38), dict(cap=1e-46), dict(cap=5e-324), dict(cap=math.inf), dict(scale=1e39), dict(scale=-3e38),
                                dict(scale=math.nan), dict(cap=1e-30, scale=1e10), dict(cap=1e-40)])
def test_refused(kw):
    for call in _calls(**kw):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("kw", [dict(cap=2e38), dict(cap=1e-37), dict(cap=0.0), dict(scale=2e38 / 1e36), dict(scale=0.0, cap=1e-40), dict(cap=1e-30, scale=-1.0)])
def test_taken(kw):
    for call in _calls(**kw):
        assert torch.isfinite(call()).all()


@pytest.mark.parametrize("shape", [(1, 3, 2, 0), (), (3, 2, 8)])
def test_heads_of_nothing_and_other_shapes_are_refused(shape):
    q = torch.zeros(shape)
    with pytest.raises(ValueError, match="span attention of"):
        F.span_attention(q, q, q)
