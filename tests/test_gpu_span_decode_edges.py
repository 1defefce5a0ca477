"""Span attention over pages where its results lie at any address that it takes."""
import pytest
import torch

from test_gpu_span_decode import _case, _check

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


# one part, a cluster of eight, more parts than a cluster (which a second kernel joins); the forward pass's join has the same stores
@pytest.mark.parametrize("ctx,splits", [(60, 1), (3000, 8), (40000, 64)])
@pytest.mark.parametrize("D,dtype", [(64, BF), (72, HF)])
def test_results_at_any_8_byte_boundary(ctx, splits, D, dtype):
    from rumus_b200.ops import native
    from rumus_b200.ops.span import span_decode
    args = _case([ctx], 4, 1, D, 64, dtype, spread=2.0)
    assert native.lib().rb_span_decode_splits(1, 4, 1, ctx) == splits
    want = _check(args, 4, cap=30.0)
    for first in (4, 8, 12, 16):
        flat = torch.full((4 * D + 32,), 7.0, dtype=dtype, device="cuda")
        got = span_decode(*args, ctx, cap=30.0, out=flat[first:first + 4 * D].view(1, 4, D))
        assert got.data_ptr() % 16 == first * 2 % 16 and torch.equal(got, want) and native.read_status() == 0
        assert (flat[:first] == 7).all() and (flat[first + 4 * D:] == 7).all()
