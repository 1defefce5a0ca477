"""Capped scores that fall with the distance: tiles so far from a row's nearest key that they have no weight are left out, and nothing else is."""
import pytest
import torch

from test_gpu_span import BF, HF, _check, _inputs, _random_spans, _run, _slopes
from test_gpu_span_decode import _case
from test_gpu_span_decode import _check as _check_decode

pytestmark = pytest.mark.gpu


def _steep(*slopes):
    return torch.tensor(slopes, device="cuda")


# heads that reach 16 places, some hundreds, and all; few rows over many keys are split over the keys
@pytest.mark.parametrize("B,Sq,Sk", [(1, 900, 900), (2, 700, 1300), (1, 20, 5000), (1, 1300, 500)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_far_tiles(B, Sq, Sk, causal, dtype):
    q, k, v, do = _inputs(B, Sq, Sk, 6, 2, 64, dtype, spread=2.0)
    _check(q, k, v, do, causal=causal, cap=5.0, slopes=_steep(10.0, 1.0, 0.3, 0.0, -0.01, 1e-30))


# without a cap the lengths of queries and keys say how far a score can be from zero: one of each is long here, and its scores win over the distance
@pytest.mark.parametrize("B,Sq,Sk", [(1, 4200, 4200), (2, 1100, 4300)])
@pytest.mark.parametrize("D,dtype", [(64, BF), (128, HF), (40, BF)])
def test_far_tiles_without_a_cap(B, Sq, Sk, D, dtype):
    from rumus_b200.ops import span
    q, k, v, do = _inputs(B, Sq, Sk, 4, 2, D, dtype, spread=0.5)
    q[:, Sq - 7, 1] *= 20
    k[:, 5, 0] = q[:, Sq - 7, 1] / 4
    slopes = _steep(2.0, 0.25, 0.05, -0.001)
    assert span._norms(q, k, 0.0, slopes) is not None
    _check(q, k, v, do, causal=Sq > 2000, slopes=slopes)


# rows whose nearest key is far: the distance counts from there
@pytest.mark.parametrize("causal", [True, False])
def test_rows_whose_keys_are_all_far(causal):
    q, k, v, do = _inputs(2, 600, 1500, 4, 4, 64, BF, spread=2.0)
    lo = torch.arange(600, device="cuda")
    near = torch.stack([lo * 0, 1 + lo // 2], -1)                  # the first keys, 900 places and more behind
    far = torch.stack([1500 - lo // 2, lo * 0 + 1500], -1)         # the last ones, ahead
    spans = torch.stack([near, far]).to(torch.int32)
    _check(q, k, v, do, causal=causal, spans=spans, cap=3.0, slopes=_steep(4.0, 0.5, 0.1, 0.01))


def test_spans_in_any_order():
    q, k, v, do = _inputs(2, 700, 1000, 4, 2, 128, BF)
    _check(q, k, v, do, causal=False, spans=_random_spans(2, 700, 1000), cap=2.0, slopes=_steep(8.0, 2.0, 0.5, 0.25))


# more query heads to a key head than have lists of their own
@pytest.mark.parametrize("group", [64, 65, 100])
def test_many_heads_share_a_key_head(group):
    q, k, v, do = _inputs(1, 400, 400, group, 1, 32, BF)
    _check(q, k, v, do, cap=2.0, slopes=_slopes(group, 16.0))


# tiles of keys that one CTA, two, some and eight share; keys that few rows see leave some of them without any
@pytest.mark.parametrize("B,S,H,Hkv,parts", [(8, 600, 8, 8, 1), (1, 700, 4, 2, 2), (2, 900, 8, 2, 7), (1, 1030, 8, 1, 8)])
@pytest.mark.parametrize("D", [64, 80, 128])
@pytest.mark.parametrize("spans", [False, True])
def test_shared_tiles(B, S, H, Hkv, parts, D, spans):
    from rumus_b200.ops import native
    assert native.lib().rb_span_bwd_parts(B, H, Hkv, S, S, 0) == parts
    q, k, v, do = _inputs(B, S, S, H, Hkv, D, BF)
    got = _check(q, k, v, do, spans=_random_spans(B, S, S) if spans else None, cap=8.0)
    again = _run(q, k, v, do, spans=_random_spans(B, S, S) if spans else None, cap=8.0)
    assert all(torch.equal(got[n], again[n]) for n in got)


@pytest.mark.parametrize("H,Hkv", [(4, 4), (8, 2), (40, 2)])
@pytest.mark.parametrize("B", [1, 60])
def test_decode(H, Hkv, B):
    args = _case([3000 - 40 * b for b in range(B)], H, Hkv, 64, 64, BF, spread=2.0)
    _check_decode(args, H, cap=5.0, slopes=_slopes(H, 4.0))
    _check_decode(args, H, cap=5.0, slopes=_steep(*[2.0] * H))
    _check_decode(args, H, cap=5.0, slopes=_steep(*[2.0] * (H - 1), 0.0))


def test_decode_without_the_last_page():
    """The nearest token that is there lies far: what counts is the distance from it."""
    q, k, v, tables, ctx = _case([2000, 2000, 1990], 4, 2, 64, 64, BF, spread=2.0)
    tables[0, -1] = -1
    tables[1, 5:] = 10 ** 9
    _check_decode((q, k, v, tables, ctx), 4, cap=5.0, slopes=_steep(3.0, 2.0, 1.0, 0.5))


def test_spans_at_an_odd_address():
    q, k, v, do = _inputs(2, 90, 90, 2, 2, 64, BF)
    spans = _random_spans(2, 90, 90)
    odd = torch.cat([spans.view(-1)[:1], spans.view(-1)])[1:].view(2, 90, 2)
    assert odd.data_ptr() % 8 == 4
    _check(q, k, v, do, spans=odd)
