"""Span attention's plain math, its spans and its refusals."""
import dataclasses
import math

import pytest
import torch

from rumus_b200.ops import functional as F
from rumus_b200.ops.span import distance_slopes, span_decode


def _heads(B=2, Sq=9, Sk=9, H=4, Hkv=2, D=8, dtype=torch.float64, seed=0):
    g = torch.Generator().manual_seed(seed)
    return tuple(torch.randn(B, S, h, D, generator=g, dtype=torch.float64).to(dtype) for S, h in ((Sq, H), (Sk, Hkv), (Sk, Hkv)))


def _brute(q, k, v, spans, causal, scale, cap, slopes):
    """Row by row."""
    B, Sq, H, D = q.shape
    Sk, G = k.shape[1], H // k.shape[2]
    out = torch.zeros_like(q)
    for b in range(B):
        for h in range(H):
            for i in range(Sq):
                lo, hi = (0, Sk) if spans is None else spans.expand(B, Sq, 2)[b, i].tolist()
                js = [j for j in range(Sk) if lo <= j < hi and (not causal or j <= i + Sk - Sq)]
                if not js:
                    continue
                x = []
                for j in js:
                    s = scale * float(q[b, i, h] @ k[b, j, h // G])
                    s = cap * math.tanh(s / cap) if cap else s
                    x.append(s - (float(slopes[h]) * abs(i + Sk - Sq - j) if slopes is not None else 0.0))
                w = torch.softmax(torch.tensor(x, dtype=q.dtype), 0)
                out[b, i, h] = sum(w[n] * v[b, j, h // G] for n, j in enumerate(js))
    return out


SPANS = torch.tensor([[0, 4], [2, 3], [3, 3], [5, 2], [-3, 2], [4, 40], [0, 9], [8, 9], [9, 12]], dtype=torch.int32)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("spans", [None, SPANS, SPANS.flip(0).expand(2, 9, 2)])
@pytest.mark.parametrize("cap,bias", [(0.0, False), (0.7, True)])
def test_plain_math(causal, spans, cap, bias):
    q, k, v = _heads()
    slopes = distance_slopes(4) if bias else None
    got = F.span_attention(q, k, v, spans, causal, 0.4, cap, slopes)
    assert torch.allclose(got, _brute(q, k, v, spans, causal, 0.4, cap, slopes), atol=1e-12)


@pytest.mark.parametrize("Sq,Sk", [(1, 1), (3, 9), (9, 3), (4, 0), (0, 4)])
def test_lengths(Sq, Sk):
    q, k, v = _heads(Sq=Sq, Sk=Sk)
    got = F.span_attention(q, k, v, cap=2.0)
    assert got.shape == q.shape and torch.allclose(got, _brute(q, k, v, None, True, 8 ** -0.5, 2.0, None), atol=1e-12)


def test_without_options_it_is_attention():
    q, k, v = _heads(dtype=torch.float32)
    assert torch.allclose(F.span_attention(q, k, v), F.flash_attention(q, k, v), atol=1e-6)


@pytest.mark.parametrize("cap,bias", [(0.0, False), (0.5, True)])
def test_gradients_against_differences(cap, bias):
    q, k, v = (t.requires_grad_(True) for t in _heads(B=1, Sq=5, Sk=5, H=2, Hkv=1, D=3))
    spans = torch.tensor([[0, 1], [1, 1], [0, 3], [2, 5], [1, 4]], dtype=torch.int32)       # a row that sees nothing
    slopes = distance_slopes(2) if bias else None
    assert torch.autograd.gradcheck(lambda *t: F.span_attention(*t, spans, False, 0.8, cap, slopes), (q, k, v))


def test_document_spans():
    docs = torch.tensor([[7, 7, 7, 1, 2, 2, -1, -1], [3, 3, 3, 3, 3, 3, 3, 3]])
    assert F.document_spans(docs)[0].tolist() == [[0, 1], [0, 2], [0, 3], [3, 4], [4, 5], [4, 6], [0, 0], [0, 0]]
    assert F.document_spans(docs, causal=False)[0].tolist() == [[0, 3]] * 3 + [[3, 4]] + [[4, 6]] * 2 + [[0, 0]] * 2
    prefix = torch.tensor([[1, 1, 0, 0, 1, 1, 1, 1], [1, 1, 1, 0, 1, 0, 0, 0]], dtype=torch.bool)
    got = F.document_spans(docs, prefix)
    assert got[0].tolist() == [[0, 2], [0, 2], [0, 3], [3, 4], [4, 6], [4, 6], [0, 0], [0, 0]]
    assert got[1].tolist() == [[0, 3]] * 3 + [[0, 4], [0, 5], [0, 6], [0, 7], [0, 8]]
    assert got.dtype == torch.int32 and F.document_spans(docs[:, :0]).shape == (2, 0, 2)
    with pytest.raises(ValueError):
        F.document_spans(docs.float())
    with pytest.raises(ValueError):
        F.document_spans(docs, prefix.long())


def _pages(ctx, Hkv=2, D=8, page=4, head_major=False):
    g = torch.Generator().manual_seed(1)
    n = sum(-(-c // page) for c in ctx) + 2
    shape = (n, Hkv, page, D) if head_major else (n, page, Hkv, D)
    k, v = (torch.randn(*shape, generator=g, dtype=torch.float64) for _ in range(2))
    order, tables, at = torch.randperm(n, generator=g), torch.zeros(len(ctx), 8, dtype=torch.int32), 0
    for b, c in enumerate(ctx):
        m = -(-c // page)
        tables[b, :m] = order[at:at + m]
        at += m
    return k, v, tables


@pytest.mark.parametrize("head_major", [False, True])
def test_a_token_over_pages_is_the_last_row_of_its_sequence(head_major):
    ctx = [5, 0, 1, 13]
    k, v, tables = _pages(ctx, head_major=head_major)
    q = torch.randn(4, 6, 8, dtype=torch.float64)
    starts, slopes = torch.tensor([2, 0, 0, 12], dtype=torch.int32), distance_slopes(6)
    got = span_decode(q, k, v, tables, torch.tensor(ctx, dtype=torch.int32), 13, cap=3.0, slopes=slopes, starts=starts, head_major=head_major)
    for b, n in enumerate(ctx):
        t = torch.arange(n)
        kk, vv = ((c[tables[b, t // 4].long(), :, t % 4] if head_major else c[tables[b, t // 4].long(), t % 4])[None] for c in (k, v))
        want = F.span_attention(q[b][None, None], kk, vv, torch.tensor([[starts[b], n]], dtype=torch.int32), True, None, 3.0, slopes)
        assert torch.allclose(got[b], want[0, 0], atol=1e-12)


def test_pages_out_of_range_count_as_unseen():
    k, v, tables = _pages([8, 8])
    q = torch.randn(2, 2, 8, dtype=torch.float64)
    tables[0, 0], tables[1, :2] = k.shape[0], -1
    got = span_decode(q, k, v, tables, torch.tensor([8, 8], dtype=torch.int32), 8)
    one = span_decode(q[:1], k, v, tables[:1], torch.tensor([8], dtype=torch.int32), 8, starts=torch.tensor([4], dtype=torch.int32))
    assert torch.allclose(got[0], one[0]) and (got[1] == 0).all()


def test_refusals():
    q, k, v = _heads()
    bad = [(q[0], k, v, {}), (q, k, v[:, :4], {}), (q, k[:1], v[:1], {}), (q[:, :, :3], k, v, {}), (q.float(), k, v, {}), (q, k[..., :4], v[..., :4], {}),
           (q, k, v, dict(cap=-1.0)), (q, k, v, dict(cap=math.nan)), (q, k, v, dict(scale=math.inf)), (q, k, v, dict(slopes=torch.ones(4, dtype=torch.float64))),
           (q, k, v, dict(slopes=torch.ones(2))), (q, k, v, dict(slopes=torch.ones(4, requires_grad=True))), (q, k, v, dict(spans=torch.zeros(9, 2))),
           (q, k, v, dict(spans=torch.zeros(3, 9, 2, dtype=torch.int32))), (q[:, :, :0], k, v, {})]
    for a, b, c, kw in bad:
        with pytest.raises((ValueError, TypeError)):
            F.span_attention(a, b, c, **kw)
    with pytest.raises(TypeError):
        F.span_attention(*(t.long() for t in (q, k, v)))
    k, v, tables = _pages([8])
    q, ctx = torch.randn(1, 2, 8, dtype=torch.float64), torch.tensor([8], dtype=torch.int32)
    for args, kw in [((q, k, v, tables.long(), ctx, 8), {}), ((q, k, v, tables, ctx[:0], 8), {}), ((q, k, v, tables, ctx, -1), {}),
                     ((q, k, v[..., :4], tables, ctx, 8), {}), ((q[:, :1].expand(1, 3, 8), k, v, tables, ctx, 8), {}),
                     ((q, k, v, tables, ctx, 8), dict(starts=ctx.long())), ((q, k, v, tables, ctx, 8), dict(out=q.float())),
                     ((q, k, v, tables, ctx, 8), dict(cap=-2.0))]:
        with pytest.raises(ValueError):
            span_decode(*args, **kw)
    both = torch.randn(4, 2, 8, dtype=torch.float64)
    span_decode(both[:1], k, v, tables, ctx, 8, out=both[1:2])
    for out in (both[:1], k.view(-1)[:16].view(1, 2, 8)):
        with pytest.raises(ValueError, match="apart"):
            span_decode(both[:1], k, v, tables, ctx, 8, out=out)
    with pytest.raises(ValueError):
        distance_slopes(0)


def test_spans_at_any_address_reach_the_kernels_aligned():
    from rumus_b200.ops.span import _spans_arg
    flat = torch.arange(2 * 5 * 2 + 3, dtype=torch.int32)
    for first in range(3):
        spans = flat[first:first + 20].view(2, 5, 2)
        got, rows = _spans_arg(spans, 5)
        assert got.data_ptr() % 8 == 0 and torch.equal(got, spans) and got.is_contiguous() and rows == 5
    assert _spans_arg(flat[1:11].view(5, 2), 5)[1] == 0


def test_the_oracle_decoder_refuses_shaped_scores():
    from rumus_b200.models.gpt import GPTConfig
    from rumus_b200.oracle import OracleDecoder
    for kw in (dict(attn_cap=5.0), dict(alibi=True)):
        with pytest.raises(ValueError, match="oracle"):
            OracleDecoder(dataclasses.replace(GPTConfig.tiny_cpu(), **kw), 2)
