"""Span attention of one token over pages against its definition in 64 bits."""
import math

import pytest
import torch

from span_oracle import SLACK, check

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def _case(ctx, H, Hkv, D, page, dtype, head_major=False, spread=1.0, seed=0):
    """Pages in random places; what no sequence holds is not a number."""
    g = torch.Generator(device="cuda").manual_seed(seed + H * 31 + D)
    B, per = len(ctx), max(1, -(-max(ctx) // page))
    pages = B * per + 3
    shape = (pages, Hkv, page, D) if head_major else (pages, page, Hkv, D)
    k, v = (torch.randn(*shape, generator=g, device="cuda").to(dtype) for _ in range(2))
    tables = torch.randperm(pages, generator=g, device="cuda")[:B * per].to(torch.int32).view(B, per)
    held = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
    for b, n in enumerate(ctx):
        t = torch.arange(n, device="cuda")
        held[tables[b, t // page].long(), t % page] = True
    for c in (k, v):
        (c.transpose(1, 2) if head_major else c)[~held] = math.nan
    q = (torch.randn(B, H, D, generator=g, device="cuda") * spread).to(dtype)
    return q, k, v, tables, torch.tensor(ctx, dtype=torch.int32, device="cuda")


def _oracle(q, k, v, tables, ctx, scale, cap=0.0, slopes=None, starts=None, head_major=False):
    B, H, D = q.shape
    page = k.shape[2 if head_major else 1]
    Hkv = k.shape[1 if head_major else 2]
    u = torch.finfo(q.dtype).eps / 2
    out, bound = torch.zeros(B, H, D, dtype=torch.float64, device="cuda"), torch.full((B, H, D), 1e-30, dtype=torch.float64, device="cuda")
    for b in range(B):
        n, first = int(ctx[b]), 0 if starts is None else max(0, int(starts[b]))
        t = torch.arange(first, max(n, first), device="cuda")
        blk = tables[b, t // page].long()
        t, blk = t[(blk >= 0) & (blk < k.shape[0])], blk[(blk >= 0) & (blk < k.shape[0])]
        if not len(t):
            continue
        kk, vv = ((c[blk, :, t % page] if head_major else c[blk, t % page]).double().transpose(0, 1).repeat_interleave(H // Hkv, 0) for c in (k, v))
        x = (q[b].double()[:, None] @ kk.transpose(1, 2))[:, 0] * scale
        if cap > 0:
            x = cap * torch.tanh(x / cap)
        if slopes is not None:
            x = x - slopes.double()[:, None] * (n - 1 - t)
        p = torch.softmax(x, -1)[:, None]
        out[b] = (p @ vv)[:, 0]
        # the weights are rounded before they meet the values, and the result
        bound[b] += u * out[b].abs() + (u + SLACK) * (p @ vv.abs())[:, 0]
    return out, bound


def _check(args, H, max_ctx=None, **kw):
    from rumus_b200.ops import native
    from rumus_b200.ops.span import span_decode
    q, k, v, tables, ctx = args
    scale = 1.0 / math.sqrt(q.shape[-1])
    got = span_decode(q, k, v, tables, ctx, max_ctx if max_ctx is not None else int(ctx.max()), **kw)
    assert native.read_status() == 0 and got.dtype == q.dtype
    want, bound = _oracle(q, k, v, tables, ctx, scale, **kw)
    check(got, want, bound, "decode")
    return got


def _slopes(H):
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], device="cuda")


# contexts of nothing, one token, one less and one more than a group of keys, a trip, a page; heads that share keys in every number a CTA holds
@pytest.mark.parametrize("H,Hkv", [(1, 1), (8, 8), (4, 1), (32, 8), (16, 1), (40, 2), (12, 4)])
@pytest.mark.parametrize("cap,bias", [(0.0, False), (30.0, True)])
@pytest.mark.parametrize("head_major", [False, True])
def test_heads(H, Hkv, cap, bias, head_major):
    args = _case([1, 0, 15, 16, 17, 63, 64, 65, 130, 255, 700], H, Hkv, 128, 64, BF, head_major, 2.0)
    got = _check(args, H, cap=cap, slopes=_slopes(H) if bias else None, head_major=head_major)
    assert (got[1] == 0).all()


@pytest.mark.parametrize("D", [8, 24, 64, 72, 80, 128])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("page", [1, 17, 64, 100])
def test_sizes_and_pages(D, dtype, page):
    _check(_case([99, 1, 333], 6, 2, D, page, dtype, spread=2.0), 6, cap=20.0, slopes=_slopes(6))


# every way of cutting: one part, clusters of 2, 4 and 8, more parts than a cluster; contexts shorter than the longest leave parts empty
@pytest.mark.parametrize("B,Hkv,ctx", [(150, 2, 600), (64, 2, 700), (30, 2, 1500), (16, 2, 4000), (2, 2, 6000), (2, 2, 13000), (1, 1, 40000)])
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_parts(B, Hkv, ctx, cap):
    from rumus_b200.ops import native
    lens = [ctx] + [max(0, ctx - 37 * b * b) for b in range(1, B)]
    args = _case(lens, 4 * Hkv, Hkv, 64, 64, BF, spread=2.0)
    splits = native.lib().rb_span_decode_splits(B, 4 * Hkv, Hkv, ctx)
    assert splits == {600: 1, 700: 2, 1500: 4, 4000: 8, 6000: 8, 13000: 26, 40000: 64}[ctx]
    _check(args, 4 * Hkv, cap=cap)
    _check(args, 4 * Hkv, cap=cap, max_ctx=1)          # a wrong bound on the contexts costs time, not results


def test_starts():
    lens = [500, 500, 500, 500, 40, 0, 3000]
    args = _case(lens, 8, 2, 128, 64, BF)
    starts = torch.tensor([0, 499, 500, 900, -7, 0, 1234], dtype=torch.int32, device="cuda")
    got = _check(args, 8, starts=starts, slopes=_slopes(8))
    assert (got[2] == 0).all() and (got[3] == 0).all() and (got[5] == 0).all()
    # a row that sees one key gives its value
    q, k, v, tables, ctx = args
    assert torch.equal(got[1], v[tables[1, 499 // 64].long(), 499 % 64].repeat_interleave(4, 0))


def test_pages_that_the_cache_does_not_have_are_not_read():
    q, k, v, tables, ctx = _case([400, 400, 64], 8, 2, 64, 64, BF)
    tables[0, 2], tables[1, 0], tables[2, 0] = -1, k.shape[0], 2 ** 31 - 1
    got = _check((q, k, v, tables, ctx), 8, cap=10.0)
    assert (got[2] == 0).all()


def test_contexts_beyond_the_table_end_with_it():
    from rumus_b200.ops.span import span_decode
    q, k, v, tables, ctx = _case([128, 128], 4, 2, 64, 64, BF)
    a = span_decode(q, k, v, tables, ctx, 128)
    b = span_decode(q, k, v, tables, torch.tensor([2 ** 31 - 1, 128], dtype=torch.int32, device="cuda"), 128)
    assert torch.equal(a, b)


def test_one_page_of_two_sequences_and_strided_queries():
    q, k, v, tables, ctx = _case([64, 64], 4, 4, 64, 64, HF)
    tables[1] = tables[0]
    wide = torch.randn(2, 3 * 4 * 64, device="cuda").to(HF)
    _check((wide[:, 256:512].view(2, 4, 64), k, v, tables, ctx), 4)
    _check((wide[:, 1:1 + 256].view(2, 4, 64), k, v, tables, ctx), 4)           # no 4-byte boundary


def test_pages_past_32_bits():
    """A pool of more than 2^32 numbers: 9 GB of keys and as much of values, of which three pages are used."""
    page, Hkv, D = 256, 8, 128
    pages = 2 ** 32 // (page * Hkv * D) + 2
    k = torch.empty(pages, page, Hkv, D, dtype=BF, device="cuda")
    v = torch.empty_like(k)
    at = torch.tensor([[pages - 1, 1, pages - 2]], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(0)
    for i in at[0].tolist():
        k[i], v[i] = (torch.randn(page, Hkv, D, generator=g, device="cuda").to(BF) for _ in range(2))
    q = torch.randn(1, 16, D, generator=g, device="cuda").to(BF)
    _check((q, k, v, at, torch.tensor([700], dtype=torch.int32, device="cuda")), 16, cap=30.0)


def test_captured_and_replayed_with_other_contexts():
    from rumus_b200.ops.span import span_decode
    q, k, v, tables, ctx = _case([700, 700, 700], 8, 2, 128, 64, BF)
    for max_ctx in (700, 2 ** 20):
        out = torch.empty_like(q)
        now = ctx.clone()
        span_decode(q, k, v, tables, now, max_ctx, cap=30.0, out=out)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            span_decode(q, k, v, tables, now, max_ctx, cap=30.0, out=out)
        for lens in ([1, 0, 700], [699, 64, 65]):
            now.copy_(torch.tensor(lens, dtype=torch.int32))
            g.replay()
            want, bound = _oracle(q, k, v, tables, now, 1 / math.sqrt(128), cap=30.0)
            check(out, want, bound, str(lens))


def test_two_streams_at_once():
    from rumus_b200.ops.span import span_decode
    a, b = _case([3000] * 4, 8, 2, 128, 64, BF, seed=1), _case([3000] * 4, 8, 2, 128, 64, BF, seed=2)
    want = [span_decode(*x, 3000, cap=30.0) for x in (a, b)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for i, x in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                outs[i].append(span_decode(*x, 3000, cap=30.0))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in outs[i])


def test_refusals():
    from rumus_b200.ops import native
    from rumus_b200.ops.span import span_decode
    q, k, v, tables, ctx = _case([64], 4, 2, 64, 64, BF)
    with pytest.raises(TypeError):
        span_decode(q.float(), k.float(), v.float(), tables, ctx, 64)
    with pytest.raises(ValueError):
        span_decode(q, k.transpose(1, 2), v.transpose(1, 2), tables, ctx, 64, head_major=True)      # pages that are not contiguous
    with pytest.raises(ValueError):
        span_decode(q, k, v, tables.cpu(), ctx, 64)
    L = native.lib()
    assert L.rb_span_decode(2, 0, None, 0, 0, None, None, None, None, None, None, None, None, None, 1, 2, 2, 64, 64, 1, 1, 3, 1.0, 0.0, None) == 20
    assert L.rb_span_decode(2, 0, None, 0, 0, None, None, None, None, None, None, None, None, None, 1, 2, 2, 64, 64, 1, 1, 9, 1.0, 0.0, None) == 20
    assert L.rb_span_decode(2, 0, None, 0, 0, None, None, None, None, None, None, None, None, None, 1, 3, 2, 64, 64, 1, 1, 1, 1.0, 0.0, None) == 20
