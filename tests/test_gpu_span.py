"""Span attention's kernels against its definition in 64 bits (``span_oracle``: every result within the bound that its roundings give)."""
import random

import pytest
import torch

from span_oracle import check, span_oracle

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def _inputs(B, Sq, Sk, H, Hkv, D, dtype, spread=1.0, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + Sq * 7 + Sk)
    mk = lambda S, h, f=1.0: (torch.randn(B, S, h, D, generator=g, device="cuda") * f).to(dtype)   # noqa: E731
    return mk(Sq, H, spread), mk(Sk, Hkv), mk(Sk, Hkv), mk(Sq, H)


def _slopes(H, f=1.0):
    return torch.tensor([f * 2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], device="cuda")


def _random_spans(B, Sq, Sk, seed=0):
    """Spans without any order: empty ones, single keys, ones that leave the keys at either end."""
    rng = random.Random(seed)
    out = []
    for _ in range(B * Sq):
        kind = rng.randrange(6)
        lo = rng.randint(-5, Sk)
        hi = lo if kind == 0 else lo + 1 if kind == 1 else rng.randint(lo, Sk + 5)
        out.append([0, Sk] if kind == 2 else [hi, lo - 1] if kind == 3 else [lo, hi])
    return torch.tensor(out, dtype=torch.int32, device="cuda").view(B, Sq, 2)


def _run(q, k, v, do, **kw):
    from rumus_b200.ops import functional as F, native
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    o = F.span_attention(*leaves, **kw)
    grads = torch.autograd.grad(o, leaves, do)
    assert native.read_status() == 0
    return dict(zip(("o", "dq", "dk", "dv"), (o.detach(), *grads)))


def _check(q, k, v, do, **kw):
    got = _run(q, k, v, do, **kw)
    want, bound = span_oracle(q, k, v, dout=do, **kw)
    for n in got:
        assert got[n].dtype == q.dtype
        check(got[n], want[n], bound[n], n)
    return got


# one row and one key, tiles with an end inside, one more and one less than a tile, fewer rows than keys and the other way round
SHAPES = [(1, 1), (1, 130), (2, 64), (63, 63), (64, 65), (127, 128), (129, 129), (130, 77), (256, 256), (257, 300), (300, 1100)]


@pytest.mark.parametrize("Sq,Sk", SHAPES)
@pytest.mark.parametrize("causal,cap,bias", [(True, 0.0, False), (False, 30.0, False), (True, 0.0, True), (True, 30.0, True), (False, 0.0, True)])
def test_sizes(Sq, Sk, causal, cap, bias):
    q, k, v, do = _inputs(2, Sq, Sk, 4, 2, 128, BF, spread=2.0)
    _check(q, k, v, do, causal=causal, cap=cap, slopes=_slopes(4) if bias else None)


@pytest.mark.parametrize("D", [8, 16, 40, 64, 72, 80, 96, 120, 128])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("cap,bias", [(0.0, False), (20.0, True)])
def test_head_sizes(D, dtype, cap, bias):
    q, k, v, do = _inputs(1, 200, 200, 3, 3, D, dtype, spread=1.5)
    _check(q, k, v, do, cap=cap, slopes=_slopes(3) if bias else None, spans=_random_spans(1, 200, 200))


@pytest.mark.parametrize("H,Hkv", [(1, 1), (6, 1), (6, 2), (8, 8), (20, 4)])
def test_shared_key_heads(H, Hkv):
    q, k, v, do = _inputs(2, 150, 150, H, Hkv, 64, BF)
    _check(q, k, v, do, cap=10.0, slopes=_slopes(H))


# scores from where the cap is a straight line to where it is flat: both forms of the tanh, and rows that take one each
@pytest.mark.parametrize("cap,spread", [(1e6, 1.0), (50.0, 1.0), (50.0, 12.0), (5.0, 4.0), (1.0, 10.0), (0.01, 3.0)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_caps(cap, spread, dtype):
    q, k, v, do = _inputs(1, 260, 260, 2, 2, 64, dtype, spread)
    q[:, ::3] *= 0.05
    _check(q, k, v, do, cap=cap)


@pytest.mark.parametrize("scale", [0.0, -0.2, 1.0])
@pytest.mark.parametrize("cap", [0.0, 8.0])
def test_scales(scale, cap):
    q, k, v, do = _inputs(1, 140, 200, 2, 2, 64, BF)
    _check(q, k, v, do, cap=cap, scale=scale)


# slopes that are steep, zero and below zero (the far keys win), both sides of the diagonal
@pytest.mark.parametrize("slopes", [[4.0, 0.0, -0.02], [-0.05, 1e-4, 0.3]])
@pytest.mark.parametrize("causal", [True, False])
def test_slopes(slopes, causal):
    q, k, v, do = _inputs(1, 333, 333, 3, 1, 64, BF)
    _check(q, k, v, do, causal=causal, slopes=torch.tensor(slopes, device="cuda"))


@pytest.mark.parametrize("Sq,Sk", [(70, 70), (300, 300), (300, 520), (520, 300)])
@pytest.mark.parametrize("causal", [True, False])
def test_spans_in_any_order(Sq, Sk, causal):
    q, k, v, do = _inputs(2, Sq, Sk, 4, 2, 128, BF)
    got = _check(q, k, v, do, causal=causal, spans=_random_spans(2, Sq, Sk), cap=15.0, slopes=_slopes(4))
    spans = _random_spans(2, Sq, Sk)
    empty = spans[..., 1].clamp(max=Sk) <= spans[..., 0].clamp(min=0)
    assert empty.any() and (got["o"][empty] == 0).all() and (got["dq"][empty] == 0).all()


def test_no_row_sees_anything():
    q, k, v, do = _inputs(1, 200, 200, 2, 2, 64, BF)
    got = _run(q, k, v, do, spans=torch.zeros(200, 2, dtype=torch.int32, device="cuda"))
    assert all((t == 0).all() for t in got.values())


def test_empty_tensors():
    from rumus_b200.ops import functional as F
    for B, Sq, Sk in ((0, 4, 4), (2, 0, 4), (2, 4, 0)):
        q, k, v, do = _inputs(B, Sq, Sk, 2, 1, 64, BF)
        got = _run(q, k, v, do)
        assert all((t == 0).all() for t in got.values()) and got["o"].shape == q.shape and got["dk"].shape == k.shape
    assert F.span_attention(*_inputs(1, 3, 0, 2, 2, 64, BF)[:3]).shape == (1, 3, 2, 64)


def test_documents_with_prefixes_and_padding():
    from rumus_b200.ops import functional as F
    docs = torch.tensor([[0] * 130 + [1] * 1 + [2] * 250 + [-1] * 19, [5] * 399 + [-1]], device="cuda")
    prefix = torch.zeros(docs.shape, dtype=torch.bool, device="cuda")
    prefix[0, 131:200] = True
    prefix[1, :256] = True
    spans = F.document_spans(docs, prefix)
    q, k, v, do = _inputs(2, 400, 400, 4, 4, 128, BF)
    got = _check(q, k, v, do, causal=False, spans=spans, cap=50.0)
    assert (got["o"][0, 381:] == 0).all() and (got["dk"][0, 381:] == 0).all()
    # a document alone gives what it gives in the pack
    alone = _run(*(t[:1, 131:381] for t in (q, k, v, do)), causal=False, spans=spans[:1, 131:381] - 131, cap=50.0)
    want, bound = span_oracle(q[:1, 131:381], k[:1, 131:381], v[:1, 131:381], spans=spans[:1, 131:381] - 131, causal=False, cap=50.0)
    check(alone["o"], want["o"], bound["o"], "alone")
    check(got["o"][:1, 131:381], want["o"], bound["o"], "packed")


# unseen keys of large numbers change nothing, also in tiles that seen ones share
def test_unseen_keys_do_not_matter():
    q, k, v, do = _inputs(1, 100, 300, 2, 2, 64, BF)
    spans = torch.tensor([[70, 190]], dtype=torch.int32, device="cuda").expand(100, 2)
    a = _run(q, k, v, do, causal=False, spans=spans)
    big = torch.finfo(BF).max / 2
    k2, v2 = k.clone(), v.clone()
    k2[:, :70], k2[:, 190:], v2[:, :70], v2[:, 190:] = -1e4, 1e4, big, -big
    b = _run(q, k2, v2, do, causal=False, spans=spans)
    assert torch.equal(a["o"], b["o"]) and torch.equal(a["dq"], b["dq"])
    assert torch.equal(a["dk"][:, 70:190], b["dk"][:, 70:190]) and (b["dk"][:, :70] == 0).all() and (b["dv"][:, 190:] == 0).all()


def test_views_and_layouts():
    B, S, H, Hkv, D = 2, 190, 4, 2, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    qkv = torch.randn(B, S, (H + 2 * Hkv) * D, generator=g, device="cuda").to(BF)
    q, k, v = qkv.split([H * D, Hkv * D, Hkv * D], -1)
    q, k, v = q.view(B, S, H, D), k.view(B, S, Hkv, D), v.view(B, S, Hkv, D)
    do = torch.randn(B, H, S, D, generator=g, device="cuda").to(BF).transpose(1, 2)
    a = _check(q, k, v, do, cap=20.0)                                        # slices of a projection, heads before rows
    odd = torch.randn(B * S * H * D + 3, generator=g, device="cuda").to(BF)[3:].view(B, S, H, D)      # no 16-byte boundary
    _check(odd, k, v, do.expand(B, S, H, D), cap=20.0)
    one = k[:, :, :1].expand(B, S, Hkv, D)                                   # a dimension that repeats
    _check(q, one, v, do[:, :1].expand(B, S, H, D), cap=20.0)
    _check(q.flip(3).transpose(2, 3).contiguous().transpose(2, 3), k, v, do)  # numbers of a row apart
    assert a["dk"].shape == k.shape


def test_same_inputs_same_gradients_on_any_stream():
    q, k, v, do = _inputs(2, 500, 500, 8, 2, 128, BF)
    a = _run(q, k, v, do, cap=30.0, slopes=_slopes(8))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = _run(q, k, v, do, cap=30.0, slopes=_slopes(8))
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a[n], b[n]) for n in a)


def test_captured_and_replayed():
    from rumus_b200.ops import functional as F, native
    q, k, v, do = _inputs(1, 300, 300, 4, 4, 128, BF)
    st = [t.clone().requires_grad_(True) for t in (q, k, v)]
    spans = _random_spans(1, 300, 300)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(F.span_attention(*st, spans=spans, cap=9.0), st, do)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = F.span_attention(*st, spans=spans, cap=9.0)
        grads = torch.autograd.grad(o, st, do)
    with torch.no_grad():
        for t, n in zip(st, _inputs(1, 300, 300, 4, 4, 128, BF, seed=5)):
            t.copy_(n)
    g.replay()
    want = _run(*(t.detach() for t in st), do, spans=spans, cap=9.0)
    assert torch.equal(o.detach(), want["o"]) and all(torch.equal(a, want[n]) for a, n in zip(grads, ("dq", "dk", "dv")))
    assert native.read_status() == 0


# few rows over many keys: the keys are cut into parts
@pytest.mark.parametrize("Sq,Sk,H,cap", [(1, 5000, 2, 0.0), (40, 9000, 4, 30.0), (300, 4096, 2, 0.0)])
def test_parts_of_long_rows(Sq, Sk, H, cap):
    from rumus_b200.ops import native
    assert native.lib().rb_span_fwd_splits(1, H, Sq, Sk) > 1
    q, k, v, do = _inputs(1, Sq, Sk, H, 1, 128, BF, spread=2.0)
    _check(q, k, v, do, cap=cap, slopes=_slopes(H))
    lo = torch.randint(0, Sk, (1, Sq), device="cuda")
    spans = torch.stack([lo, lo + torch.randint(0, Sk, (1, Sq), device="cuda")], -1).to(torch.int32)
    _check(q, k, v, do, cap=cap, spans=spans, causal=False)


def test_refusals():
    from rumus_b200.ops import functional as F
    q, k, v, _ = _inputs(1, 16, 16, 4, 2, 64, BF)
    for bad in (dict(q=q.double(), k=k.double(), v=v.double()), dict(q=q[..., :60], k=k[..., :60], v=v[..., :60]),
                dict(q=torch.cat([q, q, q], -1), k=torch.cat([k, k, k], -1), v=torch.cat([v, v, v], -1))):
        with pytest.raises(TypeError):
            F.span_attention(**bad)
    with pytest.raises(ValueError):
        F.span_attention(q, k.cpu(), v.cpu())
    with pytest.raises(ValueError):
        F.span_attention(q, k, v, slopes=torch.ones(4))
    with pytest.raises(ValueError):
        F.span_attention(q, k, v, spans=torch.zeros(16, 2, dtype=torch.int32))


def test_second_derivatives_are_refused():
    from rumus_b200.ops import functional as F
    q, k, v, do = _inputs(1, 16, 16, 2, 2, 64, BF)
    q.requires_grad_(True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(F.span_attention(q, k, v), q, do, create_graph=True)


def test_launchers_refuse_what_they_cannot_do():
    from rumus_b200.ops import native
    L = native.lib()
    none = [None] * 3
    for D, H, Hkv, splits in ((136, 2, 2, 1), (12, 2, 2, 1), (64, 3, 2, 1), (64, 2, 2, 2)):
        assert L.rb_span_fwd(2, *none, *none, None, 0, None, None, None, None, None, None, 1, H, Hkv, 4, 4, D, splits, 1, 1.0, 0.0, None) == 20
