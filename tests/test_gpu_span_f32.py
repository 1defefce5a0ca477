"""Span attention's 32-bit kernels against its definition in 64 bits."""
import pytest
import torch

from span_oracle import SLACK, span_oracle
from test_gpu_span import _random_spans, _slopes

pytestmark = pytest.mark.gpu


def _run(q, k, v, do, **kw):
    from rumus_b200.ops import functional as F, native
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    o = F.span_attention(*leaves, **kw)
    got = dict(zip(("o", "dq", "dk", "dv"), (o.detach(), *torch.autograd.grad(o, leaves, do))))
    assert native.read_status() == 0
    return got


def _check(B, Sq, Sk, H, Hkv, D, spread=1.0, **kw):
    g = torch.Generator(device="cuda").manual_seed(Sq + Sk + D)
    mk = lambda S, h, f=1.0: torch.randn(B, S, h, D, generator=g, device="cuda") * f   # noqa: E731
    q, k, v, do = mk(Sq, H, spread), mk(Sk, Hkv), mk(Sk, Hkv), mk(Sq, H)
    got = _run(q, k, v, do, **kw)
    want, bound = span_oracle(q, k, v, dout=do, **kw)
    for n in got:
        # sums of up to a thousand fp32 numbers (2^-24 sqrt(1000) = 2e-6 as a random walk) with weights whose exponents, up to 50, are off by 2^-24 each:
        # 3e-6 of a weight, and dS, a difference of two such sums, loses a factor of a few.  Where it cancels altogether (one key: dP - delta = 0) what is
        # left is the rounding of both, sums of D products each: 2^-24 sqrt(128) = 2^-20.5 of what the gradient is made of in absolute values, which the
        # oracle's bound is SLACK times of.
        off = (got[n].double() - want[n]).norm()
        assert torch.isfinite(got[n]).all() and off <= 2e-5 * want[n].norm() + 2 ** -20 * bound[n].norm() / SLACK, n
    return got


@pytest.mark.parametrize("Sq,Sk", [(1, 1), (1, 100), (33, 33), (64, 65), (130, 77), (200, 331), (700, 700)])
@pytest.mark.parametrize("causal,cap,bias", [(True, 0.0, False), (False, 3.0, False), (True, 3.0, True), (False, 0.0, True)])
def test_sizes(Sq, Sk, causal, cap, bias):
    _check(2, Sq, Sk, 4, 2, 32, 2.0, causal=causal, cap=cap, slopes=_slopes(4) if bias else None)


@pytest.mark.parametrize("D", [1, 8, 16, 20, 64, 80, 128])
@pytest.mark.parametrize("H,Hkv", [(3, 3), (6, 2)])
def test_heads(D, H, Hkv):
    _check(1, 70, 70, H, Hkv, D, cap=2.0, slopes=_slopes(H), spans=_random_spans(1, 70, 70))


def test_spans_in_any_order():
    spans = _random_spans(2, 150, 150)
    spans = torch.cat([spans.view(-1)[:1], spans.view(-1)])[1:].view(2, 150, 2)           # at an odd address
    got = _check(2, 150, 150, 4, 2, 64, causal=False, spans=spans)
    empty = spans[..., 1].clamp(max=150) <= spans[..., 0].clamp(min=0)
    assert empty.any() and (got["o"][empty] == 0).all() and (got["dq"][empty] == 0).all()


def test_views_and_empty_tensors():
    from rumus_b200.ops import functional as F
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(2, 50, 3, 4, 32, generator=g, device="cuda")
    q, k, v = (x[:, :, i].transpose(1, 2).contiguous().transpose(1, 2) for i in range(3))
    do = torch.randn(2, 50, 1, 32, generator=g, device="cuda").expand(2, 50, 4, 32)
    got = _run(q, k, v, do, cap=2.0)
    want, _ = span_oracle(q, k, v, dout=do, cap=2.0)
    assert all((got[n].double() - want[n]).norm() <= 2e-5 * want[n].norm() for n in got)
    a = F.span_attention(x[:, :, 0], x[:, :, 1], x[:, :, 2], cap=2.0)
    assert torch.equal(a, got["o"])
    for B, Sq, Sk in ((0, 4, 4), (2, 0, 4), (2, 4, 0)):
        z = _run(*(torch.ones(B, S, 2, 16, device="cuda") for S in (Sq, Sk, Sk, Sq)))
        assert all((t == 0).all() for t in z.values())


def test_gradients_against_differences():
    from rumus_b200.ops import functional as F
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k, v, do = (torch.randn(1, 24, 2, 16, generator=g, device="cuda") for _ in range(4))
    kw = dict(spans=_random_spans(1, 24, 24), causal=False, cap=1.5, slopes=_slopes(2))
    got = _run(q, k, v, do, **kw)
    for name, x in (("dq", q), ("dk", k), ("dv", v)):
        d = torch.randn(x.shape, generator=g, device="cuda")
        # central differences: the third derivative leaves h^2, rounding 2^-22 of the sum's terms over h; both near 1e-4 at h = 1e-2
        h, f = 1e-2, lambda y, x=x: (F.span_attention(*(y if t is x else t for t in (q, k, v)), **kw).double() * do.double()).sum()   # noqa: E731
        want = (f(x + h * d) - f(x - h * d)) / (2 * h)
        have = (got[name].double() * d.double()).sum()
        assert abs(have - want) < 2e-3 * got[name].double().norm() * d.double().norm(), name


def test_launchers_refuse_what_they_cannot_do():
    from rumus_b200.ops import native
    n = [None] * 3
    for D, H, Hkv, Sk in ((24, 2, 2, 4), (256, 2, 2, 4), (32, 3, 2, 4), (32, 2, 2, 0)):
        assert native.lib().rb_span_f32_fwd(D, *n, *n, None, 0, None, None, None, 1, H, Hkv, 4, Sk, 1, 1.0, 0.0, None) == 20
        assert native.lib().rb_span_f32_bwd(D, *n, *n, None, 0, *[None] * 8, 1, H, Hkv, 4, Sk, 1, 1.0, 0.0, None) == 20
