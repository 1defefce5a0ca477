"""Span attention in 32 bits where the plain operators are ahead of the kernels: the same bounds against the definition in 64 bits."""
import pytest
import torch

from span_oracle import SLACK, span_oracle
from test_gpu_span import _random_spans, _slopes
from test_gpu_span_f32 import _check, _run

pytestmark = pytest.mark.gpu


# long rows, few rows over many keys, shared key heads, rows before the first key, heads that are no kernel's size
@pytest.mark.parametrize("B,Sq,Sk,H,Hkv,D", [(1, 1500, 1500, 4, 4, 64), (2, 1, 4096, 4, 2, 32), (1, 64, 3000, 8, 1, 128), (1, 1400, 600, 8, 1, 20),
                                             (1, 900, 1300, 8, 8, 80)])
@pytest.mark.parametrize("causal,cap,bias", [(True, 0.0, False), (False, 3.0, False), (True, 3.0, True), (False, 0.0, True)])
def test_sizes(B, Sq, Sk, H, Hkv, D, causal, cap, bias, monkeypatch):
    from rumus_b200.ops import span
    calls = []
    monkeypatch.setattr(span, "_span_f32_plain", lambda *a, f=span._span_f32_plain: calls.append(a) or f(*a))
    got = _check(B, Sq, Sk, H, Hkv, D, 2.0, causal=causal, cap=cap, slopes=_slopes(H) if bias else None)
    assert calls
    if causal and Sq > Sk:
        assert (got["o"][:, :Sq - Sk] == 0).all() and (got["dq"][:, :Sq - Sk] == 0).all()


def test_views_and_without_gradients():
    from rumus_b200.ops import functional as F
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(1, 2048, 3, 4, 64, generator=g, device="cuda")
    q, k, v = x.unbind(2)
    do = torch.randn(1, 2048, 1, 64, generator=g, device="cuda").expand(1, 2048, 4, 64)
    got = _run(q, k, v, do, cap=2.0)
    want, bound = span_oracle(q, k, v, dout=do, cap=2.0)
    for n in got:       # as in the kernels' tests
        assert (got[n].double() - want[n]).norm() <= 2e-5 * want[n].norm() + 2 ** -20 * bound[n].norm() / SLACK, n
    alone = F.span_attention(q, k, v, cap=2.0)
    assert (alone.double() - want["o"]).norm() <= 2e-5 * want["o"].norm()


@pytest.mark.parametrize("cap,bias", [(0.0, False), (3.0, True)])
def test_unseen_keys_of_any_size_decide_nothing(cap, bias):
    """Rows before keys whose products leave 32 bits' range: as if these were ordinary numbers."""
    from rumus_b200.ops import functional as F
    g = torch.Generator(device="cuda").manual_seed(0)
    q, k, v = (torch.randn(1, 2048, 4, 64, generator=g, device="cuda") for _ in range(3))
    kw = dict(cap=cap, slopes=_slopes(4) if bias else None)
    want = F.span_attention(q, k, v, **kw)
    big = torch.finfo(torch.float32).max
    k[:, 2000:], v[:, 2000:] = big / 8 * k[:, 2000:].sign(), big / 8
    assert torch.equal(F.span_attention(q, k, v, **kw)[:, :2000], want[:, :2000])


def test_the_kernels_serve_what_the_operators_do_not(monkeypatch):
    """Rows with spans, and products that would be rounded: the kernels' results, in 32 bits."""
    from rumus_b200.ops import span
    monkeypatch.setattr(span, "_span_f32_plain", None)
    _check(1, 1500, 1500, 4, 4, 64, cap=3.0, spans=_random_spans(1, 1500, 1500))
    monkeypatch.setattr(torch.backends.cuda.matmul, "fp32_precision", "tf32")
    _check(1, 1500, 1500, 4, 4, 64, cap=3.0)


FIRST = """
import torch
from rumus_b200.ops import functional as F, native
native.lib()
g = torch.Generator(device="cuda").manual_seed(0)
leaves = [torch.randn(1, 2048, 4, 64, generator=g, device="cuda").requires_grad_(True) for _ in range(3)]
do = torch.randn(1, 2048, 4, 64, generator=g, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    o = F.span_attention(*leaves, cap=2.0)
    grads = torch.autograd.grad(o, leaves, do)
with torch.no_grad():
    leaves[0].mul_(0.5)
graph.replay()
now = F.span_attention(*leaves, cap=2.0)
for a, b in zip((o, *grads), (now, *torch.autograd.grad(now, leaves, do))):
    assert (a - b).norm() <= 4e-5 * b.norm()          # each within 2e-5 of the definition
print("replayed")
"""


def test_a_process_may_begin_with_a_captured_call():
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST], cwd=root, env={**os.environ, "PYTHONPATH": root}, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "replayed" in r.stdout, r.stderr[-2000:]


def test_deterministic_algorithms():
    """The kernels serve, whose results two runs share."""
    was = torch.are_deterministic_algorithms_enabled()
    try:
        torch.use_deterministic_algorithms(True)
        a, b = (_check(1, 1500, 1500, 4, 4, 64, cap=3.0) for _ in range(2))
    finally:
        torch.use_deterministic_algorithms(was)
    assert all(torch.equal(a[n], b[n]) for n in a)


def test_captured_and_replayed(monkeypatch):
    from rumus_b200.ops import functional as F, span
    g = torch.Generator(device="cuda").manual_seed(0)
    q, k, v = (torch.randn(1, 2048, 4, 64, generator=g, device="cuda") for _ in range(3))
    kw = dict(cap=2.0, slopes=_slopes(4))
    F.span_attention(q, k, v, **kw)
    torch.cuda.synchronize()
    monkeypatch.setattr(span, "_span_f32_plain", None)          # a captured call takes the kernels
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o = F.span_attention(q, k, v, **kw)
    q.copy_(torch.randn(q.shape, generator=g, device="cuda"))
    graph.replay()
    assert torch.equal(o, span._span_f32(q, k, v, None, True, 64 ** -0.5, 2.0, kw["slopes"], False))
