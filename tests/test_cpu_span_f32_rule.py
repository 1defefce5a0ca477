"""Which 32-bit calls go to the plain operators on a GPU, and that these compute what the reference math does."""
import pytest
import torch

from rumus_b200.ops.span import _f32_plain, _span_f32_plain, distance_slopes, f32_plain_is_ahead, span_reference


# (B, H, Hkv, Sq, Sk, D), and whether the operators took less time forward, and with gradients
@pytest.mark.parametrize("shape,forward,grad", [((2, 8, 8, 2048, 2048, 128), True, True), ((4, 8, 8, 1024, 1024, 64), False, True),
                                                ((1, 4, 4, 1, 4096, 64), True, True), ((1, 4, 4, 256, 256, 32), False, False),
                                                ((16, 8, 8, 256, 256, 16), False, False), ((4, 16, 4, 2048, 2048, 128), False, False),
                                                ((2, 4, 2, 700, 700, 20), True, True), ((1, 4, 4, 0, 64, 16), False, False)])
def test_the_rule_follows_its_measurements(shape, forward, grad):
    assert f32_plain_is_ahead(*shape, True, False) == forward and f32_plain_is_ahead(*shape, True, True) == grad


def test_never_where_the_scores_are_too_many_or_rounded_or_the_call_is_captured(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)       # without a GPU it raises
    q = torch.empty(1, 2048, 8, 128)
    args = (True, 1.0, 0.0, True)
    assert _f32_plain(q, q, None, *args) and not _f32_plain(q, q, torch.zeros(2048, 2, dtype=torch.int32), *args)
    assert not _f32_plain(q, q, None, True, 1.0, 1e31, True) and not f32_plain_is_ahead(8, 32, 32, 2048, 2048, 128, True, True)
    with monkeypatch.context() as m:
        m.setattr(torch, "is_autocast_enabled", lambda kind: kind == "cuda")
        assert not _f32_plain(q, q, None, *args)
    with monkeypatch.context() as m:
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        assert not _f32_plain(q, q, None, *args)
    was = torch.backends.cuda.matmul.fp32_precision
    try:
        torch.backends.cuda.matmul.fp32_precision = "tf32"
        assert not _f32_plain(q, q, None, *args)
    finally:
        torch.backends.cuda.matmul.fp32_precision = was


@pytest.mark.parametrize("Sq,Sk,H,Hkv,D", [(5, 9, 4, 2, 8), (9, 4, 6, 1, 8), (1, 7, 2, 2, 3), (8, 8, 3, 3, 16), (4, 4, 2, 2, 8)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("cap,bias", [(0.0, False), (2.0, False), (0.0, True), (2.0, True)])
def test_the_operators_compute_what_the_reference_does(Sq, Sk, H, Hkv, D, causal, cap, bias):
    g = torch.Generator().manual_seed(Sq + Sk)
    q, k, v, do = (torch.randn(2, S, h, D, generator=g, dtype=torch.float64, requires_grad=True) for S, h in ((Sq, H), (Sk, Hkv), (Sk, Hkv), (Sq, H)))
    slopes = distance_slopes(H).double() if bias else None
    a, b = _span_f32_plain(q, k, v, causal, 0.3, cap, slopes), span_reference(q, k, v, None, causal, 0.3, cap, slopes)
    assert torch.allclose(a, b, atol=1e-12)
    if causal and Sq > Sk:
        assert (a[:, :Sq - Sk] == 0).all()
    for x, y in zip(torch.autograd.grad(a, (q, k, v), do), torch.autograd.grad(b, (q, k, v), do)):
        assert torch.allclose(x, y, atol=1e-12)


def test_never_under_deterministic_algorithms(monkeypatch):
    """They refuse the library's products, unless a variable of the environment is set; the kernels need none."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    q = torch.empty(1, 2048, 8, 128)
    was = torch.are_deterministic_algorithms_enabled()
    try:
        torch.use_deterministic_algorithms(True)
        assert not _f32_plain(q, q, None, True, 1.0, 0.0, True)
    finally:
        torch.use_deterministic_algorithms(was)
    assert _f32_plain(q, q, None, True, 1.0, 0.0, True)
