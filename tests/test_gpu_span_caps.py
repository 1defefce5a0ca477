"""Caps of any size: what is far above the scores changes nothing, over pages as in prompts and gradients."""
import pytest
import torch

from span_oracle import SLACK, span_oracle
from test_gpu_span import _check, _inputs, _slopes
from test_gpu_span_decode import _case, _check as _check_decode, _oracle

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
# scores where the tanh is a straight line, bent and flat; 2e38 is near the largest that 32 bits hold in units of log 2
CAPS = [(2e38, 1.0), (1e30, 2.0), (1e9, 3.0), (1e7, 3.0), (1e5, 3.0), (1e3, 30.0), (50.0, 1.0), (50.0, 12.0), (5.0, 4.0), (1.0, 10.0), (0.01, 3.0)]


# one part, a cluster, through memory
@pytest.mark.parametrize("B,Hkv,ctx", [(150, 2, 300), (2, 2, 6000), (1, 1, 20000)])
@pytest.mark.parametrize("cap,spread", CAPS)
@pytest.mark.parametrize("dtype", [BF, HF])
def test_decoding(B, Hkv, ctx, cap, spread, dtype):
    args = _case([ctx] + [max(0, ctx - 37 * b * b) for b in range(1, B)], 4 * Hkv, Hkv, 64, 64, dtype, spread=spread)
    args[0][:, ::3] *= 0.05
    _check_decode(args, 4 * Hkv, cap=cap)


@pytest.mark.parametrize("cap", [2e38, 1e9, 1e5])
def test_decoding_with_a_bias(cap):
    args = _case([700, 0, 64, 3000], 8, 2, 128, 64, BF, spread=3.0)
    capped = _check_decode(args, 8, cap=cap, slopes=_slopes(8))
    plain = _check_decode(args, 8, slopes=_slopes(8))
    # Each is within ``bound`` of its definition (checked above), and the definitions differ by less than 1e-6 of the weights: scores of up to 40 are
    # lowered by x^3 / (3 cap^2) = 2e-6 at a cap of 1e5.  So they differ by two bounds and what SLACK in them covers.  (One step of the result is too little:
    # a weight that rounds to bfloat16 the other way moves it by 2^-8 of that weight's value, whatever the sum cancels to.)
    _, bound = _oracle(*args, 128 ** -0.5, slopes=_slopes(8))
    assert ((capped.double() - plain.double()).abs() <= 2 * bound).all()


@pytest.mark.parametrize("cap,spread", [c for c in CAPS if c[0] >= 1e7])
@pytest.mark.parametrize("bias", [False, True])
def test_prompts_and_gradients(cap, spread, bias):
    for dtype in (BF, HF):
        q, k, v, do = _inputs(1, 200, 260, 2, 2, 64, dtype, spread)
        _check(q, k, v, do, cap=cap, slopes=_slopes(2) if bias else None)


@pytest.mark.parametrize("cap", [2e38, 1e30, 1e9])
def test_32_bits(cap):
    from test_gpu_span_f32 import _run
    g = torch.Generator(device="cuda").manual_seed(0)
    q, k, v, do = (torch.randn(1, 90, 2, 32, generator=g, device="cuda") for _ in range(4))
    got = _run(q, k, v, do, cap=cap)
    want, bound = span_oracle(q, k, v, dout=do, cap=cap)
    for n in got:       # the bound of the 32-bit kernels' other tests
        assert (got[n].double() - want[n]).norm() <= 2e-5 * want[n].norm() + 2 ** -20 * bound[n].norm() / SLACK, n


# all scores are plus or minus a cap that is next to nothing: every key weighs the same, and nothing reaches the queries
@pytest.mark.parametrize("cap", [1e-30, 1e-37])
def test_caps_far_below_the_scores(cap):
    q, k, v, do = _inputs(1, 100, 130, 2, 2, 64, BF)
    got = _check(q, k, v, do, cap=cap)
    assert (got["dq"] == 0).all() and (got["dk"] == 0).all()
    _check_decode(_case([300, 1, 5000], 4, 2, 64, 64, BF), 4, cap=cap)
