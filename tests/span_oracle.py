"""Span attention in 64 bits, from its definition, and how far results in 16 bits may be from it."""
import math

import torch

# what fp32 sums, exponentials and scores of up to 100 in log2 units leave besides the 16-bit roundings: scores 100 x 2^-22, the exponential 2^-21
SLACK = 1e-4


def seen_of(Sq, Sk, causal, spans, B, device):
    i, j = torch.arange(Sq, device=device)[:, None] + Sk - Sq, torch.arange(Sk, device=device)
    seen = torch.ones(B, Sq, Sk, dtype=torch.bool, device=device)
    if causal:
        seen &= j <= i
    if spans is not None:
        s = spans.long().expand(B, Sq, 2)
        seen &= (j >= s[..., :1]) & (j < s[..., 1:])
    return seen


def span_oracle(q, k, v, spans=None, causal=True, scale=None, cap=0.0, slopes=None, dout=None):
    """{o, lse2, and with ``dout`` dq, dk, dv}, and per result the bound on the error of 16-bit kernels.  A rounding is off by half a step, u = eps / 2 of
    the value: results once; the weights (before P V and P^T dO) and dS (before dS K and dS^T Q) once more, so that what a sum is made of counts in
    absolute values; delta = dO.O takes the rounded O.  fp16 has 10 bits behind the point down to 2^-14 and the same step, 2^-24, below: a weight or
    dS smaller than that is off by up to half of it, 2^-25, whatever its size (weights relative to the row's largest score or to the sum, where none
    counts more than that)."""
    u = torch.finfo(q.dtype).eps / 2
    low = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    B, Sq, H, D = q.shape
    Sk, Hkv = k.shape[1], k.shape[2]
    G = H // Hkv
    scale = scale if scale is not None else 1.0 / math.sqrt(D)
    qd, kd, vd = (t.detach().double().transpose(1, 2) for t in (q, k, v))
    kd, vd = kd.repeat_interleave(G, 1), vd.repeat_interleave(G, 1)
    x = qd @ kd.transpose(-1, -2) * scale
    slip = torch.ones_like(x)
    if cap > 0:
        t = torch.tanh(x / cap)
        x, slip = cap * t, 1 - t * t
    if slopes is not None:
        i, j = torch.arange(Sq, device=q.device)[:, None] + Sk - Sq, torch.arange(Sk, device=q.device)
        x = x - slopes.double().view(-1, 1, 1) * (i - j).abs()
    seen = seen_of(Sq, Sk, causal, spans, B, q.device)[:, None]
    step = low * seen.double()
    x = x.masked_fill(~seen, -math.inf)
    p = torch.softmax(x, -1).nan_to_num(0.0)
    slip = slip * seen
    o = p @ vd
    r = {"o": o, "lse2": torch.logsumexp(x, -1) / math.log(2)}
    e = {"o": u * o.abs() + ((u + SLACK) * p + step) @ vd.abs()}
    if dout is not None:
        g = dout.double().transpose(1, 2)
        dp = g @ vd.transpose(-1, -2)
        delta = (g * o).sum(-1, keepdim=True)
        ds = p * (dp - delta) * slip
        # sizes of what is rounded, and of what rounding O does to delta
        off = (u + SLACK) * ds.abs() + SLACK * p * ((g.abs() @ vd.abs().transpose(-1, -2)) + (g.abs() * o.abs()).sum(-1, keepdim=True)) \
            + p * slip * (g.abs() * e["o"]).sum(-1, keepdim=True) + step
        r["dq"], e_dq = scale * (ds @ kd), abs(scale) * (off @ kd.abs())
        dk, e_dk = scale * (ds.transpose(-1, -2) @ qd), abs(scale) * (off.transpose(-1, -2) @ qd.abs())
        dv, e_dv = p.transpose(-1, -2) @ g, ((u + SLACK) * p + step).transpose(-1, -2) @ g.abs()
        r["dk"], r["dv"], e_dk, e_dv = (t.view(B, Hkv, G, Sk, D).sum(2) for t in (dk, dv, e_dk, e_dv))
        e["dq"], e["dk"], e["dv"] = e_dq + u * r["dq"].abs(), e_dk + u * r["dk"].abs(), e_dv + u * r["dv"].abs()
    tiny = torch.finfo(q.dtype).tiny * torch.finfo(q.dtype).eps if q.dtype == torch.float16 else 0.0     # fp16 results below its normal numbers
    for n in e:
        r[n], e[n] = r[n].transpose(1, 2), e[n].transpose(1, 2) + tiny + 1e-30
    return r, e


def check(got, want, bound, name):
    assert torch.isfinite(got).all(), name
    off = (got.double() - want).abs() / bound
    assert off.max().item() <= 1.0 if off.numel() else True, f"{name}: {off.max().item():.3f} of its bound at {off.argmax().item()}"
