"""Span attention: scores that are capped by a tanh and fall with the distance, rows that see a span of keys each.

    x_ij = cap tanh(scale q_i.k_j / cap) - slope_h |i + Sk - Sq - j|      (either part may be missing)
    row i sees the keys lo_i <= j < hi_i, with ``causal`` none behind its own place i + Sk - Sq
    o_i = sum_j softmax(x_i)_j v_j                                         (zeros for a row that sees no key)

Spans cover packed documents, prompts whose beginning is seen by all of it, windows and padding (``document_spans``).  On a GPU one kernel forward and
two backward (``csrc/kernels/span_attention_{fwd,bwd}.cu``; in 32 bits one each, ``span_attention_f32.cu``) and one for a new token over pages
(``span_decode.cu``); long rows in 32 bits go to plain operators where those are faster; on a CPU plain math.  The kernels sum gradients in a fixed order:
the same inputs give the same gradients.
"""
from __future__ import annotations

import math
from contextlib import nullcontext
from ctypes import addressof, c_float, c_int, c_longlong, c_void_p
from typing import Optional

import torch

from . import native
from ._lib import check, count_launch, ptr, stream_ptr

P, LL, I, Fl = c_void_p, c_longlong, c_int, c_float
native.register_signature("rb_span_fwd_splits", [I, I, I, I])
native.register_signature("rb_span_fwd", [I] + [P] * 7 + [LL] + [P] * 6 + [I] * 8 + [Fl, Fl, P])
native.register_signature("rb_span_bwd_parts", [I] * 6)
native.register_signature("rb_span_bwd", [I] + [P] * 7 + [LL] + [P] * 13 + [I] * 8 + [Fl, Fl, P])
native.register_signature("rb_span_f32_fwd", [I] + [P] * 7 + [LL] + [P] * 3 + [I] * 6 + [Fl, Fl, P])
native.register_signature("rb_span_f32_bwd", [I] + [P] * 7 + [LL] + [P] * 8 + [I] * 6 + [Fl, Fl, P])
native.register_signature("rb_span_decode_splits", [I, I, I, I])
native.register_signature("rb_span_decode", [I, I, P, LL, LL] + [P] * 9 + [I] * 8 + [Fl, Fl, P])

CLUSTER = 8             # parts of a context that one launch joins (kSdCluster)
HALVES = (torch.bfloat16, torch.float16)
_LOG2E = math.log2(math.e)


# ---------------------------------------------------------------- spans and slopes
def document_spans(documents: torch.Tensor, prefix: Optional[torch.Tensor] = None, causal: bool = True) -> torch.Tensor:
    """Spans ``int32 [B, S, 2]`` of packed documents.  ``documents``: ``[B, S]`` whole numbers, equal for neighbouring tokens of one document, negative
    for padding (sees nothing, is seen by none).  A token sees its own document: all of it, with ``causal`` up to itself.  ``prefix``: ``[B, S]``
    truth values; with ``causal`` a document's tokens up to the last of its leading run of them see one another (and all later ones of the document
    see them).  For ``span_attention`` with ``causal=False``: the spans stand in the causal mask's place, which would cut a prefix off."""
    if documents.dim() != 2 or documents.dtype.is_floating_point or documents.dtype == torch.bool:
        raise ValueError(f"documents are whole numbers [B, S], not {documents.dtype} {tuple(documents.shape)}")
    B, S = documents.shape
    place = torch.arange(S, device=documents.device).expand(B, S)
    if S == 0:
        return torch.zeros((B, 0, 2), dtype=torch.int32, device=documents.device)
    new = torch.ones((B, S), dtype=torch.bool, device=documents.device)
    new[:, 1:] = documents[:, 1:] != documents[:, :-1]
    lo = torch.where(new, place, 0).cummax(1).values
    last = torch.ones_like(new)
    last[:, :-1] = new[:, 1:]
    end = torch.where(last, place + 1, S).flip(1).cummin(1).values.flip(1)
    hi = torch.minimum(end, place + 1) if causal else end
    if prefix is not None:
        if prefix.shape != documents.shape or prefix.dtype != torch.bool or prefix.device != documents.device:
            raise ValueError(f"a prefix is truth values of the documents' shape {tuple(documents.shape)}, not {prefix.dtype} {tuple(prefix.shape)}")
        # the first token of each document that is no prefix: the least such place at or behind the document's beginning
        stop = torch.where(prefix, S, place).flip(1).cummin(1).values.flip(1)
        hi = torch.maximum(hi, torch.minimum(stop.gather(1, lo), end))
    there = documents >= 0
    return torch.stack([torch.where(there, lo, 0), torch.where(there, hi, 0)], -1).to(torch.int32)


def distance_slopes(heads: int, device=None) -> torch.Tensor:
    """``fp32 [heads]``: 2^(-8 (h + 1) / heads), the geometric slopes of linear distance biases."""
    if heads <= 0:
        raise ValueError(f"{heads} heads")
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], dtype=torch.float32, device=device)


# ---------------------------------------------------------------- arguments
def _f32(x: float) -> float:
    """The nearest 32-bit number, which is what the kernels get."""
    return c_float(x).value


def check_cap(cap: float) -> None:
    """Refuses caps that 32 bits do not hold, in units of log 2 as the kernels have them: what becomes infinite, or zero, which means none."""
    if not (cap >= 0.0 and math.isfinite(_f32(cap * _LOG2E)) and (cap == 0.0 or _f32(cap) > 0.0)):
        raise ValueError(f"a cap is a number of 32 bits above zero, or zero for none, not {cap}")


def _scores_ok(heads: int, device, scale: float, cap: float, slopes) -> None:
    if not math.isfinite(_f32(scale * _LOG2E)):
        raise ValueError(f"a scale is a number of 32 bits, not {scale}")
    check_cap(cap)
    if cap > 0.0 and not math.isfinite(_f32(2.0 * _LOG2E * scale / cap)):           # the tanh's argument of a product of one
        raise ValueError(f"a cap of {cap} is too small for a scale of {scale}")
    if slopes is not None:
        if slopes.dtype != torch.float32 or tuple(slopes.shape) != (heads,) or slopes.device != device:
            raise ValueError(f"slopes are float32 [{heads}] on {device}, not {slopes.dtype} {tuple(slopes.shape)} on {slopes.device}")
        if slopes.requires_grad:
            raise ValueError("slopes are constants: span attention has no gradient for them")


def _rows_ok(q, k, v, spans, scale, cap, slopes) -> None:
    if q.dim() != 4 or k.dim() != 4 or v.shape != k.shape:
        raise ValueError(f"span attention of {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    B, Sq, H, D = q.shape
    Bk, Sk, Hkv, Dk = k.shape
    if Bk != B or Dk != D or D == 0 or H == 0 or Hkv == 0 or H % Hkv:
        raise ValueError(f"span attention of heads {tuple(q.shape)} over {tuple(k.shape)}")
    if not (q.dtype == k.dtype == v.dtype and q.device == k.device == v.device):
        raise ValueError(f"span attention of {q.dtype}, {k.dtype}, {v.dtype} on {q.device}, {k.device}, {v.device}")
    if not q.dtype.is_floating_point:
        raise TypeError(f"span attention of {q.dtype}")
    if spans is not None:
        if spans.dtype != torch.int32 or tuple(spans.shape) not in ((B, Sq, 2), (Sq, 2)) or spans.device != q.device:
            raise ValueError(f"spans are int32 [{B}, {Sq}, 2] or [{Sq}, 2] on {q.device}, not {spans.dtype} {tuple(spans.shape)} on {spans.device}")
    _scores_ok(H, q.device, scale, cap, slopes)


def kernels_cover(dtype: torch.dtype, D: int) -> bool:
    """Whether the 16-bit GPU kernels cover heads of this type and size."""
    return dtype in HALVES and D % 8 == 0 and 0 < D <= 128


def kernels_take(q: torch.Tensor) -> bool:
    """Whether the 16-bit GPU kernels cover heads of this tensor's type and size."""
    return kernels_cover(q.dtype, q.shape[-1])


_HERE = nullcontext()


def _on(device):
    """Makes ``device`` the current one: launches go to its current stream."""
    return _HERE if device.index == torch._C._cuda_getDevice() else torch.cuda.device(device)


def _like(t: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(t, memory_format=torch.contiguous_format)


_Strides = LL * 3


def _view(t: torch.Tensor) -> torch.Tensor:
    """The view itself if the kernels read it in place (rows of neighbouring numbers, 16-byte aligned, no dimension that repeats), else a copy."""
    b, r, h, one = t.stride()
    if one == 1 and t.data_ptr() % 16 == 0:
        if not (b | r | h) & 7 and 0 < b < 2 ** 38 and 0 < r < 2 ** 38 and 0 < h < 2 ** 38:
            return t
        if all(n == 1 or (d > 0 and d % 8 == 0 and d < 2 ** 38) for n, d in zip(t.shape, (b, r, h))):
            return t
    return t.clone(memory_format=torch.contiguous_format)


def _strides(t: torch.Tensor):
    """{batch, row, head} strides of a view as the launchers take them.  A dimension of one element has any stride; the tensor maps want a multiple
    of 16 bytes."""
    b, r, h, _ = t.stride()
    if (b | r | h) & 7 or not (b and r and h):
        b, r, h = (d if n > 1 else t.shape[3] for n, d in zip(t.shape, (b, r, h)))
    return _Strides(b, r, h)


def _spans_arg(spans, rows: int):
    """(contiguous spans, 8-byte aligned: the kernels read lo and hi at once; rows from one batch's to the next's)."""
    if spans is None:
        return None, 0
    spans = spans.contiguous()
    return spans if spans.data_ptr() % 8 == 0 else spans.clone(), rows if spans.dim() == 3 else 0


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the memory that the views span has bytes in common."""
    if a.numel() == 0 or b.numel() == 0 or a.device != b.device:
        return False
    (a0, a1), (b0, b1) = ((t.data_ptr(), t.data_ptr() + (sum((n - 1) * d for n, d in zip(t.shape, t.stride())) + 1) * t.element_size()) for t in (a, b))
    return a0 < b1 and b0 < a1


# ---------------------------------------------------------------- kernels
def _norms(q, k, cap: float, slopes):
    """Room for the lengths of queries and keys, by which biased scores without a cap are known to be too far for a weight; None where they are not noted.
    One pass over both is linear in the rows, what it saves grows with their square.  Without / with it, usual slopes: 2 x 4096 rows, 32 heads over 8 of 128:
    forward 312 / 257 us, backward 993 / 844; 8192 rows, 16 heads over 4: 273 / 187 and 940 / 651; 4 x 2048 rows, 16 heads of 64: 100 / 105 and 281 / 247;
    512 rows over 8192 keys, 32 heads over 8: forward 181 / 193.  One limit serves calls with and without gradients, where either gains: with gradients
    2048 rows would gain too (8 % of the two passes), and do without."""
    if slopes is None or cap > 0 or q.shape[1] < 1024 or k.shape[1] < 4096:
        return None
    return torch.empty((q.shape[0], q.shape[2] + k.shape[2], 32), dtype=torch.float32, device=q.device)


def span_forward(q, k, v, spans, causal: bool, scale: float, cap: float, slopes, out=None, lse: bool = True, norms=None):
    """Heads ``[B, Sq, H, D]`` and, with ``lse``, the rows' log-sum-exp in units of log 2 ``[B, H, Sq]``.  For heads that ``kernels_take``.  ``out``:
    contiguous tensor to write into; ``norms``: from ``_norms``."""
    if not kernels_take(q) or not q.dtype == k.dtype == v.dtype:
        raise TypeError(f"span attention's kernels take bfloat16 or float16 heads of a multiple of 8 numbers up to 128, not {q.dtype}, {k.dtype}, {v.dtype} of "
                        f"{q.shape[3]}")
    q, k, v = _view(q), _view(k), _view(v)
    B, Sq, H, D = q.shape
    Sk, Hkv = k.shape[1], k.shape[2]
    if out is None:
        o = _like(q)
    elif not out.is_contiguous() or out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or out.data_ptr() % 16:
        raise ValueError(f"span attention writes contiguous heads {tuple(q.shape)} of {q.dtype}, not {out.dtype} {tuple(out.shape)}")
    else:
        o = out
    lse2 = q.new_empty((B, H, Sq), dtype=torch.float32) if lse else None
    if o.numel() == 0:
        return o, lse2
    if Sk == 0:
        return o.zero_(), lse2.fill_(float("-inf")) if lse else None
    spans, batch = _spans_arg(spans, Sq)
    if slopes is not None:
        slopes = slopes.contiguous()
    with _on(q.device):
        L = native.lib()
        splits = L.rb_span_fwd_splits(B, H, Sq, Sk)
        part_o = part_lse2 = None
        if splits > 1:
            part_o = torch.empty((splits, B, Sq, H, D), dtype=torch.float32, device=q.device)
            part_lse2 = torch.empty((splits, B, H, Sq), dtype=torch.float32, device=q.device)
        st = _strides(q), _strides(k), _strides(v)
        check(L.rb_span_fwd(native.dtype_code(q.dtype), ptr(q), ptr(k), ptr(v), addressof(st[0]), addressof(st[1]), addressof(st[2]), ptr(spans), batch,
                            ptr(slopes), ptr(norms), ptr(o), ptr(lse2), ptr(part_o), ptr(part_lse2), B, H, Hkv, Sq, Sk, D, splits, int(causal), scale,
                            cap, stream_ptr()), "rb_span_fwd")
        count_launch(1 + (splits > 1) + (norms is not None))
    return o, lse2


def span_backward(q, k, v, spans, causal: bool, scale: float, cap: float, slopes, o, lse2, dout, norms=None):
    """dq, dk, dv.  ``norms``: those of the forward call."""
    B, Sq, H, D = q.shape
    Sk, Hkv = k.shape[1], k.shape[2]
    dq, dk, dv = _like(q), _like(k), _like(v)
    if q.numel() == 0 or k.numel() == 0:
        return dq.zero_(), dk.zero_(), dv.zero_()
    dout = _view(dout)
    spans, batch = _spans_arg(spans, Sq)
    if slopes is not None:
        slopes = slopes.contiguous()
    with _on(q.device):
        rows = B * ((Sq + 63) // 64) * 64
        differ = slopes is not None and (cap > 0 or norms is not None)            # heads reach differently far
        scratch = q.new_empty(rows * (8 * H + 8) + rows // 32 * 16 * (H if slopes is not None else 1), dtype=torch.uint8)
        L, sums = native.lib(), None
        parts = L.rb_span_bwd_parts(B, H, Hkv, Sq, Sk, int(differ))
        if parts > 1:
            sums = torch.empty((parts, B, Hkv, (Sk + 127) // 128 * 128, 2, 64 if D <= 64 else 128), dtype=torch.float32, device=q.device)
        st = _strides(q), _strides(k), _strides(v), _strides(dout), _strides(dq), _strides(dk)
        at = [addressof(s) for s in st]
        check(L.rb_span_bwd(native.dtype_code(q.dtype), ptr(q), ptr(k), ptr(v), at[0], at[1], at[2], ptr(spans), batch, ptr(slopes), ptr(norms), ptr(o), ptr(lse2),
                            ptr(dout), at[3], ptr(scratch), ptr(sums), ptr(dq), ptr(dk), ptr(dv), at[4], at[5], B, H, Hkv, Sq, Sk, D, parts, int(causal),
                            scale, cap, stream_ptr()), "rb_span_bwd")
        count_launch(3 if parts > 1 else 2)
    return dq, dk, dv


class _SpanAttnFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, spans, causal, scale, cap, slopes):
        q, k, v = _view(q), _view(k), _view(v)
        norms = _norms(q, k, cap, slopes)
        o, lse2 = span_forward(q, k, v, spans, causal, scale, cap, slopes, norms=norms)
        ctx.args = causal, scale, cap
        ctx.save_for_backward(q, k, v, spans, slopes, o, lse2, norms)
        return o

    @staticmethod
    def backward(ctx, dout):
        if torch.is_grad_enabled():                 # create_graph: the gradients would look like constants
            raise RuntimeError("span attention has no second derivatives")
        q, k, v, spans, slopes, o, lse2, norms = ctx.saved_tensors
        causal, scale, cap = ctx.args
        dq, dk, dv = span_backward(q, k, v, spans, causal, scale, cap, slopes, o, lse2, dout, norms=norms)
        return dq, dk, dv, None, None, None, None, None


def _span_f32_forward(q, k, v, spans, causal, scale, cap, slopes, lse: bool):
    """(heads, with ``lse`` the rows' natural log-sum-exp).  Views that the kernels read in place."""
    B, Sq, H, D = q.shape
    Sk, Hkv = k.shape[1], k.shape[2]
    o, lse = _like(q), q.new_empty((B, H, Sq)) if lse else None
    if q.numel() == 0 or k.numel() == 0:
        return o.zero_(), lse
    spans, batch = _spans_arg(spans, Sq)
    slopes = None if slopes is None else slopes.contiguous()
    with _on(q.device):
        at = [_strides(t) for t in (q, k, v)]
        check(native.lib().rb_span_f32_fwd(D, ptr(q), ptr(k), ptr(v), *map(addressof, at), ptr(spans), batch, ptr(slopes), ptr(o), ptr(lse), B, H, Hkv, Sq, Sk,
                                           int(causal), scale, cap, stream_ptr()), "rb_span_f32_fwd")
        count_launch()
    return o, lse


class _SpanF32Fn(torch.autograd.Function):
    """Heads of 16, 32, 64 or 128 numbers in 32 bits."""

    @staticmethod
    def forward(ctx, q, k, v, spans, causal, scale, cap, slopes):
        q, k, v = _view(q), _view(k), _view(v)
        o, lse = _span_f32_forward(q, k, v, spans, causal, scale, cap, slopes, True)
        ctx.args = causal, scale, cap
        ctx.save_for_backward(q, k, v, spans, slopes, o, lse)
        return o

    @staticmethod
    def backward(ctx, dout):
        if torch.is_grad_enabled():
            raise RuntimeError("span attention has no second derivatives")
        q, k, v, spans, slopes, o, lse = ctx.saved_tensors
        causal, scale, cap = ctx.args
        B, Sq, H, D = q.shape
        Sk, Hkv = k.shape[1], k.shape[2]
        dq, dk, dv = _like(q), _like(k), _like(v)
        none = (None,) * 5
        if q.numel() == 0 or k.numel() == 0:
            return dq.zero_(), dk.zero_(), dv.zero_(), *none
        dout = _view(dout)
        spans, batch = _spans_arg(spans, Sq)
        slopes = None if slopes is None else slopes.contiguous()
        with _on(q.device):
            at = [_strides(t) for t in (q, k, v, dout)]
            check(native.lib().rb_span_f32_bwd(D, ptr(q), ptr(k), ptr(v), *map(addressof, at[:3]), ptr(spans), batch, ptr(slopes), ptr(o), ptr(lse), ptr(dout),
                                               addressof(at[3]), ptr(dq), ptr(dk), ptr(dv), B, H, Hkv, Sq, Sk, int(causal), scale, cap, stream_ptr()),
                  "rb_span_f32_bwd")
            count_launch()
        return dq, dk, dv, *none


_F32_SIZES = (16, 32, 64, 128)


def _span_f32(q, k, v, spans, causal, scale, cap, slopes, grad: bool):
    """Heads of other sizes as the next size that the kernels have, with zeros behind: they add nothing to a product, and come off again."""
    D = q.shape[3]
    full = next(n for n in _F32_SIZES if n >= D)
    if full != D:
        q, k, v = (torch.nn.functional.pad(t, (0, full - D)) for t in (q, k, v))
    if grad:
        return _SpanF32Fn.apply(q, k, v, spans, causal, scale, cap, slopes)[..., :D]
    return _span_f32_forward(_view(q), _view(k), _view(v), spans, causal, scale, cap, slopes, False)[0][..., :D]


def f32_plain_is_ahead(B: int, H: int, Hkv: int, Sq: int, Sk: int, D: int, causal: bool, grad: bool) -> bool:
    """Whether the plain operators (``_span_f32_plain``) take less time than the 32-bit kernels, for rows without spans.

    us of a call, estimated by what 500 shapes took (heads of 16 to 128, 4 to 128 batches and heads, 1 to 2048 rows, 128 to 4096 keys, 1 to 8 query heads a
    key head).  The kernels take their longest chain, 0.27 a key forward and 0.25 + 0.0015 D a key or row more with gradients, or the multiplications at 2.9
    million a us (0.85 with gradients), whichever is more.  The operators take what the host needs for them, 100 (390), or their passes over the scores.
    The choice was the faster one or within 1.1 of it for 95 of 100, 1.43 at worst.  Kernels / operators, the rule's in brackets: 2 x 2048 tokens, 8 heads of
    128: 1814 / [1368], with gradients 6977 / [3399]; 4 x 1024, 8 of 64: [501] / 543 and 1826 / [1310]; a row over 4096 keys, 4 heads of 64:
    1622 / [76] and 3418 / [310]; 256 tokens, 4 heads of 32: [64] / 105 and [163] / 428; 16 x 256, 8 of 16: [70] / 130 and [183] / 476.

    The operators keep 21 bytes a score: above 2^27 of them (2.8 GB) the kernels serve, which keep none."""
    rows = min(Sq, Sk) if causal else Sq                                      # that see any key
    scores = B * H * rows * Sk
    if scores == 0 or scores > 2 ** 27:
        return False
    D = next(n for n in _F32_SIZES if n >= D)
    work = B * H * D * rows * (Sk - (rows - 1) / 2 if causal else Sk)
    kernels = max(0.27 * Sk, work / 2.9e6)
    if not grad:
        return kernels > max(100.0, scores * (12.0 + 0.067 * D) * 1e-6)
    kernels += max((0.25 + 0.0015 * D) * max(Sk, rows * H // Hkv), work / 0.85e6)
    return kernels > max(390.0, scores * (26.0 + 0.19 * D) * 1e-6)


def _span_f32_plain(q, k, v, causal: bool, scale: float, cap: float, slopes):
    """The plain operators for 32-bit heads on a GPU, few passes over the scores: products with the scale (and the cap's reciprocal) in them, tanh, cap,
    bias, mask, softmax, products."""
    B, Sq, H, D = q.shape
    Sk, Hkv = k.shape[1], k.shape[2]
    first = max(Sq - Sk, 0) if causal else 0                                  # rows before it see no key
    if first:
        seen = _span_f32_plain(q[:, first:], k, v, causal, scale, cap, slopes)
        return torch.cat([seen.new_zeros(B, first, H, D), seen], 1)
    G = H // Hkv
    qh = q.reshape(B, Sq, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B * Hkv, G * Sq, D)
    kh, vh = (t.transpose(1, 2).reshape(B * Hkv, Sk, D) for t in (k, v))
    x = torch.baddbmm(q.new_empty(1, 1, 1), qh, kh.transpose(1, 2), beta=0, alpha=scale / cap if cap > 0 else scale)
    if cap > 0:
        x = torch.tanh(x) * cap
    x = x.view(B, H, Sq, Sk)
    place, key = torch.arange(Sk - Sq, Sk, device=q.device)[:, None], torch.arange(Sk, device=q.device)
    if slopes is not None:
        x = x - slopes.view(-1, 1, 1) * (place - key).abs()
    if causal and Sq > 1:
        x = x.masked_fill(key > place, -math.inf)                             # not added: what unseen keys' products are, infinite too, decides nothing
    o = torch.bmm(torch.softmax(x, -1).view(B * Hkv, G * Sq, Sk), vh)
    return o.view(B, Hkv, G, Sq, D).permute(0, 3, 1, 2, 4).reshape(B, Sq, H, D)


def _f32_plain(q, k, spans, causal: bool, scale: float, cap: float, grad: bool) -> bool:
    """Whether a call in 32 bits goes to the plain operators.  With spans, of which the host knows nothing, the kernels may have far less to do.  The
    operators have to multiply in 32 bits as the kernels do (no TF32, no automatic rounding to 16 bits), and scale / cap goes into their product: above
    1e-30, so that no score is below what 32 bits hold.  A call that is captured takes the kernels: the library of the products cannot be
    loaded then, and a thread's first call may be one.  So does one under torch's deterministic algorithms, which refuse those products."""
    B, Sq, H, D = q.shape
    return (spans is None and f32_plain_is_ahead(B, H, k.shape[2], Sq, k.shape[1], D, causal, grad) and (cap == 0.0 or abs(scale) > 1e-30 * cap)
            and torch.backends.cuda.matmul.fp32_precision in ("none", "ieee") and not torch.is_autocast_enabled("cuda")
            and not torch.are_deterministic_algorithms_enabled() and not torch.cuda.is_current_stream_capturing())


# ---------------------------------------------------------------- plain math
def _weights(raw, distance, seen, slopes, cap: float):
    """Softmax weights of scaled products ``[..., heads, rows, keys]``; rows that see nothing get zeros."""
    if cap > 0:
        raw = torch.tanh(raw / cap) * cap
    if slopes is not None:
        raw = raw - slopes.to(raw.dtype).view(-1, 1, 1) * distance
    top = raw.masked_fill(~seen, -math.inf).amax(-1, keepdim=True) if raw.shape[-1] else raw.new_zeros(raw.shape[:-1] + (1,))
    # masked places take part as zeros, not as exp(-inf - ...): their gradient is zero too, and rows without keys stay finite
    w = torch.exp(torch.where(seen, raw - torch.where(top.isinf(), 0.0, top).detach(), -math.inf))
    total = w.sum(-1, keepdim=True)
    return w / torch.where(total > 0, total, 1.0)


def span_reference(q, k, v, spans=None, causal: bool = True, scale: Optional[float] = None, cap: float = 0.0, slopes=None):
    """The same in plain math (32 bits inside; 64-bit tensors stay so)."""
    B, Sq, H, D = q.shape
    Sk, Hkv = k.shape[1], k.shape[2]
    scale = scale if scale is not None else 1.0 / math.sqrt(D)
    acc = torch.float64 if q.dtype == torch.float64 else torch.float32
    qf, kf, vf = (t.to(acc).transpose(1, 2) for t in (q, k, v))
    if Hkv != H:
        kf, vf = (t.repeat_interleave(H // Hkv, dim=1) for t in (kf, vf))
    place, key = torch.arange(Sq, device=q.device)[:, None] + (Sk - Sq), torch.arange(Sk, device=q.device)
    seen = torch.ones((1, 1, Sq, Sk), dtype=torch.bool, device=q.device)
    if causal:
        seen = seen & (key <= place)
    if spans is not None:
        lo, hi = spans.reshape(-1, 1, Sq, 1, 2).unbind(-1)
        seen = seen & (key >= lo) & (key < hi)
    w = _weights((qf @ kf.transpose(-1, -2)) * scale, (place - key).abs().to(acc), seen, slopes, cap)
    return (w @ vf).transpose(1, 2).to(q.dtype)


# ---------------------------------------------------------------- entry points
def span_attention(q, k, v, spans=None, causal: bool = True, scale: Optional[float] = None, cap: float = 0.0, slopes=None):
    """Span attention of ``q [B, Sq, H, D]`` over ``k, v [B, Sk, Hkv, D]`` (``Hkv`` divides ``H``; strided views are fine), differentiable in q, k and v.

    ``spans``: int32 ``[B, Sq, 2]`` (or ``[Sq, 2]`` for all batches), row i sees the keys ``lo <= j < hi``; parts outside the keys count as cut off, and
    a row with ``hi <= lo`` gives zeros.  ``causal``: besides, no key behind place ``i + Sk - Sq``.  ``cap``: scores s become cap tanh(s / cap), 0: they
    stay.  ``slopes``: float32 ``[H]``, what a score loses per place of distance (constants).

    Scores, scale and cap are 32-bit numbers (a scale or a cap that is none is refused): where even a row's nearest key loses b to the distance, weights (in
    the gradients) are good to 2^-22 b, and under a cap below the rounding of products, 2^-22 of what they are made of, gradients of scores next to zero
    are arbitrary.  Keys and values have to be finite, unseen ones too: a weight of zero times what is not finite is not a number.  On a GPU: bfloat16 or
    float16 with D a multiple of 8 up to 128, float32 with D up to 128 (a kernel for small models, whose rows are serial; long rows without spans take
    plain operators, which keep the scores, up to 2^27 of them)."""
    scale = float(scale) if scale is not None else 1.0 / math.sqrt(q.shape[3]) if q.dim() == 4 and q.shape[3] else 1.0      # else _rows_ok refuses
    cap = float(cap)
    _rows_ok(q, k, v, spans, scale, cap, slopes)
    if not q.is_cuda:
        return span_reference(q, k, v, spans, causal, scale, cap, slopes)
    grad = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    if q.dtype == torch.float32 and q.shape[3] <= 128:
        if _f32_plain(q, k, spans, bool(causal), scale, cap, grad):
            return _span_f32_plain(q, k, v, causal, scale, cap, slopes)
        return _span_f32(q, k, v, spans, bool(causal), scale, cap, slopes, grad)
    if not kernels_take(q):
        raise TypeError(f"span attention on a GPU takes bfloat16 or float16 heads of a multiple of 8 numbers up to 128, or float32 ones up to 128, not "
                        f"{q.dtype} of {q.shape[-1]}")
    if grad:
        return _SpanAttnFn.apply(q, k, v, spans, bool(causal), scale, cap, slopes)
    return span_forward(q, k, v, spans, bool(causal), scale, cap, slopes, lse=False, norms=_norms(q, k, cap, slopes))[0]


def span_decode(q, k_cache, v_cache, block_tables, ctx_lens, max_ctx: int, scale: Optional[float] = None, cap: float = 0.0, slopes=None, starts=None,
                head_major: bool = False, out=None):
    """Span attention of one token per sequence over pages (for serving: no gradients on a GPU): ``q [B, H, D]`` sees the tokens
    ``starts[b] <= t < ctx_lens[b]`` of its sequence, itself the last of them; returns ``[B, H, D]`` (zeros where it sees none).

    Caches ``[pages, page, Hkv, D]``, with ``head_major`` ``[pages, Hkv, page, D]``; ``block_tables`` int32 ``[B, n]``; ``ctx_lens``, ``starts`` (None:
    0) int32 ``[B]``; ``max_ctx``: no context is longer (decides how contexts are cut; longer ones are still right).  Tokens in pages that the cache
    does not have, and behind the table's end, count as unseen; what pages hold behind a context is never read.  ``cap``, ``slopes``: as in
    ``span_attention``.  ``out``: contiguous tensor to write into, 8-byte aligned, apart from the others.  On a GPU: bfloat16 or float16, D a multiple of 8 up to
    128."""
    if q.dim() != 3 or k_cache.dim() != 4 or v_cache.shape != k_cache.shape:
        raise ValueError(f"decoding of {tuple(q.shape)} over pages {tuple(k_cache.shape)}, {tuple(v_cache.shape)}")
    B, H, D = q.shape
    pages, (Hkv, page) = k_cache.shape[0], ((k_cache.shape[1], k_cache.shape[2]) if head_major else (k_cache.shape[2], k_cache.shape[1]))
    if k_cache.shape[3] != D or D == 0 or H == 0 or Hkv == 0 or page == 0 or H % Hkv:
        raise ValueError(f"decoding of heads {tuple(q.shape)} over pages {tuple(k_cache.shape)}")
    if not (q.dtype == k_cache.dtype == v_cache.dtype and q.device == k_cache.device == v_cache.device):
        raise ValueError(f"decoding of {q.dtype}, {k_cache.dtype}, {v_cache.dtype} on {q.device}, {k_cache.device}, {v_cache.device}")
    if not q.dtype.is_floating_point:
        raise TypeError(f"decoding of {q.dtype}")
    ints = [("block_tables", block_tables, 2), ("ctx_lens", ctx_lens, 1)] + ([] if starts is None else [("starts", starts, 1)])
    for name, t, dim in ints:
        if t.dtype != torch.int32 or t.dim() != dim or t.shape[0] != B or t.device != q.device:
            raise ValueError(f"{name}: int32 of {dim} dimensions for {B} sequences on {q.device}, not {t.dtype} {tuple(t.shape)} on {t.device}")
    if max_ctx < 0:
        raise ValueError(f"max_ctx {max_ctx}")
    scale = float(scale) if scale is not None else 1.0 / math.sqrt(D)
    cap = float(cap)
    _scores_ok(H, q.device, scale, cap, slopes)
    if out is None:
        out = q.new_empty((B, H, D))
    elif not out.is_contiguous() or out.shape != q.shape or out.dtype != q.dtype or out.device != q.device or out.data_ptr() % 8:
        raise ValueError(f"decoding writes contiguous heads {tuple(q.shape)} of {q.dtype} on {q.device}, 8-byte aligned, not {out.dtype} {tuple(out.shape)} on "
                         f"{out.device}")
    elif any(_overlap(out, t) for t in (q, k_cache, v_cache)):
        raise ValueError("decoding reads its queries and pages while it writes: ``out`` has to be apart from them")
    if not q.is_cuda:
        return out.copy_(_decode_reference(q, k_cache, v_cache, block_tables, ctx_lens, scale, cap, slopes, starts, head_major))
    if not kernels_take(q):
        raise TypeError(f"decoding on a GPU takes bfloat16 or float16 heads of a multiple of 8 numbers up to 128, not {q.dtype} of {D}")
    if not k_cache.is_contiguous() or not v_cache.is_contiguous() or k_cache.data_ptr() % 16 or v_cache.data_ptr() % 16:
        raise ValueError("the caches' pages are contiguous and 16-byte aligned")
    if out.numel() == 0:
        return out
    sb, sh, sd = q.stride()
    if sd != 1 or sb % 2 or sh % 2 or q.data_ptr() % 4:
        q = q.clone(memory_format=torch.contiguous_format)
        sb, sh, sd = q.stride()
    block_tables, ctx_lens = block_tables.contiguous(), ctx_lens.contiguous()
    if starts is not None:
        starts = starts.contiguous()
    if slopes is not None:
        slopes = slopes.contiguous()
    with _on(q.device):
        L = native.lib()
        splits = L.rb_span_decode_splits(B, H, Hkv, min(int(max_ctx), block_tables.shape[1] * page, 0x7fffffff))
        part_o = part_lse2 = None
        if splits > CLUSTER:
            part_o = torch.empty((splits, B, H, D), dtype=torch.float32, device=q.device)
            part_lse2 = torch.empty((splits, B, H), dtype=torch.float32, device=q.device)
        check(L.rb_span_decode(native.dtype_code(q.dtype), int(head_major), ptr(q), sb, sh, ptr(k_cache), ptr(v_cache),
                               ptr(block_tables), ptr(ctx_lens), ptr(starts), ptr(slopes), ptr(out), ptr(part_o), ptr(part_lse2), B, H, Hkv, D, page,
                               pages, block_tables.shape[1], splits, scale, cap, stream_ptr()), "rb_span_decode")
        count_launch(2 if splits > CLUSTER else 1)
    return out


def _decode_reference(q, k_cache, v_cache, block_tables, ctx_lens, scale, cap, slopes, starts, head_major):
    B, H, D = q.shape
    pages, page = k_cache.shape[0], k_cache.shape[2 if head_major else 1]
    acc = torch.float64 if q.dtype == torch.float64 else torch.float32
    outs = torch.zeros((B, H, D), dtype=acc, device=q.device)
    for b in range(B):
        n = min(int(ctx_lens[b]), block_tables.shape[1] * page)
        t = torch.arange(max(0 if starts is None else int(starts[b]), 0), max(n, 0), device=q.device)
        if t.numel() == 0:
            continue
        blk = block_tables[b, t // page].long()
        there = (blk >= 0) & (blk < pages)
        t, blk = t[there], blk[there]
        kk, vv = ((c[blk, :, t % page] if head_major else c[blk, t % page]).to(acc) for c in (k_cache, v_cache))    # [n, Hkv, D]
        rep = H // kk.shape[1]
        kk, vv = kk.repeat_interleave(rep, 1).transpose(0, 1), vv.repeat_interleave(rep, 1).transpose(0, 1)
        raw = (q[b].to(acc)[:, None] @ kk.transpose(1, 2)) * scale
        w = _weights(raw, (int(ctx_lens[b]) - 1 - t).to(acc), torch.ones_like(raw, dtype=torch.bool), slopes, cap)
        outs[b] = (w @ vv)[:, 0]
    return outs.to(q.dtype)
