"""Attention with shaped scores: what is timed, the plain form of it, and the same in 64 bits.

Three uses of one operator, each through the entry points that a user's program calls:

* ``forward``: attention of whole rows of queries without gradients, as a prompt or a portion of one takes it;
* ``train``: attention and its gradients with respect to queries, keys and values;
* ``decode``: one new token per sequence over a cache of pages.

Scores are ``cap tanh(scale q.k / cap) - slope |distance|`` (either part may be missing).  Row i of a batch sees the keys
``lo <= j < hi`` of its span, with ``causal`` none behind its own place; a row that sees no key gives zeros.
Spans are part of a batch (packed documents, prompts whose beginning is seen by all, padding): they are made with it, not in the call.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16}


# ---------------------------------------------------------------- the cases
def _rows(name, kind, batch, rows, keys, heads, kv_heads, dim, dtype="bfloat16", cap=0.0, alibi=False, causal=True, docs=0, prefix=0, pad=0, spread=1.0):
    """``docs``: documents a sequence is packed from (0: no spans); ``prefix``: first tokens of each that see one another; ``pad``: rows
    at the end that see nothing and are seen by none; ``spread``: deviation of the scores."""
    return {"name": name, "kind": kind, "batch": batch, "rows": rows, "keys": keys, "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype,
            "cap": cap, "alibi": alibi, "causal": causal, "docs": docs, "prefix": prefix, "pad": pad, "spread": spread}


def _decode(name, batch, context, heads, kv_heads, dim, page, dtype="bfloat16", cap=0.0, alibi=False, window=0, head_major=False, spread=1.0):
    """``context``: the longest sequence's tokens; ``window``: tokens that stay visible (0: all)."""
    return {"name": name, "kind": "decode", "batch": batch, "context": context, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "dtype": dtype, "cap": cap, "alibi": alibi, "window": window, "head_major": head_major, "spread": spread}


def listed():
    return [
        # a short question to a server whose model caps its scores: nothing but latency
        _rows("short prompt, capped", "forward", 1, 37, 37, 32, 8, 128, cap=50.0, spread=3.0),
        # the next portion of a long prompt: few rows over many keys
        _rows("portion of a long prompt, capped", "forward", 1, 512, 8704, 32, 8, 128, cap=30.0, spread=3.0),
        # whole prompts of a model whose scores fall with the distance
        _rows("prompts, distance bias", "forward", 2, 4096, 4096, 32, 8, 128, alibi=True),
        # pictures before their texts: a beginning that sees all of itself, ragged sizes and heads of 80
        _rows("prefix before text, heads of 80", "forward", 3, 1531, 1531, 16, 16, 80, dtype="float16", causal=False, docs=1, prefix=577, pad=130),
        # fine-tuning of a small model on short packed texts
        _rows("train small packed", "train", 3, 1000, 1000, 12, 4, 64, dtype="float16", causal=False, docs=6, prefix=20, pad=60),
        # a training step's attention of the 350M decoder with a distance bias
        _rows("train 350M, distance bias", "train", 4, 1024, 1024, 8, 8, 128, alibi=True),
        # a training step's attention of the 1.3B decoder on packed documents, scores capped
        _rows("train 1.3B packed, capped", "train", 8, 2048, 2048, 16, 16, 128, cap=50.0, docs=4, spread=3.0),
        # a long sequence, everything at once
        _rows("train long, capped and biased", "train", 1, 8192, 8192, 16, 4, 128, cap=30.0, alibi=True, spread=2.0),
        # a lone user's token
        _decode("decode 1, capped", 1, 1100, 32, 8, 128, 64, cap=50.0, spread=3.0),
        # a busy server's tokens
        _decode("decode 48, distance bias", 48, 1250, 32, 32, 128, 64, alibi=True),
        # long documents, of which a window stays visible
        _decode("decode long, capped, window", 8, 60000, 32, 8, 128, 64, cap=30.0, window=32768, head_major=True, spread=2.0),
        # many short sequences of a small model, pages of an odd size
        _decode("decode 200 small heads", 200, 333, 12, 4, 64, 17, dtype="float16", cap=20.0, alibi=True),
    ]


def _spread_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["forward", "train", "decode"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16"])
    kv_heads = rng.choice([1, 2, 3, 4, 8])
    heads = kv_heads * rng.choice([1, 1, 2, 3, 4, 8])
    cap, alibi, spread = rng.choice([0.0, 10.0, 30.0, 50.0]), rng.random() < 0.5, round(rng.uniform(0.5, 4.0), 2)
    dim = rng.choice([32, 64, 64, 80, 96, 128, 128, 128])
    if kind == "decode":
        batch, page = _spread_int(rng, 1, 200), rng.choice([16, 17, 32, 64, 64, 128])
        room = 2 ** 27 // (batch * kv_heads * dim)           # keys and values of half a GB at most
        context = _spread_int(rng, 1, max(2, min(60000, room)))
        c = _decode("", batch, context, heads, kv_heads, dim, page, dtype, cap, alibi, rng.choice([0, 0, _spread_int(rng, 1, 40000)]), rng.random() < 0.5, spread)
    else:
        pairs = 2.0 ** 28.5                                    # a head's rows x keys, over heads and batches
        rows = _spread_int(rng, 1, 6000)
        while heads * rows * rows > pairs:
            rows = rows * 3 // 4
        keys = rows
        batch = min(8, _spread_int(rng, 1, max(1.01, pairs / (heads * rows * rows))))
        docs, prefix, pad, causal = 0, 0, 0, True
        if rng.random() < 0.6 and rows > 8:
            docs, causal = rng.choice([1, 2, 5]), rng.random() < 0.5
            prefix, pad = (0 if causal else rng.randrange(rows // 2)), rng.choice([0, rng.randrange(rows // 4 + 1)])
        elif kind == "forward":
            room = int(pairs / (heads * rows * batch))
            keys = rows + rng.choice([0, rng.randrange(max(1, min(12000, room - rows)))])
            causal = rng.random() < 0.8
        else:
            causal = rng.random() < 0.8
        c = _rows("", kind, batch, rows, keys, heads, kv_heads, dim, dtype, cap, alibi, causal, docs, prefix, pad, spread)
    del c["name"]
    return c


# ---------------------------------------------------------------- the inputs
def _spans(case, seed):
    """[batch, rows, 2] on the host, or None: packed documents of random lengths, each with its prefix, and padding at the end."""
    if not case["docs"]:
        return None
    rng, n, out = random.Random(seed), case["rows"] - case["pad"], []
    for _ in range(case["batch"]):
        cuts = [0] + sorted(rng.sample(range(1, n), case["docs"] - 1)) + [n]
        spans = []
        for a, b in zip(cuts, cuts[1:]):
            first = min(b, a + case["prefix"])
            spans += [[a, b if case["causal"] else max(first, i + 1)] for i in range(a, b)]
        out.append(spans + [[0, 0]] * case["pad"])
    return torch.tensor(out, dtype=torch.int32)


def _lengths(case, seed):
    """Tokens of each sequence: from a half of the longest to all of it."""
    rng = random.Random(seed)
    return [case["context"]] + [rng.randint((case["context"] + 1) // 2, case["context"]) for _ in range(case["batch"] - 1)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, H, Hkv, D = DTYPES[case["dtype"]], case["heads"], case["kv_heads"], case["dim"]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dt)

    s = {"case": case, "scale": 1.0 / math.sqrt(D), "slopes": None}
    if case["alibi"]:
        s["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / H) for h in range(H)], dtype=torch.float32, device="cuda")
    if case["kind"] == "decode":
        page, B = case["page"], case["batch"]
        lens = _lengths(case, seed)
        per = -(-case["context"] // page)
        order = torch.randperm(B * per + 1, generator=g, device="cuda")[:B * per]
        s["tables"] = order.to(torch.int32).view(B, per)
        s["ctx"] = torch.tensor(lens, dtype=torch.int32).cuda()
        s["max_ctx"] = case["context"]
        s["starts"] = (s["ctx"] - case["window"]).clamp(min=0) if case["window"] else None
        shape = (B * per + 1, Hkv, page, D) if case["head_major"] else (B * per + 1, page, Hkv, D)
        s["k"], s["v"] = normal(*shape), normal(*shape)
        s["q"] = normal(B, H, D, scale=case["spread"])
        return s
    B, Sq, Sk = case["batch"], case["rows"], case["keys"]
    s["q"], s["k"], s["v"] = normal(B, Sq, H, D, scale=case["spread"]), normal(B, Sk, Hkv, D), normal(B, Sk, Hkv, D)
    spans = _spans(case, seed)
    s["spans"] = None if spans is None else spans.cuda()
    if case["kind"] == "train":
        s["do"] = normal(B, Sq, H, D)
        for t in (s["q"], s["k"], s["v"]):
            t.requires_grad_(True)
    return s


# ---------------------------------------------------------------- the plain form
def _weights(raw, rows, keys, visible, slopes, cap):
    """Softmax weights of scaled products ``raw [B, Hkv, G, rows, keys]``; what the cap's derivative is made of beside them."""
    t = None
    if cap > 0:
        t = torch.tanh(raw / cap)
        raw = t * cap
    if slopes is not None:
        raw = raw - slopes.view(raw.shape[1], raw.shape[2], 1, 1) * (rows[..., None] - keys[..., None, :]).abs().float()
    raw = raw.masked_fill(~visible, float("-inf"))
    top = raw.amax(-1, keepdim=True)
    p = torch.exp(raw - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total > 0, total, torch.ones_like(total)), t


def _plain_rows(s):
    case = s["case"]
    B, Sq, Sk, H, Hkv, D = case["batch"], case["rows"], case["keys"], case["heads"], case["kv_heads"], case["dim"]
    dt, scale, cap = DTYPES[case["dtype"]], s["scale"], case["cap"]
    q = s["q"].detach().float().view(B, Sq, Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4)
    k, v = (s[n].detach().float().permute(0, 2, 1, 3).unsqueeze(2) for n in ("k", "v"))
    rows = torch.arange(Sq, device=q.device) + (Sk - Sq)
    keys = torch.arange(Sk, device=q.device)
    visible = torch.ones(1, 1, 1, Sq, Sk, dtype=torch.bool, device=q.device)
    if case["causal"]:
        visible = visible & (keys <= rows[:, None])
    if s["spans"] is not None:
        lo, hi = s["spans"].view(B, 1, 1, Sq, 1, 2).unbind(-1)
        visible = visible & (keys >= lo) & (keys < hi)
    p, t = _weights(torch.matmul(q, k.transpose(-1, -2)) * scale, rows, keys, visible, s["slopes"], cap)
    o = torch.matmul(p, v)

    def back(x, heads):
        return x.permute(0, 3, 1, 2, 4).reshape(B, -1, heads, D).to(dt)

    if case["kind"] == "forward":
        return back(o, H)
    do = s["do"].float().view(B, Sq, Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4)
    dv = torch.matmul(p.transpose(-1, -2), do).sum(2, keepdim=True)
    ds = p * (torch.matmul(do, v.transpose(-1, -2)) - (do * o).sum(-1, keepdim=True))
    if t is not None:
        ds = ds * (1 - t * t)
    ds = ds * scale
    dq, dk = torch.matmul(ds, k), torch.matmul(ds.transpose(-1, -2), q).sum(2, keepdim=True)
    return {"o": back(o, H), "dq": back(dq, H), "dk": back(dk, Hkv), "dv": back(dv, Hkv)}


def _plain_decode(s):
    case = s["case"]
    B, H, Hkv, D = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    k, v = s["k"][s["tables"].long()], s["v"][s["tables"].long()]           # [B, pages, ...]
    if case["head_major"]:
        k, v = k.transpose(2, 3), v.transpose(2, 3)
    k, v = (x.reshape(B, -1, Hkv, D).permute(0, 2, 1, 3).float().unsqueeze(2) for x in (k, v))
    keys = torch.arange(k.shape[3], device=k.device)
    ctx = s["ctx"].view(B, 1, 1, 1, 1)
    visible = keys < ctx
    if s["starts"] is not None:
        visible = visible & (keys >= s["starts"].view(B, 1, 1, 1, 1))
    q = s["q"].float().view(B, Hkv, H // Hkv, 1, D)
    p, _ = _weights(torch.matmul(q, k.transpose(-1, -2)) * s["scale"], ctx[..., 0] - 1, keys, visible, s["slopes"], case["cap"])
    v = v.masked_fill(~visible.transpose(-1, -2), 0.0)          # pages hold what they will behind a sequence's end
    return torch.matmul(p, v).reshape(B, H, D).to(DTYPES[case["dtype"]])


def run(s):
    case = s["case"]
    if not own:
        return _plain_decode(s) if case["kind"] == "decode" else _plain_rows(s)
    from rumus_b200.ops import functional as F
    from rumus_b200.ops.span import span_decode
    if case["kind"] == "decode":
        return span_decode(s["q"], s["k"], s["v"], s["tables"], s["ctx"], s["max_ctx"], scale=s["scale"], cap=case["cap"], slopes=s["slopes"],
                           starts=s["starts"], head_major=case["head_major"])
    o = F.span_attention(s["q"], s["k"], s["v"], spans=s["spans"], causal=case["causal"], scale=s["scale"], cap=case["cap"], slopes=s["slopes"])
    if case["kind"] == "forward":
        return o
    dq, dk, dv = torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])
    return {"o": o.detach(), "dq": dq, "dk": dk, "dv": dv}


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    """Every input read once and every output written once; two operations for each number of each product of a row and a key that it
    sees: two products forward, four more for the gradients."""
    H, Hkv, D = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "decode":
        seen = [min(n, case["window"] or n) for n in _lengths(case, 0)]
        return {"bytes": sum(seen) * Hkv * D * 4 + case["batch"] * (H * D * 4 + 4 * -(-case["context"] // case["page"])), "flops": 4.0 * sum(seen) * H * D}
    B, Sq, Sk = case["batch"], case["rows"], case["keys"]
    spans = _spans(case, 0)
    rows = torch.arange(Sq, dtype=torch.int64) + (Sk - Sq)
    lo, hi = (torch.zeros(B, Sq, dtype=torch.int64), torch.full((B, Sq), Sk)) if spans is None else spans.long().unbind(-1)
    if case["causal"]:
        hi = torch.minimum(hi, rows + 1)
    pairs = int((hi - lo).clamp(min=0).sum()) * H
    numbers = 2 * B * (Sq * H + Sk * Hkv) * D                  # queries and results, keys and values
    grads = case["kind"] == "train"
    if grads:
        numbers += B * (2 * Sq * H + 2 * Sk * Hkv) * D         # the result's gradient, and the three
    return {"bytes": numbers * 2 + (0 if spans is None else spans.numel() * 4), "flops": (12.0 if grads else 4.0) * pairs * D}


# ---------------------------------------------------------------- the definition in 64 bits
def _exact_head(q, k, v, place, lo, hi, scale, cap, slope, do=None):
    """One head, from the definition: ``q [n, D]`` at ``place [n]``, seeing keys ``lo <= j < hi``."""
    j = torch.arange(k.shape[0], device=q.device)
    a = (q @ k.t()) * scale
    slip = None
    if cap > 0:
        a = torch.tanh(a / cap)
        slip = 1 - a.square()
        a = a * cap
    if slope:
        a = a - slope * (place[:, None] - j).abs()
    dark = (j < lo[:, None]) | (j >= hi[:, None])
    a[dark] = -math.inf
    w = torch.softmax(a, -1).nan_to_num_(0.0)
    o = w @ v
    if do is None:
        return o
    g = w * (do @ v.t() - (do * o).sum(-1, keepdim=True)) * scale
    if slip is not None:
        g = g * slip
    return o, g @ k, g.t() @ q, w.t() @ do


def exact(case, seed):
    s = prepare(case, seed)
    H, Hkv, D, B = case["heads"], case["kv_heads"], case["dim"], case["batch"]
    slopes = [0.0] * H if s["slopes"] is None else s["slopes"].double().tolist()
    q = s["q"].detach().double()
    if case["kind"] == "decode":
        out = torch.zeros(B, H, D, dtype=torch.float64, device=q.device)
        for b, n in enumerate(_lengths(case, seed)):
            at = torch.arange(n, device=q.device)
            page, slot = s["tables"][b, at // case["page"]].long(), at % case["page"]
            first = max(0, n - case["window"]) if case["window"] else 0
            for g in range(Hkv):
                k, v = ((x[page, g, slot] if case["head_major"] else x[page, slot, g])[first:].double() for x in (s["k"], s["v"]))
                heads = slice(g * (H // Hkv), (g + 1) * (H // Hkv))
                a = (q[b, heads] @ k.t()) * s["scale"]
                if case["cap"] > 0:
                    a = torch.tanh(a / case["cap"]) * case["cap"]
                a = a - torch.tensor(slopes[heads], dtype=torch.float64, device=q.device)[:, None] * (n - 1 - at[first:]).double()
                out[b, heads] = torch.softmax(a, -1) @ v
        return out
    Sq, Sk = case["rows"], case["keys"]
    place = torch.arange(Sq, device=q.device) + (Sk - Sq)
    k, v = s["k"].detach().double(), s["v"].detach().double()
    do = s["do"].double() if case["kind"] == "train" else None
    o, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for b in range(B):
        lo, hi = (torch.zeros_like(place), torch.full_like(place, Sk)) if s["spans"] is None else s["spans"][b].long().unbind(-1)
        if case["causal"]:
            hi = torch.minimum(hi, place + 1)
        for h in range(H):
            g = h // (H // Hkv)
            r = _exact_head(q[b, :, h], k[b, :, g], v[b, :, g], place, lo, hi, s["scale"], case["cap"], slopes[h], None if do is None else do[b, :, h])
            if do is None:
                o[b, :, h] = r
            else:
                o[b, :, h], dq[b, :, h] = r[0], r[1]
                dk[b, :, g] += r[2]
                dv[b, :, g] += r[3]
    return o if do is None else {"o": o, "dq": dq, "dk": dk, "dv": dv}
