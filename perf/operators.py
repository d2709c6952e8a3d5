"""The operators of a patch network in front of the rasterizer, as cases to time and check.

A network that predicts Gaussians from posed images works on image patches, here the 16x16 tiles
that the rasterizer cuts an image into: 12 tokens for a 64x48 image, 2500 for 800x800, 8160 for
1920x1080, several views to a scene, several scenes of different sizes packed one after another.
Its blocks need, beside matrix products:
  norm       layer_norm over the channels
  rotary     axial_rotary: rotary positions of three axes (view, tile row, tile column)
  attention  packed_attention: grouped heads, causal over a stream of views or over all of a
             scene's tokens, and single new queries over a cache of earlier views
each forward alone (a prediction) or forward and backward (a training step).
"""

from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-5


# ------------------------------------------------------------------ the cases
def _norm(rows, channels, dtype, weight="f32", train=True):
    return dict(op="norm", rows=rows, channels=channels, dtype=dtype, weight=weight, train=train)


def _rotary(tokens, heads, key_heads, dim, rotated, dtype, interleaved=False, train=True):
    return dict(op="rotary", tokens=tokens, heads=heads, key_heads=key_heads, dim=dim,
                rotated=rotated, dtype=dtype, interleaved=interleaved, train=train)


def _attention(sequences, shortest, longest, heads, key_heads, dim, dtype, causal=True,
               queries=0, train=True, spread=0):
    """queries = 0: a token's query, key and value go together; else so many new queries a
    sequence, against a cache of the sequence's length in a slab of `longest` rows."""
    return dict(op="attention", sequences=sequences, shortest=shortest, longest=longest,
                heads=heads, key_heads=key_heads, dim=dim, dtype=dtype, causal=causal,
                queries=queries, train=train, spread=spread)


def listed():
    return [
        # the tokens of one 64x48 image in a small network: latency
        dict(_norm(12, 384, "bf16", "bf16", train=False), name="norm_12x384_bf16"),
        # a training step on one 800x800 view, activations kept in 32 bits
        dict(_norm(2500, 768, "f32"), name="norm_train_2500x768_f32"),
        # channels and rows that no vector width divides
        dict(_norm(8163, 771, "f16", "f16"), name="norm_train_8163x771_f16"),
        # a training step on eight 1080p views, master weights in 32 bits
        dict(_norm(65280, 1024, "bf16"), name="norm_train_65280x1024_bf16"),
        # one view's tokens at a time while views stream in
        dict(_rotary(12, 16, 4, 128, 128, "bf16", train=False), name="rotary_12_bf16"),
        # one 800x800 view in 32 bits, adjacent pairs, the head's end left as it is
        dict(_rotary(2500, 12, 12, 64, 48, "f32", interleaved=True), name="rotary_train_2500_f32"),
        # a training step on eight 1080p views
        dict(_rotary(65280, 16, 4, 128, 128, "bf16"), name="rotary_train_65280_bf16"),
        # new tokens, one a scene, over caches of up to four 1080p views
        dict(_attention(16, 2500, 32640, 16, 4, 128, "bf16", queries=1, train=False, spread=1),
             name="attention_step_16x32640_bf16"),
        # a training step on a few tiny images: latency
        dict(_attention(3, 12, 12, 6, 6, 64, "f16", causal=False, spread=2),
             name="attention_train_3x12_f16"),
        # a prediction from packed scenes of very different sizes, one of a single token
        dict(_attention(7, 1, 8160, 16, 4, 128, "bf16", train=False, spread=3),
             name="attention_7x8160_bf16"),
        # a training step on four 800x800 views, each token with all of its view, odd dimension
        dict(_attention(4, 2500, 2500, 12, 12, 72, "f16", causal=False, spread=4),
             name="attention_train_4x2500_f16"),
        # a training step on two scenes of up to two 1080p views, causal: the largest
        dict(_attention(2, 8160, 16320, 16, 4, 128, "bf16", spread=5),
             name="attention_train_2x16320_bf16"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("norm", "rotary", "attention", "attention"))
    train = rng.random() < 0.6
    if op == "norm":
        return _norm(_log(rng, 1, 65280), _log(rng, 32, 1024), rng.choice(("f32", "f16", "bf16")),
                     train=train)
    if op == "rotary":
        dim = rng.choice((32, 64, 72, 96, 128))
        key_heads = rng.choice((1, 2, 4))
        return _rotary(_log(rng, 1, 65280), key_heads * rng.choice((1, 2, 4)), key_heads, dim,
                       rng.choice((dim, dim // 8 * 6)), rng.choice(("f32", "f16", "bf16")),
                       interleaved=rng.random() < 0.5, train=train)
    dim = rng.choice((32, 64, 72, 96, 128))
    key_heads = rng.choice((1, 2, 4))
    heads = key_heads * rng.choice((1, 2, 4))
    dtype = rng.choice(("f16", "bf16"))
    spread = rng.randrange(1000)
    if rng.random() < 0.35:
        sequences = _log(rng, 1, 24)
        longest = _log(rng, 16, 32640 * 16 // max(sequences, 16))
        return _attention(sequences, max(1, longest // rng.choice((1, 8, 64))), longest, heads,
                          key_heads, dim, dtype, queries=rng.choice((1, 1, 1, 5)), train=False,
                          spread=spread)
    sequences = _log(rng, 1, 12)
    longest = _log(rng, 1, 16320 / math.sqrt(sequences))
    return _attention(sequences, max(1, longest // rng.choice((1, 4, 64))), longest, heads,
                      key_heads, dim, dtype, causal=rng.random() < 0.6, train=train,
                      spread=spread)


def _lengths(case):
    """One sequence of the longest, the others spread over the logarithm of the range."""
    rng = random.Random(case["spread"])
    got = [_log(rng, case["shortest"], case["longest"]) for _ in range(case["sequences"] - 1)]
    got.insert(rng.randrange(len(got) + 1), case["longest"])
    if case["sequences"] > 2 and case["shortest"] < case["longest"]:
        got[got.index(min(got))] = case["shortest"]
    return got


def _sections(pairs):
    """An eighth or so of the pairs for the view, the rest for rows and columns."""
    view = max(1, pairs // 8)
    rows = (pairs - view) // 2
    return (view, rows, pairs - view - rows)


# ----------------------------------------------------------------- the inputs
def _frequencies(sections, base=100.0):
    return [base ** (-i / n) for n in sections for i in range(n)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dev = torch.device("cuda", torch.cuda.current_device())
    dtype = TYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(shape, generator=g, device=dev)

    s = {"op": case["op"], "train": case["train"], "dtype": dtype}
    if case["op"] == "norm":
        n, c = case["rows"], case["channels"]
        # a residual stream: channels of different scales, a few of them large, offsets
        scale = torch.exp(0.5 * randn(c)) * torch.where(randn(c) > 2.2, 12.0, 1.0)
        s["x"] = (randn(n, c) * scale + 0.5 * randn(c)).to(dtype)
        s["w"] = (1.0 + 0.2 * randn(c)).to(TYPES[case["weight"]])
        s["b"] = (0.1 * randn(c)).to(TYPES[case["weight"]])
        leaves, s["gy"] = ("x", "w", "b"), randn(n, c).to(dtype)
    elif case["op"] == "rotary":
        t, hq, hk, d = case["tokens"], case["heads"], case["key_heads"], case["dim"]
        # queries, keys and values of one product, as views into its rows
        qkv = (1.5 * randn(t, hq + 2 * hk, d)).to(dtype)
        s["q"], s["k"] = qkv[:, :hq], qkv[:, hq:hq + hk]
        at = torch.arange(t, device=dev) + torch.randint(0, 8160, (1,), generator=g, device=dev)
        s["positions"] = torch.stack([at // 8160, at // 120 % 68, at % 120], 1).to(torch.int32)
        s["sections"] = _sections(case["rotated"] // 2)
        s["frequencies"] = torch.tensor(_frequencies(s["sections"]), device=dev)
        s["interleaved"] = case["interleaved"]
        s["gq"], s["gk"] = randn(t, hq, d).to(dtype), randn(t, hk, d).to(dtype)
        leaves = ("q", "k")
    else:
        hq, hk, d = case["heads"], case["key_heads"], case["dim"]
        lengths = _lengths(case)
        new = case["queries"]
        s["causal"] = case["causal"]
        s["max_q"], s["max_k"] = new or case["longest"], case["longest"]
        if new:  # a slab of cache for each sequence, filled up to its length
            tq, tk = new * len(lengths), case["longest"] * len(lengths)
            s["q"] = (1.5 * randn(tq, hq, d)).to(dtype)
            s["k"], s["v"] = (1.5 * randn(tk, hk, d)).to(dtype), randn(tk, hk, d).to(dtype)
            step = torch.arange(len(lengths) + 1, device=dev, dtype=torch.int32)
            s["offsets_q"], s["offsets_k"] = step * new, step * case["longest"]
            s["lengths_k"] = torch.tensor(lengths, device=dev, dtype=torch.int32)
        else:
            tq = sum(lengths)
            # queries, keys and values of one product, as views into its rows
            qkv = randn(tq, hq + 2 * hk, d)
            qkv[:, :hq + hk] *= 1.5
            qkv = qkv.to(dtype)
            s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
            ends = torch.tensor([0] + lengths, device=dev).cumsum(0).to(torch.int32)
            s["offsets_q"], s["offsets_k"], s["lengths_k"] = ends, ends, None
        s["go"] = randn(tq, hq, d).to(dtype)
        leaves = ("q", "k", "v")
    if case["train"]:
        for name in leaves:
            s[name].requires_grad_(True)
    return s


# --------------------------------------------------------------- the passes
def _package():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                      "3dgs_from_scratch_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    import cuda_rasterizer

    return cuda_rasterizer


def run(state):
    return {"norm": run_norm, "rotary": run_rotary, "attention": run_attention}[state["op"]](state)


def run_norm(s):
    x, w, b, gy = s["x"], s["w"], s["b"], s["gy"]
    if own:
        y = _package().layer_norm(x, w, b, EPS)
        if not s["train"]:
            return {"y": y}
        gx, gw, gb = torch.autograd.grad(y, (x, w, b), gy)
        return {"y": y, "gx": gx, "gw": gw, "gb": gb}
    with torch.no_grad():
        x, wf = x.float(), w.float()
        centred = x - x.mean(1, keepdim=True)
        r = torch.rsqrt(centred.square().mean(1, keepdim=True) + EPS)
        h = centred * r
        y = (h * wf + b.float()).to(s["dtype"])
        if not s["train"]:
            return {"y": y}
        gy = gy.float()
        g = gy * wf
        gx = r * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
        return {"y": y, "gx": gx.to(s["dtype"]), "gw": (gy * h).sum(0).to(w.dtype),
                "gb": gy.sum(0).to(b.dtype)}


def _turn(x, cos, sin, interleaved, dtype):
    pairs = cos.shape[-1]
    head, tail = x[..., :2 * pairs].float(), x[..., 2 * pairs:]
    cos, sin = cos[:, None], sin[:, None]
    u, v = (head[..., 0::2], head[..., 1::2]) if interleaved else head.split(pairs, -1)
    u, v = u * cos - v * sin, u * sin + v * cos
    head = torch.stack((u, v), -1).flatten(-2) if interleaved else torch.cat((u, v), -1)
    return torch.cat((head.to(dtype), tail), -1)


def run_rotary(s):
    q, k = s["q"], s["k"]
    if own:
        q2, k2 = _package().axial_rotary(q, k, s["positions"], s["frequencies"], s["sections"],
                                         interleaved=s["interleaved"])
        if not s["train"]:
            return {"q": q2, "k": k2}
        gq, gk = torch.autograd.grad((q2, k2), (q, k), (s["gq"], s["gk"]))
        return {"q": q2, "k": k2, "gq": gq, "gk": gk}
    with torch.no_grad():
        a, b, c = s["sections"]
        pos, f = s["positions"].float(), s["frequencies"]
        angle = torch.cat((pos[:, :1] * f[:a], pos[:, 1:2] * f[a:a + b], pos[:, 2:] * f[a + b:]), 1)
        cos, sin = torch.cos(angle), torch.sin(angle)
        how = (s["interleaved"], s["dtype"])
        out = {"q": _turn(q, cos, sin, *how), "k": _turn(k, cos, sin, *how)}
        if s["train"]:
            out |= {"gq": _turn(s["gq"], cos, -sin, *how), "gk": _turn(s["gk"], cos, -sin, *how)}
        return out


def _rows(offsets, lengths, longest):
    """(sequences, longest) row numbers and which of them are a sequence's own."""
    at = torch.arange(longest, device=offsets.device)
    return offsets[:-1, None].long() + at, at < lengths[:, None]


def _padded(x, rows, valid, heads):
    """Packed rows as (sequences * heads, rows * group, dim), zeros where there is no row."""
    n, longest = rows.shape
    x = x.float()[torch.where(valid, rows, 0)] * valid[..., None, None]
    x = x.reshape(n, longest, heads, -1, x.shape[-1]).permute(0, 2, 3, 1, 4)
    return x.reshape(n * heads, -1, x.shape[-1])


def _packed(x, rows, valid, heads, count, dtype):
    """The reverse of _padded, into `count` rows."""
    n, longest = rows.shape
    x = x.reshape(n, heads, -1, longest, x.shape[-1]).permute(0, 3, 1, 2, 4).flatten(2, 3)
    out = torch.zeros((count + 1,) + x.shape[2:], dtype=dtype, device=x.device)
    out[torch.where(valid, rows, count).flatten()] = x.flatten(0, 1).to(dtype)
    return out[:count]


def run_attention(s):
    q, k, v = s["q"], s["k"], s["v"]
    if own:
        o = _package().packed_attention(q, k, v, s["offsets_q"], s["offsets_k"], s["lengths_k"],
                                        causal=s["causal"])
        if not s["train"]:
            return {"o": o}
        gq, gk, gv = torch.autograd.grad(o, (q, k, v), s["go"])
        return {"o": o, "gq": gq, "gk": gk, "gv": gv}
    with torch.no_grad():
        hk, scale = k.shape[1], 1.0 / math.sqrt(q.shape[2])
        lq = s["offsets_q"].diff()
        lk = s["offsets_k"].diff() if s["lengths_k"] is None else s["lengths_k"]
        rq, rk = _rows(s["offsets_q"], lq, s["max_q"]), _rows(s["offsets_k"], lk, s["max_k"])
        qp, kp, vp = _padded(q, *rq, hk), _padded(k, *rk, hk), _padded(v, *rk, hk)
        seen = rk[1][:, None, :] & rq[1][:, :, None]
        if s["causal"]:
            i = torch.arange(s["max_q"], device=q.device)[:, None]
            j = torch.arange(s["max_k"], device=q.device)
            seen = seen & (j <= i + (lk - lq)[:, None, None])
        p = torch.bmm(qp, kp.transpose(1, 2)).mul_(scale)
        shape = (lq.shape[0], hk, -1, s["max_q"], s["max_k"])
        p.view(shape).masked_fill_(~seen[:, None, None], -math.inf)
        top = p.amax(2, keepdim=True)
        p.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
        total = p.sum(2, keepdim=True)
        p.div_(torch.where(total == 0, 1.0, total))
        o = torch.bmm(p, vp)
        out = {"o": _packed(o, *rq, hk, q.shape[0], s["dtype"])}
        if s["train"]:
            go = _padded(s["go"], *rq, hk)
            gv = torch.bmm(p.transpose(1, 2), go)
            ds = torch.bmm(go, vp.transpose(1, 2))
            ds.sub_((go * o).sum(2, keepdim=True)).mul_(p).mul_(scale)
            gq, gk = torch.bmm(ds, kp), torch.bmm(ds.transpose(1, 2), qp)
            out |= {"gq": _packed(gq, *rq, hk, q.shape[0], s["dtype"]),
                    "gk": _packed(gk, *rk, hk, k.shape[0], s["dtype"]),
                    "gv": _packed(gv, *rk, hk, v.shape[0], s["dtype"])}
        return out


# ------------------------------------------------------------------ the work
def work(case):
    size = TYPES[case["dtype"]].itemsize
    if case["op"] == "norm":
        n, c = case["rows"], case["channels"]
        w = TYPES[case["weight"]].itemsize
        if not case["train"]:
            return {"bytes": 2 * n * c * size + 2 * c * w, "flops": 8 * n * c}
        return {"bytes": 4 * n * c * size + 4 * c * w, "flops": 22 * n * c}
    if case["op"] == "rotary":
        elements = case["tokens"] * (case["heads"] + case["key_heads"]) * case["dim"]
        passes = 2 if case["train"] else 1
        return {"bytes": 2 * passes * elements * size + case["tokens"] * 12,
                "flops": 3 * passes * elements}
    lengths, new = _lengths(case), case["queries"]
    pairs = 0
    for n in lengths:
        m = new or n
        both = min(m, n)
        pairs += both * n - both * (both - 1) // 2 if case["causal"] else m * n
    queries = (new * len(lengths) if new else sum(lengths)) * case["heads"] * case["dim"]
    keys = sum(lengths) * case["key_heads"] * case["dim"]
    flops = 4 * case["dim"] * case["heads"] * pairs
    if not case["train"]:
        return {"bytes": 2 * (queries + keys) * size, "flops": flops}
    return {"bytes": (4 * queries + 4 * keys) * size, "flops": flops * 14 // 4}


# ------------------------------------------------------- the same in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    d = {n: (x.detach().double() if torch.is_tensor(x) and x.is_floating_point() else x)
         for n, x in s.items()}
    if case["op"] == "norm":
        c = case["channels"]
        mean = d["x"].sum(1) / c
        away = d["x"] - mean[:, None]
        dev = torch.sqrt((away * away).sum(1) / c + EPS)
        unit = away / dev[:, None]
        out = {"y": d["w"] * unit + d["b"]}
        if case["train"]:
            scaled = d["gy"] * d["w"]
            along = (scaled * unit).sum(1) / c
            out["gx"] = (scaled - scaled.sum(1, keepdim=True) / c - unit * along[:, None]) / dev[:, None]
            out["gw"] = (d["gy"] * unit).sum(0)
            out["gb"] = d["gy"].sum(0)
        return out
    if case["op"] == "rotary":
        axis = [a for a, n in enumerate(d["sections"]) for _ in range(n)]
        pairs = len(axis)
        turn = torch.polar(torch.ones((), dtype=torch.float64, device=d["q"].device),
                           d["positions"].double()[:, axis] * d["frequencies"])[:, None]

        def turned(x, by):
            y = x.clone()
            if d["interleaved"]:
                lo, hi = slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)
            else:
                lo, hi = slice(0, pairs), slice(pairs, 2 * pairs)
            z = torch.complex(x[..., lo], x[..., hi]) * by
            y[..., lo], y[..., hi] = z.real, z.imag
            return y

        out = {"q": turned(d["q"], turn), "k": turned(d["k"], turn)}
        if case["train"]:
            out |= {"gq": turned(d["gq"], turn.conj()), "gk": turned(d["gk"], turn.conj())}
        return out
    q, k, v, go = d["q"], d["k"], d["v"], d["go"]
    group, scale = case["heads"] // case["key_heads"], case["dim"] ** -0.5
    o, gq, gk, gv = (torch.zeros_like(x) for x in (q, q, k, v))
    new = case["queries"]
    at_q = at_k = 0
    for n in _lengths(case):
        m = new or n
        hidden = torch.ones(m, n, dtype=torch.bool, device=q.device).triu(n - m + 1)
        for h in range(case["heads"]):
            rows, keys = slice(at_q, at_q + m), slice(at_k, at_k + n)
            kh, vh = k[keys, h // group], v[keys, h // group]
            score = q[rows, h] @ kh.T * scale
            if case["causal"]:
                score[hidden] = -math.inf
            seen = ~torch.isinf(score).all(1)
            p = torch.zeros_like(score)
            p[seen] = torch.softmax(score[seen], 1)
            o[rows, h] = p @ vh
            if case["train"]:
                gv[keys, h // group] += p.T @ go[rows, h]
                gp = go[rows, h] @ vh.T
                gs = p * (gp - (p * gp).sum(1, keepdim=True)) * scale
                gq[rows, h] = gs @ kh
                gk[keys, h // group] += gs.T @ q[rows, h]
        at_q, at_k = at_q + m, at_k + (case["longest"] if new else n)
    return {"o": o, "gq": gq, "gk": gk, "gv": gv} if case["train"] else {"o": o}
