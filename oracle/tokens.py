"""Patch-network operators in float64 from their definitions (test infrastructure):
layer norm, rotary positions of several axes, attention over packed sequences, each
with its gradients from the formulas.

Beside each attention result stands a bound of what a float implementation that
rounds probabilities and score gradients to a type of unit roundoff u may be off:
`slack` terms, element by element, to be multiplied by u."""

from __future__ import annotations

import math

import torch


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    x = x.double()
    mean = x.mean(-1, keepdim=True)
    h = (x - mean) / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + eps)
    y = h if weight is None else h * weight.double()
    return y if bias is None else y + bias.double()


def layer_norm_backward(grad_y, x, weight=None, eps=1e-5):
    """(grad_x, grad_weight, grad_bias) and the sums of the absolute terms of the last two."""
    x, gy = x.double().flatten(0, -2), grad_y.double().flatten(0, -2)
    mean = x.mean(1, keepdim=True)
    r = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    h = (x - mean) * r
    g = gy if weight is None else gy * weight.double()
    gx = r * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
    return (gx.reshape(grad_y.shape), (gy * h).sum(0), gy.sum(0),
            (gy * h).abs().sum(0), gy.abs().sum(0))


def rotary(x, positions, frequencies, sections, interleaved=False, inverse=False):
    x = x.double()
    y = x.clone()
    p = 0
    for axis, n in enumerate(sections):
        for _ in range(n):
            a, b = (2 * p, 2 * p + 1) if interleaved else (p, p + sum(sections))
            angle = positions[:, axis].double() * frequencies[p].double()
            c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
            s = -s if inverse else s
            y[..., a] = x[..., a] * c - x[..., b] * s
            y[..., b] = x[..., a] * s + x[..., b] * c
            p += 1
    return y


def spans(offsets_q, offsets_k, lengths_k, rows_q, rows_k):
    """(first query, end, first key, end of the keys that count) of each sequence."""
    oq, ok = [int(v) for v in offsets_q], [int(v) for v in offsets_k]
    for b in range(len(oq) - 1):
        end = ok[b + 1]
        if lengths_k is not None:
            end = min(end, ok[b] + max(0, int(lengths_k[b])))
        yield oq[b], oq[b + 1], ok[b], end


def attention(q, k, v, offsets_q, offsets_k=None, lengths_k=None, causal=False, scale=None,
              grad_out=None):
    """dict: out, log_sum, out_slack and, with grad_out, gq, gk, gv and their slacks."""
    offsets_k = offsets_q if offsets_k is None else offsets_k
    q, k, v = q.double(), k.double(), v.double()
    group = q.shape[1] // k.shape[1]
    scale = 1 / math.sqrt(q.shape[2]) if scale is None else scale
    res = {"out": torch.zeros_like(q), "out_slack": torch.zeros_like(q),
           "log_sum": torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=q.device)}
    if grad_out is not None:
        go = grad_out.double()
        for name, t in (("gq", q), ("gk", k), ("gv", v)):
            res[name], res[name + "_slack"] = torch.zeros_like(t), torch.zeros_like(t)
    for q0, q1, k0, k1 in spans(offsets_q, offsets_k, lengths_k, q.shape[0], k.shape[0]):
        lq, lk = q1 - q0, k1 - k0
        if lq == 0 or lk == 0:
            continue
        i, j = torch.arange(lq, device=q.device)[:, None], torch.arange(lk, device=q.device)
        seen = (j <= i + lk - lq) if causal else torch.ones_like(i + j, dtype=torch.bool)
        any_seen = seen.any(1, keepdim=True)
        for h in range(q.shape[1]):
            qh, kh, vh = q[q0:q1, h], k[k0:k1, h // group], v[k0:k1, h // group]
            s = torch.where(seen, qh @ kh.T * scale, -math.inf)
            lse = torch.logsumexp(s, 1, keepdim=True)
            p = torch.where(any_seen, torch.exp(s - torch.where(any_seen, lse, 0.0)), 0.0)
            o = p @ vh
            res["out"][q0:q1, h], res["log_sum"][q0:q1, h] = o, lse[:, 0]
            o_slack = 2.5 * (p @ vh.abs())
            res["out_slack"][q0:q1, h] = o_slack
            if grad_out is None:
                continue
            g = go[q0:q1, h]
            ds = p * (g @ vh.T - (g * o).sum(1, keepdim=True))
            ds_slack = 1.5 * ds.abs() + p * (g.abs() * o_slack).sum(1, keepdim=True)
            kv = slice(k0, k1), h // group
            res["gq"][q0:q1, h] = scale * (ds @ kh)
            res["gq_slack"][q0:q1, h] = abs(scale) * (ds_slack @ kh.abs() + (ds @ kh).abs())
            res["gk"][kv] += scale * (ds.T @ qh)
            res["gk_slack"][kv] += abs(scale) * (ds_slack.T @ qh.abs() + (ds.T @ qh).abs())
            res["gv"][kv] += p.T @ g
            res["gv_slack"][kv] += 2.5 * (p.T @ g.abs())
    return res


def attention_gradients(q, k, v, offsets_q, grad_out, offsets_k=None, lengths_k=None, causal=False,
                        scale=None, rest_q=None, rest_k=False):
    """dict: gq, gk, gv, and <name>_bound, how far an implementation in q's type may be off that
    holds its sums in float, rounds weights once, score gradients once (or twice as finely:
    rest_q, by default where q is float16, and rest_k), and takes delta from the output as it was
    before rounding, over the rounded weights.

    With u the type's unit roundoff and e = 2^-24:
    - a score is off by (dim + 16) e sum |q k|, a weight P relatively by that of two scores and
      4 e of the log-sum's size: d;
    - an output is sum P (1 + x) v over sum P (1 + x), |x| <= u + d, so delta is off by the sum of
      |x dS|, doubled where parts of a row are joined by their own sums;
    - dout v and delta are off by (dim + 16) e of their absolute terms, sums over n rows or keys
      by (n / 8 + dim) e of theirs;
    - float16's smallest steps, 2^-25 to either side: of the forward's weights, which are in units
      of a row's largest, of the output's rest, of results; the backward's weights are times 2^10
      and a column's score gradients brought to 2^9, so theirs are 2^-35 and 2^-34 of the largest
      (doubled where the largest came later)."""
    u = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[q.dtype]
    half = q.dtype == torch.float16
    tiny, e, dim = 2.0 ** -25 if half else 0.0, 2.0 ** -24, q.shape[2]
    rest_q = half if rest_q is None else rest_q
    offsets_k = offsets_q if offsets_k is None else offsets_k
    q, k, v, go = q.double(), k.double(), v.double(), grad_out.double()
    group = q.shape[1] // k.shape[1]
    scale = 1 / math.sqrt(dim) if scale is None else scale
    res = {}
    for name, t in (("gq", q), ("gk", k), ("gv", v)):
        res[name], res[name + "_bound"] = torch.zeros_like(t), torch.zeros_like(t)
    for q0, q1, k0, k1 in spans(offsets_q, offsets_k, lengths_k, q.shape[0], k.shape[0]):
        lq, lk = q1 - q0, k1 - k0
        if lq == 0 or lk == 0:
            continue
        i, j = torch.arange(lq, device=q.device)[:, None], torch.arange(lk, device=q.device)
        seen = (j <= i + lk - lq) if causal else torch.ones_like(i + j, dtype=torch.bool)
        for h in range(q.shape[1]):
            kv = slice(k0, k1), h // group
            qh, kh, vh, g = q[q0:q1, h], k[kv], v[kv], go[q0:q1, h]
            s = torch.where(seen, qh @ kh.T * scale, -math.inf)
            lse = torch.logsumexp(s, 1, keepdim=True)
            some = torch.isfinite(lse)
            p = torch.where(some, torch.exp(s - torch.where(some, lse, 0.0)), 0.0)
            o = p @ vh
            away = torch.where(seen, g @ vh.T - (g * o).sum(1, keepdim=True), 0.0)
            ds = p * away
            d = 2 * (dim + 16) * e * (abs(scale) * qh.abs() @ kh.abs().T).amax(1, keepdim=True)
            d = d + 4 * e * (torch.where(some, lse, 0.0).abs() + 1)
            size_o = (g.abs() * o.abs()).sum(1, keepdim=True)
            sizes = g.abs() @ vh.abs().T
            delta = (2 * (u + d) * ds.abs().sum(1, keepdim=True)
                     + 2 * tiny * away.abs().sum(1, keepdim=True) + u * u * size_o
                     + tiny * g.abs().sum(1, keepdim=True)
                     + (lk / 8 + 2 * dim) * e * (p * sizes).sum(1, keepdim=True))
            off = 2 * d * ds.abs() + p * (delta + (dim + 16) * e * (sizes + size_o))
            small = 2.0 ** -33 if half else 0.0
            off_q = off + (u * u if rest_q else u) * ds.abs() + small * ds.abs().amax(1, keepdim=True)
            off_k = off + (u * u if rest_k else u) * ds.abs() + small * ds.abs().amax(0, keepdim=True)
            sum_q, sum_k = (lk / 8 + dim) * e, (lq * group / 8 + dim) * e
            res["gq"][q0:q1, h] = scale * (ds @ kh)
            res["gq_bound"][q0:q1, h] = abs(scale) * ((off_q + sum_q * ds.abs()) @ kh.abs())
            res["gk"][kv] += scale * (ds.T @ qh)
            res["gk_bound"][kv] += abs(scale) * ((off_k + sum_k * ds.abs()).T @ qh.abs())
            res["gv"][kv] += p.T @ g
            res["gv_bound"][kv] += (((u + 2 * d) * p + tiny / 1024).T @ g.abs()
                                    + sum_k * (p.T @ g.abs()))
    for name in ("gq", "gk", "gv"):
        bound = res[name + "_bound"]
        bound += u * (res[name].abs() + bound) + tiny
    return res
