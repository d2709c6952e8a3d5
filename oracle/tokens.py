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
