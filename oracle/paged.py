"""A paged cache in float64 and plain loops from its definition (test infrastructure): appending,
attention over it with the weights that keys get, and eviction."""

from __future__ import annotations

import math

import torch


def places(tables, lengths, b, page_size, pages):
    """(slot, page, place) of the filled slots of sequence b that are there."""
    row = tables[b].tolist()
    filled = min(max(int(lengths[b]), 0), len(row) * page_size)
    return [(i, row[i // page_size], i % page_size) for i in range(filled)
            if 0 <= row[i // page_size] < pages]


def filled(tables, lengths, b, page_size):
    return min(max(int(lengths[b]), 0), tables.shape[1] * page_size)


def append(k, v, k_pages, v_pages, tables, lengths, offsets, weights=None):
    """New (k_pages, v_pages, weights)."""
    k_pages, v_pages = k_pages.clone(), v_pages.clone()
    weights = None if weights is None else weights.clone()
    pages, size = k_pages.shape[:2]
    at = offsets.tolist()
    for b in range(tables.shape[0]):
        end = min(at[b + 1], k.shape[0])
        for row in range(max(at[b], 0), end):
            slot = int(lengths[b]) - (end - row)
            if not 0 <= slot < tables.shape[1] * size:
                continue
            page = int(tables[b, slot // size])
            if not 0 <= page < pages:
                continue
            k_pages[page, slot % size], v_pages[page, slot % size] = k[row], v[row]
            if weights is not None:
                weights[page, slot % size] = 0
    return k_pages, v_pages, weights


def attention(q, k_pages, v_pages, tables, lengths, offsets, causal=False, scale=None):
    """dict of out, log_sum and out_slack as oracle/tokens.py's; weights, of the pool's first three
    dimensions: what each slot gets; and weights_terms: of how many queries that is the sum."""
    q, kp, vp = q.double(), k_pages.double(), v_pages.double()
    pages, size, key_heads, dim = kp.shape
    group = q.shape[1] // key_heads
    scale = 1 / math.sqrt(dim) if scale is None else scale
    dev = q.device
    res = {"out": torch.zeros_like(q), "out_slack": torch.zeros_like(q),
           "log_sum": torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=dev)}
    got = torch.zeros(pages, size, key_heads, dtype=torch.float64, device=dev)
    terms = torch.zeros_like(got)
    at = offsets.tolist()
    for b in range(tables.shape[0]):
        q0, q1 = max(at[b], 0), min(at[b + 1], q.shape[0])
        there = places(tables, lengths, b, size, pages)
        if q1 <= q0 or not there:
            continue
        slot, page, place = (torch.tensor(x, device=dev) for x in zip(*there))
        i = torch.arange(q1 - q0, device=dev)[:, None]
        last = i + filled(tables, lengths, b, size) - (q1 - q0)
        seen = slot <= last if causal else torch.ones_like(slot <= last)
        some = seen.any(1, keepdim=True)
        for h in range(q.shape[1]):
            qh, kh, vh = q[q0:q1, h], kp[page, place, h // group], vp[page, place, h // group]
            s = torch.where(seen, qh @ kh.T * scale, -math.inf)
            lse = torch.logsumexp(s, 1, keepdim=True)
            p = torch.where(some, torch.exp(s - torch.where(some, lse, 0.0)), 0.0)
            res["out"][q0:q1, h], res["log_sum"][q0:q1, h] = p @ vh, lse[:, 0]
            res["out_slack"][q0:q1, h] = 2.5 * (p @ vh.abs())
            at_head = page, place, torch.full_like(page, h // group)  # (a place may come twice)
            got.index_put_(at_head, p.sum(0), accumulate=True)
            terms.index_put_(at_head, seen.sum(0).double(), accumulate=True)
    return res | {"weights": got, "weights_terms": terms}


def _column(weights, slots, head):
    """The weights of (slot, page, place) of a head."""
    if not slots:
        return []
    _, page, place = (torch.tensor(x, device=weights.device) for x in zip(*slots))
    return weights[page, place, head].tolist()


def evict(k_pages, v_pages, weights, tables, lengths, new_tables, keep, recent=0):
    """(new_lengths, kept, k_pages, v_pages, weights)."""
    out = [t.clone() for t in (k_pages, v_pages, weights)]
    pages, size, heads = weights.shape
    sequences = tables.shape[0]
    kept = torch.full((sequences, heads, keep), -1, dtype=torch.int32)
    new_lengths = torch.zeros(sequences, dtype=torch.int32)
    for b in range(sequences):
        there = places(tables, lengths, b, size, pages)
        end = filled(tables, lengths, b, size)
        late = [x for x in there if x[0] >= end - recent]
        old = [x for x in there if x[0] < end - recent]
        stay = min(keep - len(late), len(old))
        new_lengths[b] = stay + len(late)
        for h in range(heads):
            lines = {x: w for x, w in zip(there, _column(weights, there, h))}

            def rank(x):
                w = lines[x]
                return (-math.inf, -1, x[0]) if w != w else (-w, 0, x[0])
            chosen = sorted(sorted(old, key=rank)[:stay] + late)
            kept[b, h, :len(chosen)] = torch.tensor([x[0] for x in chosen], dtype=torch.int32)
            row = new_tables[b].tolist()
            moves = [(x[1], x[2], row[j // size], j % size) for j, x in enumerate(chosen)
                     if 0 <= row[j // size] < pages]
            if moves:
                page, place, to, at = (torch.tensor(m, device=weights.device) for m in zip(*moves))
                for x, y in zip(out, (k_pages, v_pages, weights)):
                    x[to, at, h] = y[page, place, h]
    return new_lengths, kept, *out


