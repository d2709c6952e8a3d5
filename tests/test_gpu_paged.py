"""GPU parity of the paged cache's operators (paged_append, paged_attention, paged_evict) against
the oracle (oracle/paged.py), with NaN and infinities in every place of the pool that is no
sequence's filled slot.

Tolerances, with u the unit roundoff of the pool's type (2^-11, 2^-8) and e = 2^-24:
- what is moved is compared bit for bit;
- attention: the oracle's `slack` times u (probabilities rounded to the type, the output too), a
  float16 probability below 2^-14 absolutely, 2^-24 of the largest value at most each; scores in
  float add (dim + 16) e of sum |q k|, relative to a probability;
- a slot's weight: a probability exp(s - L) is off relatively by that of the score and of the
  log-sum, (dim + 16) e (sum |q k| + |L| + 1) each, and by 8 e of exp; sums are of chains of at
  most n / 32 + 64 additions, n the queries and heads; what was there before is added once (e).  A
  probability below 2^-126, the smallest normal float, may be 0: the hardware's exponential need not
  give smaller ones.
"""

from __future__ import annotations

import math
import random

import pytest
import torch

import helpers  # noqa: F401
import cuda_rasterizer as cr
from cuda_rasterizer.graphs import CapturedStep
from oracle import paged as op

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TYPES = [torch.float16, torch.bfloat16]


def randn(g, *shape):
    return torch.randn(shape, generator=g, device=g.device)


def offsets_of(lengths, gpu, first=0):
    return (torch.tensor([0] + lengths, device=gpu).cumsum(0) + first).to(torch.int32)


def same(a, b):
    """To the bit, NaN too."""
    bits = {2: torch.int16, 4: torch.int32}[a.element_size()]
    return a.dtype == b.dtype and a.shape == b.shape and torch.equal(a.view(bits), b.view(bits))


class Cache:
    """A pool whose pages are dealt out in no order, with some to spare; k_pages, v_pages and
    weights are NaN and infinities but in the sequences' slots below `lengths`."""

    def __init__(self, gpu, lengths, page, key_heads, dim, dtype, heads_first=False, seed=0, width=0,
                 spare=3, size=1.5):
        g = torch.Generator(device=gpu).manual_seed(31 * sum(lengths) + page + dim + seed)
        need = [-(-n // page) for n in lengths]
        width = max([width, 1] + need)
        pages = sum(need) + spare
        order = torch.randperm(pages, generator=g, device=gpu).to(torch.int32)
        self.tables = torch.full((len(lengths), width), -1, dtype=torch.int32, device=gpu)
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device=gpu)
        self.spare = order[sum(need):]
        shape = (pages, key_heads, page, dim) if heads_first else (pages, page, key_heads, dim)
        k, v = size * randn(g, *shape), randn(g, *shape)
        w = torch.exp(randn(g, *shape[:3]))
        self.k, self.v, self.w = (
            t.transpose(1, 2) if heads_first else t for t in (k.to(dtype), v.to(dtype), w))
        filled = torch.zeros(pages, page, dtype=torch.bool, device=gpu)
        at = 0
        for b, n in enumerate(lengths):
            self.tables[b, :need[b]] = order[at:at + need[b]]
            for i in range(need[b]):
                filled[order[at + i].long(), :n - i * page] = True
            at += need[b]
        self.k[~filled] = math.nan
        self.v[~filled] = math.inf if seed % 2 else math.nan
        self.w[~filled] = math.nan

    def args(self):
        return self.k, self.v, self.tables, self.lengths


def queries(gpu, rows, heads, dim, dtype, seed=0, size=1.5):
    g = torch.Generator(device=gpu).manual_seed(rows + heads + dim + seed)
    return (size * randn(g, rows, heads, dim)).to(dtype)


def within(got, want, tolerance, what=""):
    got = got.double()
    assert got.shape == want.shape
    assert bool(torch.isfinite(got).all()), what
    over = (got - want).abs() - tolerance
    assert not over.numel() or float(over.max()) <= 0.0, (
        what, float((got - want).abs().max()), float(over.max()))


def check_attention(q, c, offsets, causal=True, scale=None):
    """All forms of the call against the oracle; the output and what the slots got."""
    k, v, tables, lengths = c.args()
    before = c.w.clone()
    out, log_sum = cr.paged_attention(q, k, v, tables, lengths, offsets, causal, scale,
                                      weights=c.w, return_log_sum=True)
    after = c.w.clone()
    c.w.copy_(before)
    ref = op.attention(q, k, v, tables, lengths, offsets, causal, scale)
    dim, dtype = q.shape[2], q.dtype
    factor = abs(dim ** -0.5 if scale is None else scale)
    there = ref["weights_terms"] > 0
    norm = k.double().norm(dim=3)[there]
    reach = factor * float(q.double().norm(dim=2).max()) * float(norm.max() if norm.numel() else 0.0)
    largest = float(v.double().abs()[there].max()) if bool(there.any()) else 0.0
    most = max(int(n) for n in lengths) if len(lengths) else 0
    slack = ref["out_slack"]
    tolerance = U[dtype] * slack + 2 * (dim + 16) * E * reach * slack + 1e-30
    if dtype == torch.float16:
        tolerance = tolerance + E * most * largest
    within(out, ref["out"], tolerance, "out")
    empty = torch.isinf(ref["log_sum"])
    assert torch.equal(empty, log_sum == -math.inf)
    size = ref["log_sum"][~empty].abs()
    within(log_sum[~empty], ref["log_sum"][~empty], (dim + 16) * E * (reach + size + 1), "log_sum")
    off = 2 * (dim + 16) * E * (reach + (float(size.max()) if size.numel() else 0.0) + 1) + 8 * E
    off = off + (ref["weights_terms"] / 32 + 64) * E
    want = before.double() + ref["weights"]
    off = off * ref["weights"] + 2 * E * want + 2.0 ** -126 * ref["weights_terms"]
    within(after[there], want[there], off[there], "weights")
    assert same(after[~there], before[~there])
    assert out.is_contiguous() and out.shape == q.shape
    # without what is not asked for, and with it again
    assert torch.equal(cr.paged_attention(q, k, v, tables, lengths, offsets, causal, scale), out)
    again = cr.paged_attention(q, k, v, tables, lengths, offsets, causal, scale, weights=c.w)
    assert torch.equal(again, out) and same(c.w, after)
    c.w.copy_(before)
    return out, after


# --------------------------------------------------------------------- append
def check_append(c, k, v, offsets, with_weights=True):
    w = c.w if with_weights else None
    before = c.w.clone()
    want = op.append(k, v, c.k, c.v, c.tables, c.lengths, offsets, w)
    assert cr.paged_append(k, v, c.k, c.v, c.tables, c.lengths, offsets, w) is None
    assert same(c.k, want[0]) and same(c.v, want[1])
    assert same(c.w, want[2] if with_weights else before)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads_first", [False, True])
@pytest.mark.parametrize("page,key_heads,dim", [(1, 1, 8), (5, 3, 72), (16, 4, 128), (64, 2, 64),
                                                (100, 1, 104)])
def test_append(gpu, page, key_heads, dim, heads_first, dtype):
    lengths, new = [70, 1, 0, 300, 64, 33], [1, 1, 0, 130, 64, 0]
    c = Cache(gpu, lengths, page, key_heads, dim, dtype, heads_first)
    k, v = (queries(gpu, sum(new), key_heads, dim, dtype, s) for s in (1, 2))
    for with_weights in (True, False):
        check_append(c, k, v, offsets_of(new, gpu), with_weights)
    # rows of one product
    qkv = torch.cat((k, k, v), 1)
    check_append(c, -qkv[:, key_heads:2 * key_heads], -qkv[:, 2 * key_heads:], offsets_of(new, gpu))
    check_append(c, qkv[:, key_heads:2 * key_heads], qkv[:, 2 * key_heads:], offsets_of(new, gpu))
    # two bytes off, heads apart, a broadcast head
    odd = torch.empty(k.numel() + 1, dtype=dtype, device=gpu)[1:].view(k.shape).copy_(v)
    apart = k.transpose(0, 1).contiguous().transpose(0, 1)
    check_append(c, odd, apart, offsets_of(new, gpu))
    check_append(c, k[:, :1].expand_as(k), v[:1].expand_as(v), offsets_of(new, gpu))


def test_append_of_what_has_no_place(gpu):
    """More tokens than lengths count, more than the table holds, pages that are not there, rows of
    no sequence, no rows, no sequences."""
    for page in (4, 32):
        c = Cache(gpu, [40, 40, 3, 40, 0], page, 2, 64, torch.float16)
        c.tables[1, 0], c.tables[3, -1] = 1 << 30, c.k.shape[0]
        new = [40, 40, 10, 17, 2]
        c.lengths.copy_(torch.tensor([1000, 40, 3, 40, -7], device=gpu))
        k, v = (queries(gpu, sum(new) + 9, 2, 64, torch.float16, s) for s in (1, 2))
        check_append(c, k, v, offsets_of(new, gpu, 5))
        at = offsets_of(new, gpu)
        at[-1] = 100_000
        check_append(c, k, v, at)
        check_append(c, k, v, at - 3)
        check_append(c, k[:0], v[:0], at * 0)
        none = torch.zeros(0, 7, dtype=torch.int32, device=gpu)
        before = c.k.clone()
        cr.paged_append(k, v, c.k, c.v, none, c.lengths[:0], at[:1])
        assert same(c.k, before)
        cr.paged_append(k, v, c.k, c.v, c.tables[:, :0], c.lengths, at)
        assert same(c.k, before)


def test_append_past_32_bits(gpu):
    """A pool whose elements pass 2^31, and a table of many entries."""
    pool = torch.zeros(70_000, 2, 1, 16_384 + 64, dtype=torch.float16, device=gpu)
    k_pages, v_pages = pool[..., :64], pool[..., 16_384:]
    tables = torch.tensor([[69_999, 3, 65_536]], dtype=torch.int32, device=gpu)
    lengths = torch.tensor([6], dtype=torch.int32, device=gpu)
    k, v = (queries(gpu, 6, 1, 64, torch.float16, s) for s in (1, 2))
    cr.paged_append(k, v, k_pages, v_pages, tables, lengths, offsets_of([6], gpu))
    at = tables[0].long()
    assert same(k_pages[at].reshape(6, 1, 64), k) and same(v_pages[at].reshape(6, 1, 64), v)
    assert int((pool != 0).any(3).sum()) == 6
    q = queries(gpu, 3, 2, 64, torch.float16)
    got = cr.paged_attention(q, k_pages, v_pages, tables, lengths, offsets_of([3], gpu), True)
    near = Cache(gpu, [6], 2, 1, 64, torch.float16)
    cr.paged_append(k, v, *near.args(), offsets_of([6], gpu))
    assert torch.equal(got, cr.paged_attention(q, *near.args(), offsets_of([3], gpu), True))
    new_tables = torch.tensor([[69_998, 4]], dtype=torch.int32, device=gpu)
    weights = torch.zeros(70_000, 2, 1, device=gpu)
    weights[at[0], 1] = 1.0
    lengths, kept = cr.paged_evict(k_pages, v_pages, weights, tables, lengths, new_tables, 3, 2)
    assert lengths.tolist() == [3] and kept.tolist() == [[[1, 4, 5]]]
    assert same(k_pages[new_tables[0].long()].reshape(4, 1, 64)[:3], k[[1, 4, 5]])
    assert same(v_pages[new_tables[0].long()].reshape(4, 1, 64)[:3], v[[1, 4, 5]])


@pytest.mark.parametrize("page", [4, 64])
def test_append_past_the_table(gpu, page):
    """New tokens that the table has no slot for go nowhere, and the earlier ones stay."""
    c = Cache(gpu, [64, 64, 64], page, 2, 64, torch.bfloat16)
    before = [t.clone() for t in (c.k, c.v, c.w)]
    c.lengths.copy_(torch.tensor([70, 64, 1000], device=gpu))
    new = [10, 10, 10]
    k, v = (queries(gpu, 30, 2, 64, torch.bfloat16, s) for s in (1, 2))
    check_append(c, k, v, offsets_of(new, gpu))
    for b, (first, n) in enumerate(((60, 4), (54, 10), (64, 0))):
        slots = torch.arange(64, device=gpu)
        at = c.tables[b, slots // page].long(), slots % page
        for got, was, rows in zip((c.k, c.v, c.w), before, (k, v, torch.zeros(30, 2, device=gpu))):
            assert same(got[at][:first], was[at][:first])
            assert same(got[at][first:], rows[10 * b:10 * b + n])


def test_append_to_more_than_2_30_sequences(gpu):
    """(Of which the last three have a token: 4 GB of offsets, and as much of lengths.)"""
    n = (1 << 30) + 100
    offsets = torch.zeros(n + 1, dtype=torch.int32, device=gpu)
    offsets[-3:] = torch.tensor([1, 2, 3], device=gpu)
    lengths = torch.zeros(n, dtype=torch.int32, device=gpu)
    lengths[-3:] = torch.tensor([5, 1, 3], device=gpu)
    tables = torch.zeros(1, 1, dtype=torch.int32, device=gpu).expand(n, 1)
    pool = [torch.zeros(1, 8, 2, 16, dtype=torch.float16, device=gpu) for _ in range(2)]
    k, v = (queries(gpu, 3, 2, 16, torch.float16, s) for s in (1, 2))
    cr.paged_append(k, v, *pool, tables, lengths, offsets)
    for got, new in zip(pool, (k, v)):
        want = torch.zeros_like(got)
        want[0, [4, 0, 2]] = new
        assert same(got, want)


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("page", [1, 7, 16, 48, 64, 128, 200])
@pytest.mark.parametrize("lengths,new", [([1], [1]), ([300, 1, 77], [1, 1, 1]), ([64], [64]),
                                         ([200, 0, 129, 33], [5, 0, 129, 7]), ([65, 500], [200, 3]),
                                         ([700, 5, 128], [300, 5, 0])])
def test_attention_of_lengths(gpu, lengths, new, page, causal, dtype):
    c = Cache(gpu, lengths, page, 2, 64, dtype, seed=page)
    check_attention(queries(gpu, sum(new), 4, 64, dtype), c, offsets_of(new, gpu), causal)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [8, 16, 24, 40, 64, 72, 96, 104, 128])
def test_attention_dimensions(gpu, dim, dtype):
    for page in (24, 64):
        for new in ([90, 37], [1, 1]):
            c = Cache(gpu, [130, 37], page, 1, dim, dtype, heads_first=dim % 16 == 0)
            check_attention(queries(gpu, sum(new), 2, dim, dtype), c, offsets_of(new, gpu))


@pytest.mark.parametrize("heads,key_heads", [(1, 1), (3, 3), (3, 1), (8, 1), (10, 2), (40, 1)])
def test_attention_grouped_heads(gpu, heads, key_heads):
    for page in (10, 128):
        c = Cache(gpu, [90, 260, 1], page, key_heads, 32, torch.bfloat16)
        for new in ([50, 40, 1], [1, 1, 1], [0, 3, 0]):
            check_attention(queries(gpu, sum(new), heads, 32, torch.bfloat16), c, offsets_of(new, gpu))


@pytest.mark.parametrize("page", [3, 40, 64, 256])
@pytest.mark.parametrize("new", [1, 2, 300])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_over_long_caches(gpu, dim, new, page):
    for dtype in TYPES:
        c = Cache(gpu, [5000, 64, 1, 20_001, 0, 9000], page, 2, dim, dtype, heads_first=dim == 64)
        check_attention(queries(gpu, 6 * new, 8, dim, dtype), c, offsets_of([new] * 6, gpu))


@pytest.mark.parametrize("page", [1, 16, 24, 64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_without_some_pages(gpu, causal, page):
    """Pages that are not there: at the start, at the end, most, all; a table with too few."""
    for dtype in TYPES:
        for new in ([1] * 6, [40, 3, 200, 17, 1, 2]):
            lengths = [400, 130, 300, 129, 300, 900]
            c = Cache(gpu, lengths, page, 2, 64, dtype)
            g = torch.Generator(device=gpu).manual_seed(page)
            c.tables[0, 0] = -1
            c.tables[1, -(-130 // page) - 1] = c.k.shape[0]
            hide = torch.rand(c.tables.shape[1], generator=g, device=gpu) < 0.7
            c.tables[2, hide] = torch.iinfo(torch.int32).min
            c.tables[3] = torch.iinfo(torch.int32).max
            c.lengths[4] = 1 << 30
            c.lengths[5] = -1
            # (past the table's end that is filled)
            c.tables[4, 300 // page:] = -1
            check_attention(queries(gpu, sum(new), 4, 64, dtype), c, offsets_of(new, gpu), causal)


@pytest.mark.parametrize("page", [24, 64])
def test_attention_over_wide_tables(gpu, page):
    """Tables far wider than what is filled: few rows whose scores would take too much room."""
    for dtype, dim in zip(TYPES, (64, 128)):
        for new in ([1] * 4, [3, 0, 1, 2]):
            c = Cache(gpu, [700, 64, 0, 129], page, 2, dim, dtype, width=(1 << 22) // page)
            q = queries(gpu, sum(new), 8, dim, dtype)
            check_attention(q, c, offsets_of(new, gpu))
            check_attention(q, c, offsets_of(new, gpu), causal=False, scale=-0.2)


def test_attention_of_rows_of_no_sequence(gpu):
    c = Cache(gpu, [60, 70], 16, 2, 64, torch.float16)
    q = queries(gpu, 150, 4, 64, torch.float16)
    out, _ = check_attention(q, c, offsets_of([60, 70], gpu, 10), causal=True)
    assert bool((out[:10] == 0).all()) and bool((out[140:] == 0).all())
    k, v, tables, lengths = c.args()
    none = cr.paged_attention(q, k, v, tables[:0], lengths[:0], offsets_of([], gpu), weights=c.w)
    assert bool((none == 0).all())
    none = cr.paged_attention(q, k, v, tables[:, :0], lengths, offsets_of([60, 70], gpu), weights=c.w)
    assert bool((none == 0).all())
    none = cr.paged_attention(q, k[:0], v[:0], tables, lengths, offsets_of([60, 70], gpu),
                              weights=c.w[:0])
    assert bool((none == 0).all())
    assert cr.paged_attention(q[:0], k, v, tables, lengths, offsets_of([0, 0], gpu)).shape == (0, 4, 64)
    good = cr.paged_attention(q[:130], k, v, tables, lengths, offsets_of([60, 70], gpu), True)
    at = torch.tensor([-5, 60, 1_000_000], dtype=torch.int32, device=gpu)
    assert torch.equal(cr.paged_attention(q[:130], k, v, tables, lengths, at, True), good)


@pytest.mark.parametrize("page", [24, 64])
@pytest.mark.parametrize("dtype", TYPES)
def test_attention_of_large_scores_and_scales(gpu, dtype, page):
    for new in ([1], [150]):
        c = Cache(gpu, [200], page, 1, 64, dtype, size=6.0)
        q = queries(gpu, new[0], 2, 64, dtype, size=6.0)
        at = offsets_of(new, gpu)
        for scale in (1.0, -0.5, 0.0):
            check_attention(q, c, at, scale=scale)


def test_attention_equals_packed(gpu):
    """The pages one after another are packed rows: the same kernels' sums, to the bit."""
    for dtype in TYPES:
        for lengths, new in (([640, 200], [130, 200]), ([3000, 64], [1, 1])):
            c = Cache(gpu, lengths, 64, 2, 128, dtype)
            q = queries(gpu, sum(new), 8, 128, dtype)
            at = offsets_of(new, gpu)
            packed = [torch.cat([t[c.tables[b, :-(-n // 64)].long()].flatten(0, 1)[:n]
                                 for b, n in enumerate(lengths)]) for t in (c.k, c.v)]
            want = cr.packed_attention(q, *packed, at, offsets_of(lengths, gpu), causal=True)
            got = cr.paged_attention(q, *c.args(), at, causal=True)
            assert float((got.double() - want.double()).norm()) <= 2 * U[dtype] * float(want.double().norm())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths,new,bits", [([640, 200], [130, 200], True), ([3000, 64], [1, 1], True),
                                              ([9000, 500, 64], [1, 1, 1], True),
                                              ([9000, 500], [300, 20], False)])
def test_attention_equals_packed_element_by_element(gpu, lengths, new, bits, dtype):
    """Pages one after another are packed rows.  Where both calls split the keys alike, which for few rows
    and for tiles of rows over less than 2048 slots they do, the same to the bit; else each is within
    check_attention's bound of the definition, and so within twice that of the other."""
    c = Cache(gpu, lengths, 64, 2, 128, dtype)
    q = queries(gpu, sum(new), 8, 128, dtype)
    at = offsets_of(new, gpu)
    packed = [torch.cat([t[c.tables[b, :-(-n // 64)].long()].flatten(0, 1)[:n]
                         for b, n in enumerate(lengths)]) for t in (c.k, c.v)]
    want = cr.packed_attention(q, *packed, at, offsets_of(lengths, gpu), causal=True)
    got = cr.paged_attention(q, *c.args(), at, causal=True)
    if bits:
        assert same(got, want)
        return
    slack = op.attention(q, *c.args(), at, True)["out_slack"]
    reach = 128 ** -0.5 * float(q.double().norm(dim=2).max()) * float(packed[0].double().norm(dim=2).max())
    bound = U[dtype] * slack + 2 * (128 + 16) * E * reach * slack + 1e-30
    if dtype == torch.float16:
        bound = bound + E * max(lengths) * float(packed[1].double().abs().max())
    within(got, want.double(), 2 * bound, "out")


def test_attention_of_what_is_not_finite(gpu):
    """A NaN in a query makes its output and the weights that it gives NaN, and no other's; an
    infinity in a value that a query sees comes out in its column; values that it does not see
    change nothing."""
    for dtype in TYPES:
        for page in (24, 64):
            for lengths, new in (([300], [300]), ([3000], [40]), ([700], [1])):
                c = Cache(gpu, lengths, page, 2, 64, dtype, size=0.3)
                q = queries(gpu, new[0], 4, 64, dtype, size=0.3)
                at = offsets_of(new, gpu)
                clean, _ = check_attention(q, c, at)
                row = new[0] // 2
                bad = q.clone()
                bad[row, 1, 3] = math.nan
                w = torch.zeros_like(c.w)
                got = cr.paged_attention(bad, *c.args(), at, True, weights=w)
                assert bool(torch.isnan(got[row, 1]).all())
                others = torch.ones(q.shape[:2], dtype=torch.bool, device=gpu)
                others[row, 1] = False
                assert torch.equal(got[others], clean[others])
                seen = lengths[0] - new[0] + row
                slots = torch.arange(lengths[0], device=gpu)
                lines = w[c.tables[0, slots // page].long(), slots % page]
                assert torch.equal(torch.isnan(lines[:, 0]), slots <= seen)
                assert bool(torch.isfinite(lines[:, 1]).all())
                slot = lengths[0] - max(1, new[0] // 4)
                there = c.tables[0, slot // page].long(), slot % page
                was = c.v[there].clone()
                c.v[there][0, 5], c.v[there][1, 7] = math.inf, math.nan
                got = cr.paged_attention(q, *c.args(), at, True)
                first = slot - (lengths[0] - new[0])  # the first query that sees it
                assert bool((got[max(first, 0):, :2, 5] == math.inf).all())
                assert bool(torch.isnan(got[max(first, 0):, 2:, 7]).all())
                mask = torch.isfinite(got)
                assert torch.equal(got[mask], clean[mask])
                assert int((~mask).sum()) == 4 * (new[0] - max(first, 0))
                c.v[there] = was


@pytest.mark.parametrize("page", [24, 64])
def test_attention_of_skewed_chunks(gpu, page):
    """One long chunk among single tokens, and one long cache among short ones."""
    for dtype in TYPES:
        for lengths, new in (([2000] + [30] * 40, [300] + [1] * 40), ([20, 9000, 1] + [5] * 70, [1] * 73),
                             ([6000, 300, 2500], [130, 1, 0])):
            c = Cache(gpu, lengths, page, 2, 64, dtype)
            check_attention(queries(gpu, sum(new), 4, 64, dtype), c, offsets_of(new, gpu))


@pytest.mark.parametrize("page", [24, 64])
@pytest.mark.parametrize("sequences", [63, 64, 65, 125, 126, 127, 128, 129, 300])
def test_attention_of_many_sequences(gpu, sequences, page):
    """Single tokens, and chunks: as many sequences as lanes hold, one more, and looks through many of them."""
    rng = random.Random(sequences + page)
    for dtype in TYPES:
        lengths = [rng.choice([0, 1, 30, 64, 100, 300]) for _ in range(sequences)]
        lengths[rng.randrange(sequences)] = 3000
        for most in (1, 3, 40):
            new = [rng.choice([0, min(n, most), most]) for n in lengths]
            c = Cache(gpu, lengths, page, 2, 64, dtype, seed=most)
            check_attention(queries(gpu, sum(new), 4, 64, dtype), c, offsets_of(new, gpu))


@pytest.mark.parametrize("page", [24, 64])
def test_attention_of_many_sequences_over_wide_tables(gpu, page):
    """Few rows whose scores are not kept, of more sequences than a look through them takes."""
    lengths, rng = [20, 300, 0, 64, 129] * 30, random.Random(page)
    new = [rng.choice([0, 1, 1]) for _ in lengths]
    c = Cache(gpu, lengths, page, 2, 64, torch.float16, width=(1 << 18) // page)
    check_attention(queries(gpu, sum(new), 8, 64, torch.float16), c, offsets_of(new, gpu))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page", [24, 64])
@pytest.mark.parametrize("new,width", [([1] * 6, 0), ([2] * 6, 0), ([1] * 6, (1 << 25) // 24), ([60] * 6, 0),
                                       ([70, 1, 0, 200, 5, 90], 0)])
def test_weights_of_shared_pages(gpu, new, width, page, dtype):
    """A page of several sequences, or twice in a table, gets what each of its places adds.  The bound is
    check_attention's, and a rounding (e of the sum) for each place that adds."""
    lengths = [400, 300, 130, 500, 64, 200]
    c = Cache(gpu, lengths, page, 2, 64, dtype, width=width)
    pages = 128 // page
    c.tables[1:, :pages] = c.tables[0, :pages]  # the first slots are all sequences'
    c.tables[3, pages + 1:300 // page] = c.tables[3, pages]  # and one page is all over a table
    q = queries(gpu, sum(new), 4, 64, dtype)
    k, v, tables, lengths = c.args()
    at = offsets_of(new, gpu)
    for causal in (True, False):
        ref = op.attention(q, k, v, tables, lengths, at, causal)
        there = ref["weights_terms"] > 0
        reach = 64 ** -0.5 * float(q.double().norm(dim=2).max()) * float(k.double().norm(dim=3)[there].max())
        size = ref["log_sum"][~torch.isinf(ref["log_sum"])].abs()
        off = 2 * (64 + 16) * E * (reach + float(size.max()) + 1) + 8 * E
        off = off + (ref["weights_terms"] / 32 + 64) * E
        places = 6 + 300 // page
        for _ in range(3):
            w = c.w.clone()
            cr.paged_attention(q, k, v, tables, lengths, at, causal, weights=w)
            want = c.w.double() + ref["weights"]
            bound = off * ref["weights"] + (1 + places) * E * want + 2.0 ** -126 * ref["weights_terms"]
            within(w[there], want[there], bound[there], "weights")
            assert same(w[~there], c.w[~there])


@pytest.mark.parametrize("page", [24, 64])
@pytest.mark.parametrize("key_heads", [4, 5, 6, 8, 12])
def test_weights_of_many_key_heads(gpu, key_heads, page):
    """Few rows, fewer than the key heads or more: heads one by one, in pairs, in fours."""
    lengths = [300, 0, 1, 65, 5000, 64, 129]
    for dtype in TYPES:
        for group, new in ((1, [1] * 7), (2, [1, 0, 1, 1, 2, 1, 0]), (3, [2] * 7), (8, [1] * 7),
                           (1, [40, 0, 1, 1, 1, 1, 1])):
            c = Cache(gpu, lengths, page, key_heads, 32, dtype, heads_first=group == 2)
            check_attention(queries(gpu, sum(new), key_heads * group, 32, dtype), c, offsets_of(new, gpu))


@pytest.mark.parametrize("page", [24, 64])
def test_weights_below_the_smallest_normal_float(gpu, page):
    """They stay as they are where nothing is added, as every other weight."""
    for new in (1, 200):
        c = Cache(gpu, [300], page, 1, 64, torch.float16)
        slots = torch.arange(300, device=gpu)
        at = c.tables[0, slots // page].long(), slots % page
        c.k[at] = 0.0
        seen = at[0][7], at[1][7]
        c.k[seen] = 16.0  # its score is 2048, the others' 0: their probabilities are 0 in float
        q = torch.full((new, 1, 64), 16.0, dtype=torch.float16, device=gpu)
        for small in (1e-40, 2.0 ** -149, -3e-39):
            c.w[at] = small
            want = c.w.clone()
            cr.paged_attention(q, *c.args(), offsets_of([new], gpu), weights=c.w)
            # a probability of 1 from a score and a log-sum of 2048 each, as check_attention's bound has it
            assert abs(float(c.w[seen]) - new) <= 2 * (64 + 16) * E * (2048 + 2048 + 1) * new
            c.w[seen] = want[seen]
            assert same(c.w, want)


@pytest.mark.parametrize("page", [24, 64])
@pytest.mark.parametrize("lengths,new", [([300], [300]), ([5000], [1]), ([3000], [100])])
def test_attention_of_keys_that_all_score_minus_infinity(gpu, lengths, new, page):
    """Seen, they give NaN and no weight; on pages that are not there, zeros."""
    for dtype in TYPES:
        c = Cache(gpu, lengths, page, 1, 64, dtype)
        slots = torch.arange(lengths[0], device=gpu)
        at = c.tables[0, slots // page].long(), slots % page
        c.k[at], c.v[at], c.w[at] = -math.inf, 1.0, 0.5
        q, offsets = torch.ones(new[0], 2, 64, dtype=dtype, device=gpu), offsets_of(new, gpu)
        out = cr.paged_attention(q, *c.args(), offsets, weights=c.w)
        assert bool(torch.isnan(out).all()) and bool((c.w[at] == 0.5).all())
        c.tables.fill_(-1)
        out = cr.paged_attention(q, *c.args(), offsets, weights=c.w)
        assert bool((out == 0).all()) and bool((c.w[at] == 0.5).all())


# ------------------------------------------------------------------- eviction
def check_evict(c, new_tables, keep, recent=0):
    want = op.evict(c.k, c.v, c.w, c.tables, c.lengths, new_tables, keep, recent)
    lengths, kept = cr.paged_evict(c.k, c.v, c.w, c.tables, c.lengths, new_tables, keep, recent)
    assert same(lengths.cpu(), want[0]), (lengths, want[0])
    assert same(kept.cpu(), want[1])
    for got, ref in zip((c.k, c.v, c.w), want[2:]):
        assert same(got, ref)
    return lengths, kept


@pytest.mark.parametrize("heads_first", [False, True])
@pytest.mark.parametrize("page", [1, 7, 16, 64])
@pytest.mark.parametrize("keep,recent", [(1, 0), (1, 1), (10, 3), (33, 33), (64, 0), (100, 20),
                                         (250, 100), (500, 7)])
def test_evict(gpu, keep, recent, page, heads_first):
    for dtype, dim in zip(TYPES, (64, 72)):
        lengths = [300, 1, 0, 64, 129, 33, 100, 101]
        fresh = -(-keep // page)
        c = Cache(gpu, lengths, page, 3, dim, dtype, heads_first, spare=fresh * len(lengths) + 2)
        check_evict(c, c.spare[:fresh * len(lengths)].view(len(lengths), fresh), keep, recent)


@pytest.mark.parametrize("kind", ["all alike", "few values", "zeros", "negative", "not finite", "near"])
def test_evict_of_equal_and_odd_weights(gpu, kind):
    """Ties go to the lower slot; both zeros are one; NaN is above infinity."""
    lengths = [2000, 700, 65]
    for keep, recent in ((64, 0), (300, 50), (1500, 1)):
        fresh = -(-keep // 16)
        c = Cache(gpu, lengths, 16, 2, 8, torch.float16, spare=3 * fresh, seed=keep)
        g = torch.Generator(device=gpu).manual_seed(keep)
        w = randn(g, *c.w.shape)
        if kind == "all alike":
            w.fill_(0.25)
        elif kind == "few values":
            w = torch.floor(w * 2) / 2
        elif kind == "zeros":
            w = torch.where(w > 0.5, w, torch.where(w > -0.5, 0.0, -0.0))
        elif kind == "negative":
            w = -w.abs() * 1e-40
        elif kind == "not finite":
            w = torch.where(w > 1, math.nan, torch.where(w > 0.5, math.inf, torch.where(w < -1, -math.inf, w)))
            w = torch.where(w < -0.5, -torch.tensor(math.nan, device=gpu), w)
        else:  # differences in the last bits only
            w = (1.0 + torch.round(w * 3).clamp(-6, 6) * 2.0 ** -23)
        c.w.copy_(w)
        check_evict(c, c.spare.view(3, fresh), keep, recent)


def test_evict_without_some_pages(gpu):
    """Old pages and new ones that are not there."""
    for page in (8, 64):
        keep = 100
        fresh = -(-keep // page) + 1
        c = Cache(gpu, [300, 300, 90, 300], page, 2, 64, torch.bfloat16, spare=4 * fresh)
        c.tables[0, 1], c.tables[1, :] = -1, 1 << 29
        c.tables[3, (300 - 1) // page] = c.k.shape[0]  # the most recent
        c.lengths[2] = 1 << 30
        c.tables[2, 90 // page:] = -1
        new_tables = c.spare.view(4, fresh).clone()
        new_tables[0, 0], new_tables[3, 1] = -1, 1 << 30
        check_evict(c, new_tables, keep, 30)


@pytest.mark.parametrize("length,keep", [(20_000, 9000), (32_768, 20_000), (32_769, 100), (70_000, 30_000),
                                         (140_001, 3), (40_000, 39_999)])
@pytest.mark.parametrize("page", [24, 64])
def test_evict_of_long_sequences(gpu, length, keep, page):
    fresh = -(-keep // page)
    c = Cache(gpu, [length, 500], page, 2, 8, torch.float16, spare=2 * fresh)
    check_evict(c, c.spare.view(2, fresh), keep, min(keep, 1000))
    c.w.copy_(torch.floor(c.w))  # most alike
    check_evict(c, c.spare.view(2, fresh), keep, 0)


def test_evict_of_many_sequences(gpu):
    g = torch.Generator().manual_seed(5)
    lengths = torch.randint(0, 90, (700,), generator=g).tolist()
    c = Cache(gpu, lengths, 16, 2, 16, torch.float16, spare=700 * 2)
    check_evict(c, c.spare.view(700, 2), 32, 8)


@pytest.mark.parametrize("sequences", [65_535, 65_536, 66_001, 140_000])
def test_evict_of_more_sequences_than_a_grid_has_rows(gpu, sequences):
    """Three slots on a page of four, down to two: slots and weights follow from the sequence's number."""
    b = torch.arange(sequences, device=gpu)
    slots = torch.arange(4, device=gpu)
    k = torch.zeros(2 * sequences, 4, 1, 8, dtype=torch.float16, device=gpu)
    k[:sequences] = ((b[:, None] * 4 + slots) % 2039)[..., None, None].to(torch.float16)
    v = -k
    w = torch.zeros(2 * sequences, 4, 1, device=gpu)
    w[:sequences, :, 0] = ((b[:, None] * 7 + slots * 5) % 11).float()
    tables, new_tables = b[:, None].to(torch.int32), (b[:, None] + sequences).to(torch.int32)
    filled = b % 4  # none to three
    order = torch.where(slots < filled[:, None], w[:sequences, :, 0], -1.0)
    order = torch.sort(order, dim=1, descending=True, stable=True)[1][:, :2].sort(1)[0]
    there = slots[:2] < filled.clamp(max=2)[:, None]
    # (of fewer slots than two, the first)
    order = torch.where(filled[:, None] < 2, slots[:2], order)
    want = [t.clone() for t in (k, v, w)]
    for t in want:
        moved = t[b[:, None], order]
        t[sequences:, :2] = torch.where(there.view(there.shape + (1,) * (t.dim() - 2)), moved, t[sequences:, :2])
    lengths, kept = cr.paged_evict(k, v, w, tables, filled.to(torch.int32), new_tables, 2)
    assert torch.equal(lengths.long(), filled.clamp(max=2))
    assert torch.equal(kept[:, 0].long(), torch.where(there, order, -1))
    assert all(same(a, x) for a, x in zip((k, v, w), want))


# ---------------------------------------------------------------------- drawn
@pytest.mark.parametrize("seed", range(48))
def test_drawn_caches(gpu, seed):
    """All three operators at sizes, layouts and masks that are drawn together."""
    rng = random.Random(seed)

    def log(low, high):
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    dtype, dim = TYPES[seed % 2], rng.choice([8, 24, 32, 64, 72, 96, 104, 128])
    key_heads, group = rng.choice([1, 2, 3, 5]), rng.choice([1, 2, 3, 8, 17])
    page = rng.choice([1, 2, 5, 13, 16, 24, 32, 63, 64, 65, 128, 192, 300])
    sequences = rng.choice([1, 2, 3, 5, 20, 70])
    longest, most = log(2, max(3, 4000 // sequences)), rng.choice([1, 1, 2, 8, 60, 300])
    lengths = [rng.choice([0, log(1, longest), longest]) for _ in range(sequences)]
    new = [rng.choice([0, min(n, most), rng.randint(0, most)]) for n in lengths]
    keep = log(1, longest)
    fresh = -(-keep // page)
    c = Cache(gpu, lengths, page, key_heads, dim, dtype, rng.random() < 0.5, seed, rng.choice([0, 50]),
              fresh * sequences + 1)
    if rng.random() < 0.4:
        g = torch.Generator(device=gpu).manual_seed(seed)
        hide = torch.rand(c.tables.shape, generator=g, device=gpu) < rng.choice([0.05, 0.5, 0.95])
        c.tables[hide] = rng.choice([-1, c.k.shape[0], 2 ** 31 - 1, -2 ** 31])
    at = offsets_of(new, gpu)
    k, v = (queries(gpu, sum(new), key_heads, dim, dtype, s + seed) for s in (1, 2))
    check_append(c, k, v, at)
    if sum(new):
        check_attention(queries(gpu, sum(new), key_heads * group, dim, dtype, seed), c, at,
                        rng.random() < 0.7, rng.choice([None, None, 1.0, -0.3, 0.0]))
    if rng.random() < 0.3:
        c.w.copy_(torch.floor(c.w * rng.choice([0.1, 1, 3])))
    check_evict(c, c.spare[:fresh * sequences].view(sequences, fresh), keep, rng.randint(0, keep))


# ------------------------------------------------------------------- together
def stream(cache, new_tables, steps, gpu, keep, run=None):
    """Views appended and attended to, then an eviction, and a view more: outputs."""
    out = []
    for q, k, v, offsets, lengths in steps:
        cache.lengths.copy_(lengths)
        cr.paged_append(k, v, *cache.args(), offsets, weights=cache.w)
        out.append(cr.paged_attention(q, *cache.args(), offsets, causal=True, weights=cache.w))
    lengths, kept = cr.paged_evict(cache.k, cache.v, cache.w, cache.tables, cache.lengths, new_tables,
                                   keep, 12)
    q, k, v, offsets, _ = steps[-1]
    lengths = lengths + offsets.diff().to(torch.int32)
    cr.paged_append(k, v, cache.k, cache.v, new_tables, lengths, offsets, weights=cache.w)
    out.append(cr.paged_attention(q, cache.k, cache.v, new_tables, lengths, offsets, causal=True,
                                  weights=cache.w))
    return (*out, kept, lengths)


def stream_inputs(gpu, seed=0, page=16):
    dtype, counts = torch.bfloat16, [[12, 30, 0], [12, 1, 25], [12, 12, 12]]
    total = [sum(x) for x in zip(*counts)]
    cache = Cache(gpu, total, page, 2, 64, dtype, spare=3 * (-(-60 // page)), seed=seed)
    steps, lengths = [], torch.zeros(3, dtype=torch.int32, device=gpu)
    for i, new in enumerate(counts):
        lengths = lengths + torch.tensor(new, dtype=torch.int32, device=gpu)
        steps.append((queries(gpu, sum(new), 4, 64, dtype, 3 * i + seed),
                      *(queries(gpu, sum(new), 2, 64, dtype, 3 * i + s + seed) for s in (1, 2)),
                      offsets_of(new, gpu), lengths))
    return cache, cache.spare.view(3, -1), steps


@pytest.mark.parametrize("page", [16, 64])
def test_a_stream_of_views(gpu, page):
    """Append, attend with weights, evict, append, attend: each step against the oracle on what
    the step before left."""
    c, new_tables, steps = stream_inputs(gpu, page=page)
    for q, k, v, offsets, lengths in steps:
        c.lengths.copy_(lengths)
        check_append(c, k, v, offsets)
        out, after = check_attention(q, c, offsets)
        c.w.copy_(after)
    lengths, _ = check_evict(c, new_tables, 36, 12)
    q, k, v, offsets, _ = steps[-1]
    c.tables, c.lengths = new_tables, lengths + offsets.diff().to(torch.int32)
    check_append(c, k, v, offsets)
    check_attention(q, c, offsets)


def test_views_over_pages_equal_all_at_once(gpu):
    """What each view's tokens give over the pages is what packed_attention gives for all tokens
    together, causal."""
    dtype, counts = torch.float16, [40, 1, 70, 12]
    total = sum(counts)
    q, k, v = (queries(gpu, total, h, 64, dtype, s) for h, s in ((4, 0), (2, 1), (2, 2)))
    want = cr.packed_attention(q, k, v, offsets_of([total], gpu), causal=True)
    for page in (24, 64):
        c = Cache(gpu, [total], page, 2, 64, dtype)
        at = 0
        for n in counts:
            c.lengths.fill_(at + n)
            rows = slice(at, at + n)
            cr.paged_append(k[rows], v[rows], *c.args(), offsets_of([n], gpu))
            got = cr.paged_attention(q[rows], *c.args(), offsets_of([n], gpu), causal=True)
            far = (got.double() - want[rows].double()).norm() / want[rows].double().norm()
            assert float(far) <= 4 * U[dtype]
            at += n


def test_on_another_stream_and_in_a_graph(gpu):
    """On a side stream, and captured: each replay with other inputs, lengths and tables against
    the eager calls, with eager work between the replays."""
    want, caches = [], [stream_inputs(gpu) for _ in range(3)]
    want = stream(*caches[0], gpu, 36)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = stream(*caches[1], gpu, 36)
    torch.cuda.current_stream().wait_stream(side)
    assert all(same(a, b) for a, b in zip(want, other))
    eager, _, eager_steps = caches[0]
    held, held_tables, held_steps = caches[2]
    captured = CapturedStep(lambda: stream(held, held_tables, held_steps, gpu, 36))
    for seed in range(3):
        fresh, new_tables, steps = stream_inputs(gpu, seed=2 * seed + 1)
        for t in ("k", "v", "w", "tables"):
            getattr(held, t).copy_(getattr(fresh, t))
        held_tables.copy_(new_tables)
        for mine, theirs in zip(held_steps, steps):
            for a, b in zip(mine, theirs):
                a.copy_(b)
        captured.replay()
        now = stream(fresh, new_tables, steps, gpu, 36)
        torch.cuda.synchronize()
        assert all(same(a, b) for a, b in zip(now, captured.output))
        for t in ("k", "v", "w"):
            assert same(getattr(held, t), getattr(fresh, t))


def test_two_captured_calls_at_once(gpu):
    """Two captured steps that need workspaces, replayed in turn and on two streams at once, with eager
    calls between."""
    held = []
    for lengths, new, seed in (([9000, 300], [40, 40], 2), ([5000, 7000, 12], [1, 1, 1], 4)):
        c = Cache(gpu, lengths, 64, 2, 128, torch.bfloat16, seed=seed)
        q = queries(gpu, sum(new), 8, 128, torch.bfloat16, seed)
        w = torch.zeros_like(c.w)

        def step(c=c, q=q, w=w, at=offsets_of(new, gpu)):
            w.zero_()
            return cr.paged_attention(q, *c.args(), at, True, weights=w, return_log_sum=True)

        want = [t.clone() for t in step()] + [w.clone()]
        held.append((CapturedStep(step), step, w, want))
    streams = [torch.cuda.Stream() for _ in held]
    for at_once in (False, True, False, True):
        for (captured, _, w, _), one in zip(held, streams):
            for t in (*captured.output, w):
                t.fill_(math.nan)
        torch.cuda.synchronize()
        for (captured, _, _, _), one in zip(held, streams):
            with torch.cuda.stream(one):
                captured.replay()
            if not at_once:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        for captured, step, w, want in held:
            assert all(same(a, b) for a, b in zip((*captured.output, w), want))
            assert all(same(a, b) for a, b in zip(step(), want))
        torch.cuda.synchronize()


def test_two_streams_at_once(gpu):
    """Two calls of the same operators at once, each with its own workspace."""
    a, b = ([Cache(gpu, [9000, 300], 64, 2, 128, torch.bfloat16, seed=s), s] for s in (2, 4))
    want = []
    for c, s in (a, b):
        q = queries(gpu, 80, 8, 128, torch.bfloat16, s)
        want.append(cr.paged_attention(q, *c.args(), offsets_of([40, 40], gpu), True, weights=c.w))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        got = []
        for (c, s), one in zip((a, b), streams):
            q = queries(gpu, 80, 8, 128, torch.bfloat16, s)
            at = offsets_of([40, 40], gpu)
            torch.cuda.synchronize()
            with torch.cuda.stream(one):
                got.append(cr.paged_attention(q, *c.args(), at, True, weights=c.w))
        torch.cuda.synchronize()
        assert all(same(x, y) for x, y in zip(got, want))


def test_weights_on_two_streams_at_once(gpu):
    """Two calls at once, with and without kept scores: outputs and weights as those of the calls alone."""
    for new, heads in (([40, 40], 8), ([1, 1], 8), ([1, 1], 2)):
        held = []
        for s in (2, 4):
            c = Cache(gpu, [9000, 300], 64, 2, 128, torch.bfloat16, seed=s)
            q, at = queries(gpu, sum(new), heads, 128, torch.bfloat16, s), offsets_of(new, gpu)
            w = c.w.clone()
            out = cr.paged_attention(q, *c.args(), at, True, weights=w)
            held.append((c, q, at, out, w))
        streams = [torch.cuda.Stream() for _ in held]
        for _ in range(4):
            weights = [c.w.clone() for c, *_ in held]
            torch.cuda.synchronize()
            got = []
            for (c, q, at, _, _), w, one in zip(held, weights, streams):
                with torch.cuda.stream(one):
                    got.append(cr.paged_attention(q, *c.args(), at, True, weights=w))
            torch.cuda.synchronize()
            for (_, _, _, out, w), mine, now in zip(held, weights, got):
                assert same(now, out) and same(mine, w)


# --------------------------------------------------------------------- layouts
@pytest.mark.parametrize("layout", ["keys and values in turn", "a layer of several", "some of the heads",
                                    "every other page", "weights in another order"])
@pytest.mark.parametrize("page", [16, 64])
def test_pools_in_larger_ones(gpu, layout, page):
    """Pools, tables, lengths and offsets that are parts of other tensors, which stay as they are."""
    dtype, heads, dim, lengths, new = torch.float16, 2, 64, [200, 33, 70], [30, 1, 0]
    c = Cache(gpu, lengths, page, heads, dim, dtype, spare=3 * (-(-50 // page)))
    pages = c.k.shape[0]
    whole = {"keys and values in turn": (pages, 2, page, heads, dim),
             "a layer of several": (pages, 5, page, heads, dim),
             "some of the heads": (pages, page, heads + 3, dim),
             "every other page": (2 * pages, page, heads, dim + 8),
             "weights in another order": (pages, page, heads, dim)}[layout]
    pools = [torch.full(whole, math.nan, dtype=dtype, device=gpu) for _ in range(2)]
    if layout == "keys and values in turn":
        pools[1] = pools[0]
        k, v = pools[0][:, 0], pools[0][:, 1]
    else:
        k, v = {"a layer of several": lambda t: t[:, 3], "some of the heads": lambda t: t[:, :, 1:1 + heads],
                "every other page": lambda t: t[::2, ..., :dim],
                "weights in another order": lambda t: t}[layout](pools[0]), None
        v = pools[1].as_strided(k.shape, k.stride(), k.storage_offset())
    k.copy_(c.k), v.copy_(c.v)
    outside = [t.clone() for t in pools]
    w = c.w.clone()
    if layout == "weights in another order":
        w = torch.empty(heads, pages, page, device=gpu).permute(1, 2, 0).copy_(c.w)
    wide = torch.full((3, c.tables.shape[1] + 5), 1 << 20, dtype=torch.int32, device=gpu)
    tables = wide[:, 2:2 + c.tables.shape[1]].copy_(c.tables)
    spread = torch.stack((c.lengths, c.lengths + 7), 1)[:, 0]
    offsets = torch.stack((offsets_of(new, gpu),) * 3, 1)[:, 1]
    fresh = torch.full((3, -(-50 // page) + 1), -1, dtype=torch.int32, device=gpu)
    new_tables = fresh[:, :-1].copy_(c.spare.view(3, -1))
    q, nk, nv = (queries(gpu, sum(new), h, dim, dtype, h) for h in (4, heads, heads))

    def run(k, v, w, tables, lengths, offsets, new_tables):
        cr.paged_append(nk, nv, k, v, tables, lengths, offsets, w)
        out = cr.paged_attention(q, k, v, tables, lengths, offsets, True, weights=w)
        return (out, *cr.paged_evict(k, v, w, tables, lengths, new_tables, 50, 20))

    want = run(c.k, c.v, c.w, c.tables, c.lengths, offsets.contiguous(), new_tables.contiguous())
    got = run(k, v, w, tables, spread, offsets, new_tables)
    assert all(same(a, b) for a, b in zip(got, want))
    assert same(k.contiguous(), c.k) and same(v.contiguous(), c.v) and same(w.contiguous(), c.w)
    k.zero_(), v.zero_()
    for t, before in zip(pools, outside):  # what is not the pool's
        mask = t != 0
        assert same(torch.where(mask, t, 0.0), torch.where(mask, before, 0.0))


# -------------------------------------------------------------------- refusals
def test_refusals(gpu):
    c = Cache(gpu, [40, 9], 16, 2, 64, torch.float16)
    new = offsets_of([3, 1], gpu)
    q, k, v = (queries(gpu, 4, h, 64, torch.float16, h) for h in (4, 2, 2))
    pool = dict(k_pages=c.k, v_pages=c.v, tables=c.tables, lengths=c.lengths)
    fresh = c.spare[:2].view(2, 1)
    calls = {
        "paged_append": (cr.paged_append, dict(pool, k=k, v=v, offsets=new, weights=c.w)),
        "paged_attention": (cr.paged_attention, dict(pool, q=q, offsets=new, weights=c.w)),
        "paged_evict": (cr.paged_evict, dict(pool, weights=c.w, new_tables=fresh, keep=16)),
    }
    wide = torch.zeros(5, 16, 2, 65, dtype=torch.float16, device=gpu)
    both = [dict(k_pages=a, v_pages=b) for a, b in (
        (c.k, c.v[:-1]), (c.k, c.v.transpose(1, 2).contiguous().transpose(1, 2)),
        (c.k.float(), c.v.float()), (c.k, c.v.bfloat16()), (c.k.cpu(), c.v), (c.k, c.v.cpu()),
        (c.k[0], c.v[0]), (c.k[..., :60], c.v[..., :60]), (c.k[:, :0], c.v[:, :0]),
        (wide[..., :64], wide[..., :64]), (wide[..., 1:], wide[..., 1:]),
        (c.k[:1].expand(5, -1, -1, -1), c.v[:1].expand(5, -1, -1, -1)),
        (c.k.transpose(2, 3), c.v.transpose(2, 3)), ("pages", c.v))]
    for what, (call, good) in calls.items():
        call(**good)
        bad = both + [dict(tables=c.tables.long()), dict(tables=c.tables[0]), dict(tables=c.tables.cpu()),
                      dict(tables=None), dict(lengths=c.lengths.float()), dict(lengths=c.lengths[:1]),
                      dict(lengths=c.lengths[None]), dict(weights=c.w.half()), dict(weights=c.w[:-1]),
                      dict(weights=c.w[..., :1].expand_as(c.w)), dict(weights=c.w.cpu())]
        if "offsets" in good:
            bad += [dict(offsets=new.long()), dict(offsets=new[:2]), dict(offsets=new.cpu())]
        if what == "paged_append":
            bad += [dict(k=k.bfloat16()), dict(k=k[:3]), dict(v=v[..., :56]), dict(k=k[:, :1], v=v[:, :1]),
                    dict(k=k[0]), dict(v=v.cpu())]
        if what == "paged_attention":
            bad += [dict(q=q.bfloat16()), dict(q=q[:, :3]), dict(q=q[:, :0]), dict(q=q[..., :56]),
                    dict(q=q[0]), dict(q=q.cpu())]
        if what == "paged_evict":
            bad += [dict(new_tables=fresh.long()), dict(new_tables=fresh[:1]), dict(new_tables=fresh[0]),
                    dict(keep=17), dict(weights=None)]
            with pytest.raises(ValueError, match="other pages"):
                call(**{**good, "new_tables": c.tables})
            for keep, recent in ((0, 0), (16, 17), (16, -1), (-3, 0)):
                with pytest.raises(ValueError, match=what):
                    call(**{**good, "keep": keep, "recent": recent})
        for change in bad:
            with pytest.raises(RuntimeError, match=what):
                call(**{**good, **change})
        # no derivatives
        name = {"paged_append": "k", "paged_attention": "q", "paged_evict": "k_pages"}[what]
        leaf = good[name].clone().requires_grad_(True)
        with pytest.raises(RuntimeError, match="no gradient"):
            call(**{**good, name: leaf})
        with torch.no_grad():
            call(**{**good, name: leaf})
        import torch.autograd.forward_ad as ad
        with ad.dual_level(), pytest.raises(NotImplementedError, match=what):
            call(**{**good, name: ad.make_dual(good[name], torch.zeros_like(good[name]))})
    with pytest.raises(ValueError, match="scale"):
        cr.paged_attention(**calls["paged_attention"][1], scale=math.inf)
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(lambda x: cr.paged_attention(**{**calls["paged_attention"][1], "q": x}), q)


def test_evict_refuses_the_tables_it_reads_in_any_layout(gpu):
    c = Cache(gpu, [40, 9], 16, 2, 64, torch.float16)
    by_page = c.tables.t().contiguous().t()  # neighbours in the first dimension
    assert by_page.stride(1) != 1
    for tables in (c.tables, by_page):
        before = [t.clone() for t in (c.k, c.v, c.w)]
        with pytest.raises(ValueError, match="other pages"):
            cr.paged_evict(c.k, c.v, c.w, tables, c.lengths, tables, 16)
        assert all(same(a, b) for a, b in zip(before, (c.k, c.v, c.w)))


def test_what_autograd_saved_is_told_of_writes(gpu):
    """A cache that an earlier operation's gradient needs is not overwritten unnoticed."""
    c = Cache(gpu, [40], 16, 2, 64, torch.float16)
    k = queries(gpu, 4, 2, 64, torch.float16)
    at = offsets_of([4], gpu)
    leaf = torch.ones_like(c.k).requires_grad_(True)
    calls = (lambda: cr.paged_append(k, k, *c.args(), at, weights=c.w),
             lambda: cr.paged_evict(c.k, c.v, c.w, c.tables, c.lengths, c.spare.view(1, -1), 16))
    for call in calls:
        y = (leaf * c.k).sum()
        call()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    with torch.inference_mode():
        pool = c.k.clone()
        cr.paged_append(k, k, pool, c.v.clone(), c.tables, c.lengths, at)
        assert torch.equal(pool[c.tables[0, 2].long(), 4:8], k)
