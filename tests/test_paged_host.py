"""CPU tests of the paged cache: the C entries' refusals (none of these calls launches anything),
the Python layer without a GPU, and the oracle against hand-made cases."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import helpers  # noqa: F401
import cuda_rasterizer as cr
from cuda_rasterizer import _lib
from cuda_rasterizer._lib import GsPagedQueries, GsPages
from cuda_rasterizer.paged import _layout, _pool_strides, _weight_strides
from oracle import paged as op
from oracle import tokens as ot

FAKE = 1 << 20  # 16-byte aligned, never read


def pages(**change):
    values = dict(pages=10, page_stride=16 * 2 * 64, slot_stride=2 * 64, head_stride=64, sum_page=32,
                  sum_slot=2, sum_head=1, tables=FAKE, lengths=FAKE, table_stride=4, table_width=4,
                  sequences=3, page_size=16, heads=2, dim=64, type=1)
    return GsPages(*{**values, **change}.values())


def queries(**change):
    values = dict(rows_q=5, row_stride=256, head_stride=64, offsets=FAKE, heads_q=4, causal=1, scale=0.125)
    return GsPagedQueries(*{**values, **change}.values())


INVALID, SMALL, UNSUPPORTED = -1, -2, -4
BAD_PAGES = [
    (dict(pages=-1), INVALID), (dict(sequences=-1), INVALID), (dict(page_size=0), INVALID),
    (dict(heads=0), INVALID), (dict(dim=0), INVALID), (dict(table_width=-1), INVALID),
    (dict(table_stride=-4), INVALID), (dict(page_stride=-8), INVALID), (dict(type=7), INVALID),
    (dict(tables=None), INVALID), (dict(lengths=None), INVALID), (dict(type=0), UNSUPPORTED),
    (dict(dim=60), UNSUPPORTED), (dict(dim=136, slot_stride=136), UNSUPPORTED),
    (dict(pages=1 << 31), UNSUPPORTED), (dict(page_size=1 << 20, table_width=1 << 11), UNSUPPORTED),
    (dict(slot_stride=56), UNSUPPORTED), (dict(slot_stride=(1 << 23) + 8), UNSUPPORTED),
    (dict(page_stride=1 << 31), UNSUPPORTED), (dict(head_stride=1 << 31), UNSUPPORTED),
    (dict(page_stride=1028), UNSUPPORTED), (dict(head_stride=4), UNSUPPORTED)]


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def append(lib, p, k=FAKE, row=128, rows=5, offsets=FAKE, pool=FAKE, weights=FAKE):
    return lib.gs_paged_append(ctypes.byref(p) if p else None, k, row, 64, FAKE, 128, 64, rows, offsets,
                               pool, FAKE, weights, None)


def attention(lib, p, a, q=FAKE, pool=FAKE, out=FAKE, log_sum=FAKE, weights=FAKE, ws=FAKE, size=1 << 40):
    return lib.gs_paged_attention(ctypes.byref(p) if p else None, ctypes.byref(a) if a else None, q, pool,
                                  FAKE, out, log_sum, weights, ws, size, None)


def evict(lib, p, pool=FAKE, weights=FAKE, new_tables=FAKE, width=2, keep=32, recent=4, out=FAKE):
    return lib.gs_paged_evict(ctypes.byref(p) if p else None, pool, FAKE, weights, new_tables, 2, width,
                              keep, recent, out, FAKE, None)


@pytest.mark.parametrize("change,status", BAD_PAGES)
def test_descriptions_that_are_refused(lib, change, status):
    p = pages(**change)
    size = ctypes.c_size_t(0)
    assert append(lib, p) == status
    assert attention(lib, p, queries()) == status
    assert evict(lib, p) == status
    assert lib.gs_paged_attention_workspace_size(ctypes.byref(p), ctypes.byref(queries()), 1,
                                                 ctypes.byref(size)) == status


def test_refused_arguments(lib):
    p, a = pages(), queries()
    assert append(lib, None) == attention(lib, None, a) == evict(lib, None) == INVALID
    for change in (dict(k=None), dict(rows=-1), dict(offsets=None), dict(pool=None), dict(row=-8)):
        assert append(lib, p, **change) == INVALID
    for change in (dict(k=FAKE + 2), dict(pool=FAKE + 8), dict(row=132), dict(rows=1 << 31)):
        assert append(lib, p, **change) == UNSUPPORTED
    assert attention(lib, p, None) == INVALID
    for change in (dict(rows_q=-1), dict(heads_q=0), dict(heads_q=3), dict(offsets=None),
                   dict(scale=math.nan), dict(row_stride=-8), dict(head_stride=-8)):
        assert attention(lib, p, queries(**change)) == INVALID
    for change in (dict(row_stride=260), dict(head_stride=4), dict(row_stride=56),
                   dict(row_stride=(1 << 23) + 8), dict(rows_q=1 << 31)):
        assert attention(lib, p, queries(**change)) == UNSUPPORTED
    for change in (dict(q=None), dict(out=None), dict(pool=None), dict(log_sum=None)):
        assert attention(lib, p, a, **change) == INVALID
    for change in (dict(q=FAKE + 2), dict(out=FAKE + 4), dict(pool=FAKE + 8)):
        assert attention(lib, p, a, **change) == UNSUPPORTED
    for change in (dict(keep=0), dict(recent=-1), dict(recent=33), dict(width=1), dict(new_tables=None),
                   dict(pool=None), dict(weights=None), dict(out=None)):
        assert evict(lib, p, **change) == INVALID
    assert evict(lib, p, pool=FAKE + 2) == UNSUPPORTED
    assert evict(lib, pages(sum_page=-1)) == INVALID
    for stride in ("sum_page", "sum_slot", "sum_head"):
        assert evict(lib, pages(**{stride: 1 << 31})) == UNSUPPORTED


@pytest.mark.parametrize("change", [dict(sequences=(1 << 31) - 1), dict(page_size=(1 << 31) - 1, table_width=0),
                                    dict(heads=1 << 28)])
def test_counts_near_2_31(lib, change):
    """What is one more, or a row's heads in eights, stays in 32 bits."""
    p = pages(**change)
    assert append(lib, p, rows=1) == attention(lib, p, queries(heads_q=p.heads)) == UNSUPPORTED
    assert evict(lib, p, keep=1) == UNSUPPORTED


def test_more_kept_than_slots_have_numbers(lib):
    most = (1 << 31) - 1 - 65536
    for keep in (most + 1, (1 << 31) - 1):
        assert evict(lib, pages(), keep=keep, width=1 << 27) == UNSUPPORTED


def test_more_tiles_of_weights_than_have_numbers(lib):
    """A tile of slots' weights is 128 of them: 2^24 - 520 in a table here, times sequences and heads."""
    p = pages(page_size=1 << 10, table_width=(1 << 21) - 65, sequences=65)
    assert attention(lib, p, queries()) == UNSUPPORTED
    size = ctypes.c_size_t(0)
    for sequences, weights, status in ((65, 1, UNSUPPORTED), (64, 1, 0), (1 << 16, 0, 0)):
        p.sequences = sequences
        assert lib.gs_paged_attention_workspace_size(ctypes.byref(p), ctypes.byref(queries()), weights,
                                                     ctypes.byref(size)) == status


def test_more_threads_than_a_launch_takes(lib):
    """A launch has fewer than 2^32 threads: 1024 for each sequence and head that an eviction chooses for,
    one for each 8 elements that it moves or that are appended, 256 for each tile of attention."""
    for change in (dict(sequences=1 << 21), dict(sequences=1 << 22, heads=1), dict(sequences=1 << 30)):
        assert evict(lib, pages(**change)) == UNSUPPORTED
    assert evict(lib, pages(), keep=1 << 28, width=1 << 24) == UNSUPPORTED
    assert append(lib, pages(), rows=1 << 28) == UNSUPPORTED
    p, a = pages(sequences=1 << 23), queries(rows_q=(1 << 27) + 1)
    assert attention(lib, p, a, weights=None, log_sum=None) == UNSUPPORTED


def test_more_items_of_few_rows_than_have_numbers(lib):
    """Single tokens of 2^28 sequences, 16 key heads each: an item is a sequence's tile, split and head."""
    a = queries(rows_q=1 << 28, heads_q=16, row_stride=16 * 64)
    p = pages(sequences=1 << 28, heads=16, slot_stride=16 * 64, page_stride=16 * 16 * 64)
    assert attention(lib, p, a, weights=None, log_sum=None) == UNSUPPORTED


def test_counts_that_pass_32_bits():
    """(Sizes alone: with a table of no pages they cost next to nothing.)"""
    shape, w = (1, 16, 2, 64), (None, None)
    strides = (2048, 128, 64, 1)
    assert _layout("x", shape, strides, shape, strides, *w, (3, 0), (3,))
    with pytest.raises(RuntimeError, match="too many"):
        _layout("x", shape, strides, shape, strides, *w, ((1 << 32) + 3, 0), ((1 << 32) + 3,))
    for shape, strides in (((1, 1 << 32, 1, 8), (1 << 35, 8, 8, 1)), ((1, 1, 1 << 32, 8), (8, 8, 8, 1))):
        with pytest.raises(RuntimeError, match="too many|strides"):
            _layout("x", shape, strides, shape, strides, *w, (3, 0), (3,))


def test_nothing_to_do(lib):
    """No rows or no sequences: no launch, so that the call succeeds without a GPU."""
    assert append(lib, pages(), rows=0) == 0
    assert append(lib, pages(sequences=0)) == 0
    assert attention(lib, pages(), queries(rows_q=0)) == 0
    assert evict(lib, pages(sequences=0)) == 0


def test_refuses_cpu_tensors():
    pool = torch.zeros(4, 16, 2, 64, dtype=torch.float16)
    tables = torch.zeros(1, 2, dtype=torch.int32)
    lengths, offsets = torch.ones(1, dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32)
    row = torch.zeros(1, 2, 64, dtype=torch.float16)
    weights = torch.zeros(4, 16, 2)
    with pytest.raises(RuntimeError, match="GPU only"):
        cr.paged_append(row, row, pool, pool, tables, lengths, offsets)
    with pytest.raises(RuntimeError, match="GPU only"):
        cr.paged_attention(row, pool, pool, tables, lengths, offsets)
    with pytest.raises(RuntimeError, match="GPU only"):
        cr.paged_evict(pool, pool, weights, tables, lengths, tables, 16)


def test_rows_that_overlap_are_found():
    def apart(t):
        return _pool_strides(t.shape, t.stride()) is not None

    t = torch.zeros(6, 5, 4, 8)
    assert apart(t) and apart(t.transpose(1, 2)) and apart(t[::2, 1:, :2]) and apart(t[:0])
    assert not apart(t[:1].expand(6, 5, 4, 8)) and not apart(t[:, :, :1].expand(6, 5, 4, 8))
    assert not apart(t.as_strided((6, 5, 4, 8), (160, 32, 4, 1)))
    assert not apart(t.as_strided((6, 5, 4, 8), (160, 24, 8, 1)))
    assert not apart(t.as_strided((2, 2, 2, 8), (64, 32, 12, 1))) and not apart(t[..., ::2])
    assert _pool_strides((1, 5, 1, 8), (0, 8, 3, 1)) == (0, 8, 0)
    assert _pool_strides((6, 1, 4, 8), (32, 3, 8, 1)) == (32, 8, 8)
    assert _pool_strides((6, 5, 1, 8), (1 << 31, 8, 8, 1)) is None
    assert _pool_strides((6, 5, 1, 8), (1 << 30, 1 << 24, 8, 1)) is None
    w = t[..., 0]
    assert _weight_strides(w.shape, w.stride()) == (160, 32, 8)
    assert _weight_strides((6, 5, 4), (20, 4, 0)) is None and _weight_strides((6, 5, 4), (1, 6, 30))
    assert _weight_strides((6, 5, 4), (1 << 31, 4, 1)) is None


# ----------------------------------------------------------------- the oracle
def small():
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(5, 4, 2, 8, generator=g) for _ in range(2))
    tables = torch.tensor([[3, 0, -1], [1, 4, 2]], dtype=torch.int32)
    return k, v, torch.rand(5, 4, 2, generator=g), tables


def test_oracle_appends_to_the_last_slots():
    k, v, w, tables = small()
    lengths = torch.tensor([6, 9], dtype=torch.int32)
    new = torch.randn(5, 2, 8)
    offsets = torch.tensor([0, 3, 5], dtype=torch.int32)
    k2, v2, w2 = op.append(new, -new, k, v, tables, lengths, offsets, w)
    at = [(3, 3), (0, 0), (0, 1), (4, 3), (2, 0)]  # slots 3, 4, 5 and 7, 8
    for row, (page, place) in enumerate(at):
        assert torch.equal(k2[page, place], new[row]) and torch.equal(v2[page, place], -new[row])
        assert bool((w2[page, place] == 0).all())
    assert int((k2 != k).any(3).any(2).sum()) == 5 and int((w2 != w).any(2).sum()) == 5


def test_oracle_appends_nothing_past_the_table():
    k, v, w, tables = small()
    lengths, offsets = torch.tensor([10, 13], dtype=torch.int32), torch.tensor([0, 0, 4], dtype=torch.int32)
    new = torch.randn(4, 2, 8)
    k2, _, w2 = op.append(new, new, k, v, tables, lengths, offsets, w)  # slots 9 to 12 of 12
    assert torch.equal(k2[2, 1:], new[:3]) and bool((w2[2, 1:] == 0).all())
    assert int((k2 != k).any(3).any(2).sum()) == 3


def test_oracle_attention_is_that_of_packed_rows():
    k, v, _, tables = small()
    lengths = torch.tensor([7, 10], dtype=torch.int32)
    q = torch.randn(5, 4, 8, generator=torch.Generator().manual_seed(1))
    offsets = torch.tensor([0, 3, 5], dtype=torch.int32)
    lines = [torch.cat([t[tables[b].long().clamp(min=0)].flatten(0, 1)[:n] for b, n in enumerate((7, 10))])
             for t in (k, v)]
    for causal in (False, True):
        got = op.attention(q, k, v, tables, lengths, offsets, causal)
        want = ot.attention(q, *lines, offsets, torch.tensor([0, 7, 17]), causal=causal)
        for name in ("out", "log_sum", "out_slack"):
            assert torch.allclose(got[name], want[name], rtol=1e-12)
        # every query's probabilities sum to 1
        assert math.isclose(float(got["weights"].sum()), 5 * 4, rel_tol=1e-12)
        assert int(got["weights_terms"].sum()) == (
            2 * 2 * ((5 + 6 + 7) + (9 + 10)) if causal else 2 * 2 * (3 * 7 + 2 * 10))


def test_oracle_evicts_by_hand():
    k, v, w, tables = small()
    w[3, :, 0], w[0, :, 0] = torch.tensor([1.0, 5.0, 1.0, 0.0]), torch.tensor([1.0, 2.0, 0.0, 9.0])
    lengths = torch.tensor([7, 0], dtype=torch.int32)
    new_tables = torch.tensor([[2, 4], [-1, -1]], dtype=torch.int32)
    n, kept, k2, _, w2 = op.evict(k, v, w, tables, lengths, new_tables, 5, 2)
    assert n.tolist() == [5, 0]
    assert kept[0, 0].tolist() == [0, 1, 2, 5, 6] and kept[1].flatten().tolist() == [-1] * 10
    assert torch.equal(k2[2, 1, 0], k[3, 1, 0]) and torch.equal(k2[4, 0, 0], k[0, 2, 0])
    assert w2[2, :, 0].tolist() == [1.0, 5.0, 1.0, 2.0]
