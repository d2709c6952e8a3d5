"""CPU tests of the example's page bookkeeping (PagedCache of examples/views_to_gaussians.py): what is left
where there is no room, with the oracle's eviction in place of the kernels'."""

from __future__ import annotations

import os
import sys
import types

import pytest
import torch

import helpers  # noqa: F401
from oracle import paged as op

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "3dgs_from_scratch_amd", "examples"))
import views_to_gaussians as example  # noqa: E402


def evict(k_pages, v_pages, weights, tables, lengths, new_tables, keep, recent):
    if keep < 1 or not 0 <= recent <= keep:
        raise ValueError("paged_evict: keep must be at least 1 and recent from 0 to keep")
    fresh = new_tables.flatten().tolist()
    assert len(set(fresh)) == len(fresh) and not set(fresh) & set(tables.flatten().tolist())
    lengths, kept, *pools = op.evict(k_pages, v_pages, weights, tables, lengths, new_tables, keep, recent)
    for t, new in zip((k_pages, v_pages, weights), pools):
        t.copy_(new)
    return lengths, kept


@pytest.fixture
def cache(monkeypatch):
    """make(pages, width): three scenes in pages of 4."""
    monkeypatch.setattr(example, "paged_evict", evict)
    network = types.SimpleNamespace(layers=2, key_heads=1, dim=8)

    def make(pages, width=None):
        return example.PagedCache(network, 3, pages, 4, width, device="cpu")
    return make


def state(c):
    return (c.filled[:], [o[:] for o in c.owned], c.free[:], c.tables.tolist(), c.lengths.tolist())


def fill(c, new):
    """What a view's tokens leave: their room, the slots' numbers as keys, and the lengths."""
    c.grow(new)
    c.lengths += torch.tensor(new, dtype=torch.int32)
    for b, n in enumerate(c.filled):
        for slot in range(n):
            at = (slice(None), c.owned[b][slot // c.page], slot % c.page)
            c.k[at], c.v[at], c.weights[at] = slot, 100 * b + slot, (slot * 7) % 5


def dealt(c):
    """Every page is free or one scene's, and the tables and lengths say the same."""
    assert sorted(c.free + [p for o in c.owned for p in o]) == list(range(c.k.shape[1]))
    assert c.lengths.tolist() == c.filled
    for row, owned, n in zip(c.tables.tolist(), c.owned, c.filled):
        assert row == owned + [-1] * (len(row) - len(owned)) and len(owned) == -(-n // c.page)


@pytest.mark.parametrize("pages,width,message", [(7, None, "free"), (20, 2, "tables")])
def test_no_room_to_grow_changes_nothing(cache, pages, width, message):
    c = cache(pages, width)
    fill(c, [8, 4, 5])
    before = state(c)
    with pytest.raises(RuntimeError, match=message):
        c.grow([0, 5, 4])  # three pages more, and three a scene
    assert state(c) == before
    fill(c, [0, 4, 3])
    dealt(c)


def test_an_eviction_without_room_changes_nothing(cache):
    c = cache(9)
    fill(c, [12, 12, 10])
    before = state(c)
    with pytest.raises(RuntimeError, match="free"):
        c.evict(5, 2)
    assert state(c) == before


def test_an_eviction_that_is_refused_changes_nothing(cache):
    c = cache(30)
    fill(c, [12, 12, 10])
    before = state(c)
    for keep, recent in ((5, 6), (5, -1), (0, 0)):
        with pytest.raises(ValueError, match="paged_evict"):
            c.evict(keep, recent)
        assert state(c) == before


@pytest.mark.parametrize("pages", [11, 12, 13, 30])
def test_scenes_leave_in_turn_where_few_pages_are_free(cache, pages):
    c = cache(pages)
    fill(c, [12, 12, 10])
    c.evict(5, 2)
    dealt(c)
    assert c.filled == [5, 5, 5]
    for b, n in enumerate((12, 12, 10)):
        rank = sorted(range(n - 2), key=lambda s: (-((s * 7) % 5), s))[:3]
        kept = sorted(rank) + [n - 2, n - 1]
        for layer in range(2):
            got = [int(c.v[layer, c.owned[b][i // 4], i % 4, 0, 0]) for i in range(5)]
            assert got == [int(torch.tensor(100.0 * b + s).bfloat16()) for s in kept]
    c.grow([3, 0, 1])
