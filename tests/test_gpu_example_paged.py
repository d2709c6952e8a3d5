"""The example network's paged cache (examples/views_to_gaussians.py): views streamed through pages
against all views at once and against the slabs, pages given back by an eviction.

Tolerances as in tests/test_gpu_example.py: 24 independent roundings to bfloat16 give about
sqrt(24) 2^-9 = 1%, three times that."""

from __future__ import annotations

import os
import sys

import pytest
import torch

import helpers

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "3dgs_from_scratch_amd", "examples"))
import views_to_gaussians as example  # noqa: E402

pytestmark = pytest.mark.gpu


def dealt(cache):
    """Every page is free or one scene's."""
    pages = sorted(cache.free + [p for owned in cache.owned for p in owned])
    assert pages == list(range(cache.k.shape[1]))
    assert cache.lengths.tolist() == cache.filled
    assert all(len(o) == -(-n // cache.page) for o, n in zip(cache.owned, cache.filled))


@pytest.mark.parametrize("page", [5, 16, 64])
def test_views_over_pages_match_all_at_once(gpu, page):
    scenes = [example.make_scene(n, 64, 48, n) for n in (1, 4, 2)]
    network = example.Network(seed=2)
    with torch.no_grad():
        tokens, positions, offsets = example.packed(scenes)
        whole = network(tokens, positions, offsets)
    cache = example.PagedCache(network, len(scenes), 3 * (48 // page + 1), page)
    slabs = example.Cache(network, len(scenes), 4 * 12)
    starts = offsets[:-1].tolist()
    for i in range(4):
        views = [s[i] if i < len(s) else None for s in scenes]
        got = example.predict_next(network, cache, views, i)
        want = torch.cat([whole[starts[b] + 12 * i:starts[b] + 12 * (i + 1)]
                          for b, v in enumerate(views) if v is not None])
        assert helpers.rel_l2(got, want) <= 0.03, i
        assert helpers.rel_l2(got, example.predict_next(network, slabs, views, i)) <= 0.03, i
        dealt(cache)
    assert cache.lengths.tolist() == [12, 48, 24]
    # every query's probabilities sum to 1 in each layer: as many as there are queries and heads
    for weights in cache.weights:
        at = cache.tables[cache.tables >= 0].long()
        assert abs(float(weights[at].double().sum()) / ((12 + 48 + 24) * network.heads) - 1) <= 1e-4


def test_views_over_pages_with_evictions(gpu):
    scenes = [example.make_scene(n, 64, 48, n) for n in (6, 1, 4)]
    network = example.Network(seed=3)
    cache = example.PagedCache(network, len(scenes), 16, 8)
    free = example.PagedCache(network, len(scenes), 30, 8)
    for i in range(6):
        views = [s[i] if i < len(s) else None for s in scenes]
        got, all_kept = (example.predict_next(network, c, views, i) for c in (cache, free))
        assert bool(torch.isfinite(got).all())
        if i < 2:  # nothing has been evicted yet
            assert helpers.rel_l2(got, all_kept) <= 1e-6
        cache.evict(20, 12)
        dealt(cache)
        assert max(cache.filled) <= 20
    assert cache.filled == [20, 12, 20] and free.filled == [72, 12, 48]
    with pytest.raises(RuntimeError, match="free"):
        cache.grow([1000, 0, 0])
