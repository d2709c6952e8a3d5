"""The example network (examples/views_to_gaussians.py) with its three operators together: a
training step against the same network on plain float32 operations, training that learns, and
views streamed through a cache against all views at once.

Tolerances: the activations are bfloat16, unit roundoff 2^-8, rounded after each of about
twelve operations a block; 24 of them in two blocks, independent, give about sqrt(24) 2^-9 =
1%.  Three times that for outputs, and ten times for gradients, which pass through the
rasterizer as well and sum over few tokens."""

from __future__ import annotations

import os
import sys

import pytest
import torch

import helpers  # noqa: F401

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "3dgs_from_scratch_amd", "examples"))
import views_to_gaussians as example  # noqa: E402

pytestmark = pytest.mark.gpu


def plain(network, tokens, positions, offsets):
    """The network in float32 with elementary operations."""
    w, dim = network.weights, network.dim
    group = network.heads // network.key_heads

    def norm(x, name):
        x = x - x.mean(1, keepdim=True)
        return x / torch.sqrt((x * x).mean(1, keepdim=True) + 1e-5) * w[name + "_scale"] + w[name + "_shift"]

    def turned(x):
        axis = [a for a, n in enumerate(network.sections) for _ in range(n)]
        angle = (positions.double()[:, axis] * network.frequencies.double())[:, None]
        c, s = torch.cos(angle).float(), torch.sin(angle).float()
        u, v = x.split(dim // 2, -1)
        return torch.cat((u * c - v * s, u * s + v * c), -1)

    x = tokens @ w["embed"].t()
    bounds = offsets.tolist()
    for i in range(network.layers):
        y = (norm(x, f"attention{i}") @ w[f"qkv{i}"].t()).view(x.shape[0], -1, dim)
        q, k, v = y.split((network.heads, network.key_heads, network.key_heads), 1)
        q, k = turned(q), turned(k).repeat_interleave(group, 1)
        v = v.repeat_interleave(group, 1)
        parts = []
        for b, e in zip(bounds, bounds[1:]):
            s = torch.einsum("ihd,jhd->hij", q[b:e], k[b:e]) * dim ** -0.5
            s = s.masked_fill(torch.ones_like(s[0], dtype=torch.bool).triu(1), -float("inf"))
            parts.append(torch.einsum("hij,jhd->ihd", torch.softmax(s, 2), v[b:e]))
        x = x + torch.cat(parts).reshape(x.shape) @ w[f"proj{i}"].t()
        x = x + torch.nn.functional.gelu(norm(x, f"mlp{i}") @ w[f"up{i}"].t()) @ w[f"down{i}"].t()
    return norm(x, "last") @ w["out"].t()


def test_network_matches_plain_operations(gpu):
    scenes = [example.make_scene(n, 64, 48, 10 + n) for n in (1, 3)]
    network = example.Network(seed=1)
    batch = example.packed(scenes)
    got = network(*batch)
    want = plain(network, *batch)
    assert helpers.rel_l2(got, want) <= 0.03
    upstream = torch.randn(want.shape, generator=torch.Generator().manual_seed(0)).to(gpu)
    names = list(network.weights)
    leaves = [network.weights[n] for n in names]
    a = torch.autograd.grad(got, leaves, upstream)
    b = torch.autograd.grad(want, leaves, upstream)
    for n, x, y in zip(names, a, b):
        assert x.dtype == torch.float32 and helpers.rel_l2(x, y) <= 0.1, n


def test_training_learns_through_the_rasterizer(gpu):
    losses, network, scenes, batch = example.train(steps=25, width=64, height=48, say=None)
    assert all(x == x for x in losses) and losses[-1] < 0.9 * losses[0], losses
    grads = {n: t.grad for n, t in network.weights.items()}
    assert all(g is not None and bool(torch.isfinite(g).all()) for g in grads.values())
    assert sum(float(g.abs().max()) > 0 for g in grads.values()) == len(grads)


def test_views_one_by_one_match_all_at_once(gpu):
    scenes = [example.make_scene(n, 64, 48, n) for n in (1, 4, 2)]
    network = example.Network(seed=2)
    with torch.no_grad():
        tokens, positions, offsets = example.packed(scenes)
        whole = network(tokens, positions, offsets)
    cache = example.Cache(network, len(scenes), 4 * 12)
    starts = offsets[:-1].tolist()
    for i in range(4):
        views = [s[i] if i < len(s) else None for s in scenes]
        got = example.predict_next(network, cache, views, i)
        want = torch.cat([whole[starts[b] + 12 * i:starts[b] + 12 * (i + 1)]
                          for b, v in enumerate(views) if v is not None])
        assert helpers.rel_l2(got, want) <= 0.03, i
    assert cache.lengths.tolist() == [12, 48, 24]
