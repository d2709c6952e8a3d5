"""A small network that predicts Gaussians from posed images, trained through the rasterizer.

Every 16x16 tile of a view is a token: its pixels and the rays through them.  Tokens of a
scene's views follow one another, scenes of different numbers of views are packed, and each
token sees its scene's views up to its own place (causal), so that views may arrive one by one:
`predict_next` gives a new view's Gaussians from its tokens and a cache of the earlier views'
keys and values, without looking at those again.

A block is  x += attention(layer_norm(x));  x += mlp(layer_norm(x))  with
  layer_norm        normalisation (bfloat16 tokens, float32 weights)
  axial_rotary      rotary positions by view, tile row and tile column
  packed_attention  grouped heads over the packed scenes, or over the cache
and the last layer gives each token a grid of Gaussians along its rays, which render_l1 draws and
compares with a view; the loss goes back through all of it into float32 weights.

    PYTHONPATH=3dgs_from_scratch_amd python 3dgs_from_scratch_amd/examples/views_to_gaussians.py
"""

from __future__ import annotations

import argparse
import math

import torch

from cuda_rasterizer import axial_frequencies, axial_rotary, layer_norm, packed_attention
from cuda_rasterizer.fused import render_l1
from cuda_rasterizer.train import FusedAdam
from cuda_rasterizer.wrapper import render

TILE = 16
GRID = 4                 # Gaussians of a token: GRID x GRID, one for 4 x 4 pixels
SIDE = TILE // GRID
PER_GAUSSIAN = 12        # depth, offset (2), log-scale (3), quaternion (4), opacity, spare
NEAR, FAR = 1.5, 6.5


class Network:
    """Weights by name (float32 leaves) and the passes over them."""

    def __init__(self, width=256, heads=4, key_heads=2, layers=2, device="cuda", seed=0):
        g = torch.Generator().manual_seed(seed)
        self.heads, self.key_heads, self.layers, self.width = heads, key_heads, layers, width
        self.dim = width // heads
        pairs = self.dim // 2
        rows = (pairs - pairs // 8) // 2
        self.sections = (pairs // 8, rows, pairs - pairs // 8 - rows)
        self.frequencies = axial_frequencies(self.sections, 100.0, device)
        inputs, outputs = TILE * TILE * 9, GRID * GRID * PER_GAUSSIAN

        def matrix(rows, columns, scale=1.0):
            return torch.randn(rows, columns, generator=g) * (scale / math.sqrt(columns))

        self.weights = {"embed": matrix(width, inputs), "out": matrix(outputs, width, 0.1)}
        for i in range(layers):
            self.weights |= {
                f"qkv{i}": matrix((heads + 2 * key_heads) * self.dim, width),
                f"proj{i}": matrix(width, width, 0.5),
                f"up{i}": matrix(4 * width, width), f"down{i}": matrix(width, 4 * width, 0.5)}
        for name in [f"{n}{i}" for i in range(layers) for n in ("attention", "mlp")] + ["last"]:
            self.weights[name + "_scale"] = torch.ones(width)
            self.weights[name + "_shift"] = torch.zeros(width)
        self.weights = {k: v.to(device).requires_grad_(True) for k, v in self.weights.items()}

    def _times(self, x, name):
        return x @ self.weights[name].to(x.dtype).t()

    def _norm(self, x, name):
        return layer_norm(x, self.weights[name + "_scale"], self.weights[name + "_shift"])

    def __call__(self, tokens, positions, offsets, cache=None):
        """A grid of Gaussians for each token; offsets say where the scenes begin.  With a
        cache (see Cache) the tokens are new ones of its scenes, and it is filled."""
        x = self._times(tokens.to(torch.bfloat16), "embed")
        for i in range(self.layers):
            y = self._times(self._norm(x, f"attention{i}"), f"qkv{i}")
            q, k, v = y.view(x.shape[0], -1, self.dim).split(
                (self.heads, self.key_heads, self.key_heads), 1)
            q, k = axial_rotary(q, k, positions, self.frequencies, self.sections)
            if cache is None:
                y = packed_attention(q, k, v, offsets, causal=True)
            else:
                y = cache.attend(i, q, k, v, offsets)
            x = x + self._times(y.reshape(x.shape), f"proj{i}")
            y = torch.nn.functional.gelu(self._times(self._norm(x, f"mlp{i}"), f"up{i}"))
            x = x + self._times(y, f"down{i}")
        if cache is not None:
            cache.lengths += offsets.diff()
        return self._times(self._norm(x, "last"), "out").float()


class Cache:
    """Keys and values of the views so far: `slab` tokens a scene, `lengths` of them filled."""

    def __init__(self, network, scenes, slab, device="cuda"):
        shape = (network.layers, scenes * slab, network.key_heads, network.dim)
        self.k = torch.empty(shape, dtype=torch.bfloat16, device=device)
        self.v = torch.empty(shape, dtype=torch.bfloat16, device=device)
        self.lengths = torch.zeros(scenes, dtype=torch.int32, device=device)
        self.offsets = torch.arange(scenes + 1, dtype=torch.int32, device=device) * slab

    def attend(self, layer, q, k, v, offsets):
        new = offsets.diff()
        scene = torch.repeat_interleave(torch.arange(new.shape[0], device=q.device), new,
                                        output_size=q.shape[0])
        at = (self.offsets[:-1] + self.lengths - offsets[:-1])[scene] + torch.arange(
            q.shape[0], device=q.device)
        self.k[layer, at], self.v[layer, at] = k, v
        return packed_attention(q, self.k[layer], self.v[layer], offsets, self.offsets,
                                self.lengths + new, causal=True)


# --------------------------------------------------------------- views and tokens
def rays(w2c, K, width, height):
    """Origins and directions (camera z = 1) of the pixels' rays in the world, (H, W, 3)."""
    v, u = torch.meshgrid(torch.arange(height, device=w2c.device) + 0.5,
                          torch.arange(width, device=w2c.device) + 0.5, indexing="ij")
    local = torch.stack([(u - K[0, 2]) / K[0, 0], (v - K[1, 2]) / K[1, 1], torch.ones_like(u)], -1)
    return (-w2c[:3, :3].t() @ w2c[:3, 3]).expand_as(local), local @ w2c[:3, :3]


def tokens_of(view, number):
    """(tokens, positions) of one view: its tiles' pixels, colours and rays, row by row."""
    image, w2c, K = view
    h, w = image.shape[:2]
    origin, direction = rays(w2c, K, w, h)
    x = torch.cat((image * 2 - 1, origin / 4, direction), 2)
    x = x.view(h // TILE, TILE, w // TILE, TILE, 9).permute(0, 2, 1, 3, 4)
    x = x.reshape(-1, TILE * TILE * 9)
    row, column = torch.meshgrid(torch.arange(h // TILE), torch.arange(w // TILE), indexing="ij")
    at = torch.stack([torch.full_like(row, number), row, column], -1).view(-1, 3)
    return x, at.to(device=image.device, dtype=torch.int32)


def gaussians_of(grids, view):
    """Raw parameters for render_l1 from the grids of one view's tokens: each Gaussian lies on
    the ray of its 4 x 4 pixels, as far as the network says, in the colour of the image there."""
    image, w2c, K = view
    h, w = image.shape[:2]
    origin, direction = rays(w2c, K, w, h)

    def cells(x):
        x = x.view(h // TILE, GRID, SIDE, w // TILE, GRID, SIDE, 3).mean((2, 5))
        return x.permute(0, 2, 1, 3, 4).reshape(-1, 3)

    p = grids.reshape(-1, PER_GAUSSIAN)
    depth = NEAR + (FAR - NEAR) * torch.sigmoid(p[:, :1])
    size = depth * (SIDE / 2) / K[0, 0]
    means = cells(origin) + depth * cells(direction)
    aside = torch.cat((torch.tanh(p[:, 1:3]), torch.zeros_like(depth)), 1)
    means = means + 0.5 * size * aside @ w2c[:3, :3]
    scales = torch.log(size) + torch.tanh(p[:, 3:6])
    quats = p[:, 6:10] + p.new_tensor([0.0, 0.0, 0.0, 1.0])
    dc = (cells(image) - 0.5) / 0.28209479177387814
    return means, scales, quats, p[:, 10] + 2.0, dc, dc.new_zeros(p.shape[0], 15, 3)


def make_scene(views, width, height, seed, device="cuda"):
    """A ball of random Gaussians seen from an arc: [(image in [0, 1], w2c, K)]."""
    g = torch.Generator().manual_seed(seed)
    n = 400
    means = torch.randn(n, 3, generator=g) * 0.5
    scales = torch.exp(torch.randn(n, 3, generator=g) * 0.3 - 2.2)
    quats = torch.nn.functional.normalize(torch.randn(n, 4, generator=g), dim=1)
    opacity, dc = torch.rand(n, generator=g) * 0.5 + 0.5, torch.randn(n, 3, generator=g) * 0.8
    K = torch.tensor([[1.2 * width, 0, width / 2], [0, 1.2 * width, height / 2], [0, 0, 1.0]])
    out = []
    for i in range(views):
        angle = 0.35 * (i - (views - 1) / 2)
        forward = torch.tensor([math.sin(angle), 0.0, math.cos(angle)])
        right = torch.tensor([math.cos(angle), 0.0, -math.sin(angle)])
        w2c = torch.eye(4)
        w2c[:3, :3] = torch.stack([right, torch.tensor([0.0, 1.0, 0.0]), forward])
        w2c[:3, 3] = -w2c[:3, :3] @ (-4.0 * forward)
        args = [t.to(device) for t in (w2c, K)]
        with torch.no_grad():
            image = render(*args, width, height, *(t.to(device) for t in (
                means, scales, quats, opacity, dc, torch.zeros(n, 15, 3))))[0] / 255
        out.append((image, *args))
    return out


def packed(scenes):
    """Tokens and positions of all views of all scenes, and where the scenes begin."""
    parts = [[tokens_of(v, i) for i, v in enumerate(views)] for views in scenes]
    lengths = [sum(t.shape[0] for t, _ in scene) for scene in parts]
    flat = [p for scene in parts for p in scene]
    device = flat[0][0].device
    offsets = torch.tensor([0] + lengths, device=device).cumsum(0).to(torch.int32)
    return torch.cat([t for t, _ in flat]), torch.cat([p for _, p in flat]), offsets


def loss_of(network, scenes, batch):
    """Each scene's Gaussians of all its views, drawn into its first and its last view."""
    grids = network(*batch)
    loss, at = 0.0, 0
    for views in scenes:
        parts = []
        for view in views:
            n = view[0].shape[0] * view[0].shape[1] // TILE ** 2
            parts.append(gaussians_of(grids[at:at + n], view))
            at += n
        raw = [torch.cat(p) for p in zip(*parts)]
        for image, w2c, K in (views[0], views[-1]):
            h, w = image.shape[:2]
            loss = loss + render_l1(w2c, K, w, h, *raw, image, far_plane=50.0)[0] / (2 * len(scenes))
    return loss


def train(steps=60, width=128, height=96, seed=0, lr=1e-3, say=print):
    """Losses of the steps, and the network, scenes and their tokens."""
    scenes = [make_scene(n, width, height, seed + n) for n in (1, 4, 2)]
    network = Network(seed=seed)
    batch = packed(scenes)
    optimizer = FusedAdam(network.weights, {k: lr for k in network.weights}, eps=1e-8)
    losses = []
    for step in range(steps):
        optimizer.zero_grad()
        loss = loss_of(network, scenes, batch)
        loss.backward()
        optimizer.step()
        losses.append(loss.detach())
        if say and step % 10 == 0:
            say(f"step {step}: loss {float(losses[-1]):.4f}")
    return [float(x) for x in losses], network, scenes, batch


@torch.no_grad()
def predict_next(network, cache, views, number):
    """Grids of the next view of each scene (None: no new view), the cache's scenes as they are."""
    parts = [tokens_of(v, number) for v in views if v is not None]
    lengths = [0 if v is None else v[0].shape[0] * v[0].shape[1] // TILE ** 2 for v in views]
    offsets = torch.tensor([0] + lengths, device=cache.lengths.device).cumsum(0).to(torch.int32)
    return network(torch.cat([t for t, _ in parts]), torch.cat([p for _, p in parts]), offsets, cache)


def main():
    args = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    args.add_argument("--steps", type=int, default=200)
    args.add_argument("--width", type=int, default=128, help="of a view, a multiple of 16")
    args.add_argument("--height", type=int, default=96)
    a = args.parse_args()
    losses, network, scenes, batch = train(a.steps, a.width, a.height)
    print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f}")
    # the same Gaussians, a view at a time
    with torch.no_grad():
        whole = network(*batch)
    per_view = a.width * a.height // TILE ** 2
    most = max(len(s) for s in scenes)
    cache = Cache(network, len(scenes), most * per_view)
    worst, starts = 0.0, batch[2][:-1].tolist()
    for i in range(most):
        there = [b for b, s in enumerate(scenes) if i < len(s)]
        got = predict_next(network, cache, [s[i] if i < len(s) else None for s in scenes], i)
        want = torch.cat([whole[starts[b] + i * per_view:starts[b] + (i + 1) * per_view] for b in there])
        worst = max(worst, float((got - want).norm() / want.norm()))
    print(f"a view at a time against all at once: {worst:.4f} apart")


if __name__ == "__main__":
    main()
