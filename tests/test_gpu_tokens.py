"""GPU parity of the patch-network operators (layer_norm, axial_rotary,
packed_attention) against the float64 oracle (oracle/tokens.py).

Tolerances, with u the unit roundoff of the output's type (2^-24, 2^-11, 2^-8) and
e = 2^-24:
- layer norm: an output is rounded once (u), its float arithmetic is a few e of the
  values that meet in it; u + 64 e relative to a row's largest value.  A weight's
  gradient: u of itself and 272 e of the sum of its absolute terms (chains of at
  most 256 float additions).
- rotary: 2 values of at most the pair's length, u + 8 e of that length.
- attention: `slack` of the oracle times u: probabilities and score gradients
  rounded to the type, delta from the rounded output.  float16 probabilities below
  2^-14 are rounded absolutely, 2^-24 at most each.  Scores in float add
  (dim + 16) e of sum |q k|, relative to a probability.
"""

from __future__ import annotations

import math

import pytest
import torch

import helpers  # noqa: F401
import cuda_rasterizer as cr
from cuda_rasterizer import tokens
from cuda_rasterizer.graphs import CapturedStep
from oracle import tokens as ot

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def within(got, want, tolerance, what=""):
    got = got.double()
    assert got.shape == want.shape
    assert bool(torch.isfinite(got).all()) or not bool(torch.isfinite(want).all()), what
    over = (got - want).abs() - tolerance
    assert not over.numel() or float(over.max()) <= 0.0, (
        what, float((got - want).abs().max()), float(over.max()))


def rng(gpu, seed):
    return torch.Generator(device=gpu).manual_seed(seed)


def randn(g, *shape):
    return torch.randn(shape, generator=g, device=g.device)


# ------------------------------------------------------------------ layer norm
def norm_inputs(gpu, rows, channels, dtype, wdtype, seed=0):
    g = rng(gpu, 1000 * rows + channels + seed)
    x = (randn(g, rows, channels) * torch.exp(randn(g, channels)) + 3 * randn(g, channels)).to(dtype)
    w, b = (1 + 0.3 * randn(g, channels)).to(wdtype), (0.2 * randn(g, channels)).to(wdtype)
    return x, w, b, randn(g, rows, channels).to(dtype)


def check_norm(x, w, b, gy, eps=1e-5, run=None):
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x, w, b)]
    y = (run or cr.layer_norm)(*leaves, eps)
    given = [t for t in leaves if t is not None]
    grads = iter(torch.autograd.grad(y, given, gy))
    gx, gw, gb = (next(grads) if t is not None else None for t in leaves)
    want = ot.layer_norm(x, w, b, eps)
    u = U[x.dtype] + 64 * E
    if x.numel():
        size = x.double().abs().amax(-1, keepdim=True)
        away = (x.double() - x.double().mean(-1, keepdim=True))
        # a channel's value loses e of the row's largest value before it is divided
        r = 1 / torch.sqrt((away ** 2).mean(-1, keepdim=True) + eps)
        wide = 1.0 if w is None else w.double().abs()
        within(y.detach(), want, u * want.abs() + 64 * E * ((size * r + 1) * wide + want.abs()), "y")
        wx, ww, wb, sw, sb = ot.layer_norm_backward(gy, x, w, eps)
        scale = (r * (gy.double() * wide).abs().amax(-1, keepdim=True) * (1 + size * r))
        within(gx, wx, U[x.dtype] * wx.abs() + 64 * E * scale, "gx")
        if gw is not None:
            lost = 64 * E * (gy.double().abs() * (size * r)).flatten(0, -2).sum(0)
            within(gw, ww, U[w.dtype] * ww.abs() + 272 * E * sw + lost, "gw")
        if gb is not None:
            within(gb, wb, U[b.dtype] * wb.abs() + 272 * E * sb, "gb")
    assert y.dtype == x.dtype and y.is_contiguous()
    return y, gx, gw, gb


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,channels", [(1, 1), (3, 7), (1, 768), (17, 64), (130, 100),
                                           (33, 1000), (300, 771), (65, 1024), (5, 4096),
                                           (2, 8192), (3, 9001), (2, 40000)])
def test_layer_norm(gpu, rows, channels, dtype):
    check_norm(*norm_inputs(gpu, rows, channels, dtype, torch.float32))


@pytest.mark.parametrize("dtype,wdtype", [(torch.float16, torch.float16),
                                          (torch.bfloat16, torch.bfloat16),
                                          (torch.float32, torch.bfloat16)])
def test_layer_norm_weight_types(gpu, dtype, wdtype):
    check_norm(*norm_inputs(gpu, 1000, 384, dtype, wdtype))


def test_layer_norm_many_rows(gpu):
    check_norm(*norm_inputs(gpu, 40_001, 96, torch.bfloat16, torch.float32))
    check_norm(*norm_inputs(gpu, 70_003, 9, torch.float32, torch.float32))


def test_layer_norm_without_weights_and_gradients(gpu):
    x, w, b, gy = norm_inputs(gpu, 20, 130, torch.float16, torch.float32)
    check_norm(x, None, None, gy)
    check_norm(x, w, None, gy)
    check_norm(x, None, b, gy)
    only = w.clone().requires_grad_(True)  # a frozen x and bias
    (gw,) = torch.autograd.grad(cr.layer_norm(x, only, b), only, gy)
    whole = check_norm(x, w, b, gy)
    _, ww, _, sw, _ = ot.layer_norm_backward(gy, x, w)
    within(gw, ww, U[w.dtype] * ww.abs() + 400 * E * sw)
    with torch.no_grad():
        assert torch.equal(cr.layer_norm(x, w, b), whole[0])


@pytest.mark.parametrize("channels", [64, 66, 71])
def test_layer_norm_strided_rows_and_shapes(gpu, channels):
    x, w, b, gy = norm_inputs(gpu, 24, channels, torch.bfloat16, torch.float32)
    wide = torch.full((24, channels + 9), math.nan, dtype=x.dtype, device=gpu)
    wide[:, 5:5 + channels] = x
    base = check_norm(x, w, b, gy)
    check_norm(wide[:, 5:5 + channels], w, b, gy)
    check_norm(wide[:, 5:5 + channels], w, b, wide[:, 5:5 + channels])
    y = cr.layer_norm(x.view(2, 3, 4, channels), w, b)
    assert torch.equal(y.view(24, channels), base[0]) and y.shape == (2, 3, 4, channels)
    y = cr.layer_norm(x.t().contiguous().t(), w, b)  # channels apart in memory
    assert torch.equal(y, base[0])
    spread = gy[:1].expand(24, channels)  # a broadcast gradient: row stride 0
    check_norm(x, w, b, spread)
    assert cr.layer_norm(x[3], w, b).equal(base[0][3])


def test_layer_norm_no_rows_and_constant_rows(gpu):
    x = torch.zeros(0, 33, device=gpu)
    w = torch.ones(33, device=gpu)
    y, gx, gw, gb = check_norm(x, w, w, x)
    assert gx.shape == (0, 33) and bool((gw == 0).all()) and bool((gb == 0).all())
    x = torch.full((5, 64), 3.0, device=gpu)
    assert bool((cr.layer_norm(x) == 0).all())
    # a row with a NaN is NaN, the others are not touched by it
    x = randn(rng(gpu, 5), 6, 40)
    x[2, 7] = math.nan
    x[4, 1] = math.inf
    y = cr.layer_norm(x)
    bad = torch.isnan(y).all(1)
    assert bad.tolist() == [False, False, True, False, True, False]
    assert bool(torch.isfinite(y[[0, 1, 3, 5]]).all())


def test_layer_norm_offset_far_from_zero(gpu):
    """Means of a thousand deviations: the variance is not a difference of squares."""
    g = rng(gpu, 6)
    x = 1000.0 + randn(g, 50, 512)
    check_norm(x, None, None, randn(g, 50, 512))


def test_layer_norm_rows_past_32_bits(gpu):
    wide = torch.zeros(40_000, 65_536, dtype=torch.float16, device=gpu)  # 2.6e9 elements
    x, w, b, gy = norm_inputs(gpu, 40_000, 16, torch.float16, torch.float32)
    wide[:, :16] = x
    check_norm(wide[:, :16], w, b, gy)


def test_layer_norm_is_deterministic(gpu):
    args = norm_inputs(gpu, 5000, 200, torch.bfloat16, torch.float32)
    one, two = check_norm(*args), check_norm(*args)
    assert all(torch.equal(a, b) for a, b in zip(one, two))


def test_layer_norm_refusals(gpu):
    x = torch.zeros(4, 8, device=gpu)
    for bad in (dict(weight=torch.zeros(7, device=gpu)), dict(weight=torch.zeros(2, 4, device=gpu)),
                dict(weight=torch.zeros(8, device=gpu), bias=torch.zeros(8, device=gpu).half()),
                dict(weight=torch.zeros(8)), dict(bias=torch.zeros(8, device=gpu).double())):
        with pytest.raises(RuntimeError, match="layer_norm"):
            cr.layer_norm(x, **bad)
    with pytest.raises(RuntimeError, match="layer_norm"):
        cr.layer_norm(x.double())
    with pytest.raises(RuntimeError, match="layer_norm"):
        cr.layer_norm(x[:, :0])
    with pytest.raises(ValueError, match="eps"):
        cr.layer_norm(x, eps=-1.0)


# ---------------------------------------------------------------------- rotary
def check_rotary(q, k, positions, f, sections, interleaved, gq=None, gk=None):
    q, k = q.detach().requires_grad_(True), None if k is None else k.detach().requires_grad_(True)
    out = cr.axial_rotary(q, k, positions, f, sections, interleaved=interleaved)
    given = [(t, o, g) for t, o, g in zip((q, k), out, (gq, gk)) if t is not None]
    grads = torch.autograd.grad([o for _, o, _ in given], [t for t, _, _ in given],
                                [g for _, _, g in given])
    for (t, o, g), gt in zip(given, grads):
        for got, x, back in ((o.detach(), t.detach(), False), (gt, g, True)):
            want = ot.rotary(x, positions, f, sections, interleaved, back)
            p = sum(sections)
            size = torch.zeros_like(want)
            a, b = (slice(0, 2 * p, 2), slice(1, 2 * p, 2)) if interleaved else (slice(0, p),
                                                                              slice(p, 2 * p))
            length = torch.hypot(x.double()[..., a], x.double()[..., b])
            size[..., a], size[..., b] = length, length
            within(got, want, (U[x.dtype] + 8 * E) * size)
            assert got.is_contiguous() and torch.equal(got[..., 2 * p:], x[..., 2 * p:])
    return out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens_,heads,key_heads,dim,sections", [
    (1, 1, 1, 2, (1,)), (5, 3, 1, 64, (4, 14, 14)), (77, 4, 4, 72, (6, 10, 20)),
    (33, 2, 1, 128, (8, 28, 28)), (1000, 16, 4, 96, (6, 10, 12, 8)), (13, 5, 5, 10, (1, 2)),
    (9, 2, 2, 7, (0, 3)), (6, 2, 1, 16, (0, 0)), (3, 1, 1, 520, (100, 120))])
def test_axial_rotary(gpu, tokens_, heads, key_heads, dim, sections, interleaved, dtype):
    g = rng(gpu, tokens_ + dim)
    positions = torch.randint(0, 300, (tokens_, len(sections)), generator=g, device=gpu,
                              dtype=torch.int32)
    f = cr.axial_frequencies(sections, 100.0, gpu)
    q, gq = (randn(g, tokens_, heads, dim).to(dtype) for _ in range(2))
    k, gk = (randn(g, tokens_, key_heads, dim).to(dtype) for _ in range(2))
    check_rotary(q, k, positions, f, sections, interleaved, gq, gk)


@pytest.mark.parametrize("ptype", [torch.int64, torch.float32])
def test_axial_rotary_position_types_and_large_positions(gpu, ptype):
    """Positions up to 10^6 (and between the numbers): the angle is not a float product."""
    g = rng(gpu, 8)
    positions = torch.randint(-10**6, 10**6, (50, 2), generator=g, device=gpu).to(ptype)
    if ptype == torch.float32:
        positions = positions / 7
    q, gq = (randn(g, 50, 2, 32) for _ in range(2))
    f = cr.axial_frequencies((7, 9), 100.0, gpu)
    check_rotary(q, None, positions, f, (7, 9), False, gq)


def test_axial_rotary_layouts(gpu):
    g = rng(gpu, 9)
    t, f = 40, cr.axial_frequencies((8, 24), 100.0, gpu)
    positions = torch.randint(0, 100, (t, 3), generator=g, device=gpu, dtype=torch.int32)[:, 1:]
    for dtype in TYPES:
        qkv = randn(g, t, 8, 64).to(dtype)
        gq, gk = randn(g, t, 4, 64).to(dtype), randn(g, t, 2, 64).to(dtype)
        dense = check_rotary(qkv[:, :4].contiguous(), qkv[:, 4:6].contiguous(), positions, f,
                             (8, 24), False, gq, gk)
        apart = qkv.transpose(0, 1).contiguous().transpose(0, 1)  # heads outermost
        odd = torch.empty(t * 8 * 64 + 1, dtype=dtype, device=gpu)[1:].view(t, 8, 64)
        odd.copy_(qkv)  # not on a 16-byte boundary
        gaps = torch.empty(t, 8, 67, dtype=dtype, device=gpu)[..., 1:65]
        gaps.copy_(qkv)
        for x in (qkv, apart, odd, gaps):
            got = check_rotary(x[:, :4], x[:, 4:6], positions, f, (8, 24), False, gq, gk)
            assert torch.equal(got[0], dense[0]) and torch.equal(got[1], dense[1])
        wide = gq[:1].expand(t, 4, 64)
        check_rotary(qkv[:, :4], None, positions, f, (8, 24), False, wide)
    # no tokens, and a gradient of one output only
    none = cr.axial_rotary(qkv[:0, :4], qkv[:0, 4:6], positions[:0], f, (8, 24))
    assert none[0].shape == (0, 4, 64)
    q, k = qkv[:, :4].clone().requires_grad_(True), qkv[:, 4:6].clone().requires_grad_(True)
    a, _ = cr.axial_rotary(q, k, positions, f, (8, 24))
    gq2, gk2 = torch.autograd.grad(a, (q, k), gq, allow_unused=True)
    assert gk2 is None and gq2.shape == q.shape


def test_axial_rotary_rows_past_32_bits(gpu):
    wide = torch.zeros(40_000, 1, 65_536, dtype=torch.float16, device=gpu)
    g = rng(gpu, 10)
    x = randn(g, 40_000, 1, 16).half()
    wide[..., :16] = x
    positions = torch.randint(0, 100, (40_000, 1), generator=g, device=gpu, dtype=torch.int32)
    f = cr.axial_frequencies((8,), 100.0, gpu)
    assert torch.equal(cr.axial_rotary(wide[..., :16], None, positions, f, (8,))[0],
                       cr.axial_rotary(x, None, positions, f, (8,))[0])


def test_axial_rotary_refusals(gpu):
    q = torch.zeros(4, 2, 16, device=gpu)
    pos, f = torch.zeros(4, 2, dtype=torch.int32, device=gpu), torch.ones(8, device=gpu)
    good = dict(q=q, k=q, positions=pos, frequencies=f, sections=(4, 4))
    cr.axial_rotary(**good)
    for bad in (dict(sections=(4, 5)), dict(sections=(4,)), dict(sections=(1, 1, 1, 1, 4)),
                dict(sections=(9, -1)), dict(sections=()), dict(k=q.half()), dict(k=q[:3]),
                dict(k=q[..., :8]), dict(positions=pos[:3]), dict(positions=pos.half()),
                dict(positions=pos.cpu()), dict(frequencies=f[:7]), dict(frequencies=f.double()),
                dict(q=q.double()), dict(q=q[0])):
        with pytest.raises(RuntimeError, match="axial_rotary"):
            cr.axial_rotary(**{**good, **bad})


# ------------------------------------------------------------------- attention
def offsets_of(lengths, gpu, first=0):
    return torch.tensor([first] + lengths, device=gpu).cumsum(0).to(torch.int32)


def bounds(ref, name, dtype, dim, reach, f16_terms):
    """Tolerance of an output: see the module's text."""
    u = U[dtype] * ref[name + "_slack"] + 2 * (dim + 16) * E * reach * ref[name + "_slack"]
    return u + (2.0 ** -24 * f16_terms if dtype == torch.float16 else 0.0) + 1e-30


def check_attention(q, k, v, oq, ok=None, lk=None, causal=False, scale=None, go=None):
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out, log_sum = cr.packed_attention(*leaves, oq, ok, lk, causal=causal, scale=scale,
                                       return_log_sum=True)
    grads = torch.autograd.grad(out, leaves, go) if go is not None else ()
    # rows that no query sees may hold anything: the oracle gets zeros there
    kc, vc = k.clone(), v.clone()
    seen = torch.zeros(k.shape[0], dtype=torch.bool, device=k.device)
    for _, _, k0, k1 in ot.spans(oq, oq if ok is None else ok, lk, q.shape[0], k.shape[0]):
        seen[k0:k1] = True
    kc[~seen], vc[~seen] = 0, 0
    ref = ot.attention(q, kc, vc, oq, ok, lk, causal, scale, go)
    dim, dtype = q.shape[2], q.dtype
    c = abs(dim ** -0.5 if scale is None else scale)
    size = lambda t: float(t.double().abs().amax()) if t.numel() else 0.0  # noqa: E731
    reach = c * size(q.double().norm(dim=2)) * size(kc.double().norm(dim=2))
    keys = max([k1 - k0 for _, _, k0, k1 in ot.spans(oq, oq if ok is None else ok, lk, 0, 0)] + [0])
    within(out.detach(), ref["out"], bounds(ref, "out", dtype, dim, reach, keys * size(vc)), "out")
    empty = torch.isinf(ref["log_sum"])
    assert torch.equal(empty, log_sum == -math.inf)
    within(log_sum[~empty], ref["log_sum"][~empty],
           (dim + 16) * E * (reach + ref["log_sum"][~empty].abs() + 1), "log_sum")
    if go is not None:
        rows = q.shape[0] * q.shape[1]
        s = max(1.0, dim * size(go) * size(vc))
        for name, grad, terms in (("gq", grads[0], keys * c * size(kc) * s),
                                  ("gk", grads[1], rows * c * size(q) * s),
                                  ("gv", grads[2], rows * size(go))):
            within(grad, ref[name], bounds(ref, name, dtype, dim, reach, terms), name)
        assert bool((grads[1][~seen] == 0).all()) and bool((grads[2][~seen] == 0).all())
        assert all(g.is_contiguous() for g in grads)
    assert out.is_contiguous()
    with torch.no_grad():
        assert torch.equal(cr.packed_attention(q, k, v, oq, ok, lk, causal=causal, scale=scale), out)
    return (out.detach(), log_sum, *grads)


def attention_inputs(gpu, tq, tk, heads, key_heads, dim, dtype, seed=0, size=1.5):
    g = rng(gpu, 7 * tq + 3 * tk + dim + heads + seed)
    return ((size * randn(g, tq, heads, dim)).to(dtype), (size * randn(g, tk, key_heads, dim)).to(dtype),
            randn(g, tk, key_heads, dim).to(dtype), randn(g, tq, heads, dim).to(dtype))


@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths", [[1], [2, 1, 3], [31, 0, 33], [64], [65, 63], [1, 128, 0, 129],
                                     [257], [700, 5, 100]])
def test_attention_of_packed_lengths(gpu, lengths, causal, dtype):
    q, k, v, go = attention_inputs(gpu, sum(lengths), sum(lengths), 4, 2, 64, dtype)
    check_attention(q, k, v, offsets_of(lengths, gpu), causal=causal, go=go)


@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("dim", [8, 16, 24, 40, 48, 56, 72, 80, 96, 104, 120, 128])
def test_attention_dimensions(gpu, dim, dtype):
    lengths = [100, 37]
    q, k, v, go = attention_inputs(gpu, 137, 137, 2, 1, dim, dtype)
    check_attention(q, k, v, offsets_of(lengths, gpu), causal=dim % 16 == 0, go=go)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads,key_heads", [(1, 1), (3, 3), (3, 1), (8, 1), (10, 2), (7, 1),
                                             (40, 1), (130, 1)])
def test_attention_grouped_heads(gpu, heads, key_heads, causal):
    q, k, v, go = attention_inputs(gpu, 90, 90, heads, key_heads, 32, torch.bfloat16)
    check_attention(q, k, v, offsets_of([50, 40], gpu), causal=causal, go=go)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lq,lk", [([1, 1, 1], [300, 1, 77]), ([5, 130, 7], [200, 10, 7]),
                                   ([0, 4], [9, 0]), ([200, 3], [64, 500]), ([1, 2], [5000, 3]),
                                   ([33], [1]), ([1], [20_001]), ([70], [3000])])
def test_attention_of_other_keys(gpu, lq, lk, causal):
    """Fewer and more keys than queries: causal rows above the first key see nothing."""
    for dtype in TYPES[1:]:
        q, k, v, go = attention_inputs(gpu, sum(lq), sum(lk), 4, 1, 64, dtype)
        check_attention(q, k, v, offsets_of(lq, gpu), offsets_of(lk, gpu), causal=causal, go=go)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new", [1, 3, 40])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_over_a_cache(gpu, new, causal, dim):
    """Slabs filled up to a length, NaN and infinities past it, a slab that is empty, a
    length past its slab, a negative one."""
    slab, lengths = 500, [1, 500, 0, 123, 64, 900, -3, 128]
    n = len(lengths)
    lk = torch.tensor(lengths, dtype=torch.int32, device=gpu)
    for dtype in TYPES[1:]:
        q, k, v, go = attention_inputs(gpu, n * new, n * slab, 8, 2, dim, dtype)
        for b, filled in enumerate(lengths):
            past = slice(b * slab + min(max(filled, 0), slab), (b + 1) * slab)
            k[past] = math.nan
            v[past] = math.inf if b % 2 else math.nan
        check_attention(q, k, v, offsets_of([new] * n, gpu), offsets_of([slab] * n, gpu), lk,
                        causal=causal, go=go)


def test_attention_over_long_caches(gpu):
    """A gigabyte of cache, so that copies of tiles wait for memory; the same twice over."""
    lengths = [30_000, 32_640, 3, 2500, 18_967, 7600, 21_404, 8160]
    slab, n = 32_640, len(lengths)
    lk = torch.tensor(lengths, dtype=torch.int32, device=gpu)
    for dtype in TYPES[1:]:
        q, k, v, _ = attention_inputs(gpu, n, n * slab, 16, 8, 128, dtype)
        args = (q, k, v, offsets_of([1] * n, gpu), offsets_of([slab] * n, gpu), lk)
        first = check_attention(*args, causal=True)[0]
        for _ in range(5):
            assert torch.equal(cr.packed_attention(*args, causal=True), first)


def test_attention_twice_over(gpu):
    """Many workgroups at work: the same values every time, gradients too."""
    q, k, v, go = attention_inputs(gpu, 9000, 9000, 8, 2, 128, torch.bfloat16)
    at = offsets_of([4000, 5000], gpu)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    first = None
    for _ in range(4):
        out = cr.packed_attention(*leaves, at, causal=True)
        got = (out.detach(), *torch.autograd.grad(out, leaves, go))
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(got, first))


def test_attention_rows_of_no_sequence(gpu):
    q, k, v, go = attention_inputs(gpu, 150, 150, 2, 2, 64, torch.float16)
    k[:9], v[140:], k[145:] = math.nan, math.nan, math.inf
    got = check_attention(q, k, v, offsets_of([60, 70], gpu, 10), go=go)
    assert all(bool((g[:10] == 0).all()) and bool((g[140:] == 0).all()) for g in got[::2])
    # no sequences at all
    got = check_attention(q, k, v, torch.zeros(1, dtype=torch.int32, device=gpu), go=go)
    assert all(bool((g == 0).all()) for g in (got[0], *got[2:]))


def test_attention_of_no_rows(gpu):
    q, k, v, go = attention_inputs(gpu, 0, 20, 2, 1, 64, torch.bfloat16)
    zero = torch.zeros(2, dtype=torch.int32, device=gpu)
    got = check_attention(q, k, v, zero, offsets_of([20], gpu), go=go)
    assert bool((got[3] == 0).all()) and bool((got[4] == 0).all())
    q, k, v, go = attention_inputs(gpu, 20, 0, 2, 1, 64, torch.bfloat16)
    got = check_attention(q, k, v, offsets_of([20], gpu), zero, go=go)
    assert bool((got[0] == 0).all()) and bool((got[2] == 0).all())


@pytest.mark.parametrize("dtype", TYPES[1:])
def test_attention_of_large_scores(gpu, dtype):
    """Scores in the hundreds, all equal scores, and a scale of 0 and below: the softmax is
    taken against the running maximum."""
    q, k, v, go = attention_inputs(gpu, 200, 200, 2, 1, 64, dtype, size=6.0)
    at = offsets_of([200], gpu)
    check_attention(q, k, v, at, causal=True, scale=1.0)
    check_attention(q, k, v, at, scale=-0.5, go=go)
    check_attention(q, k, v, at, causal=True, scale=0.0, go=go)
    check_attention(q, torch.ones_like(k), v, at, causal=True, go=go)


@pytest.mark.parametrize("exponent", [-13, 8])
def test_attention_of_small_and_large_gradients(gpu, exponent):
    """float16 output gradients near the type's ends, and of very different rows: no score
    gradient vanishes or overflows before its product.  Outputs below 2^-14 are rounded to
    2^-24 units, no other absolute term."""
    q, k, v, go = attention_inputs(gpu, 600, 600, 4, 2, 64, torch.float16)
    go = (go * 2.0 ** exponent).half()
    go[::7] = (go[::7] / 64).half()
    go[3:9] = 0
    at = offsets_of([250, 350], gpu)
    for causal in (False, True):
        ref = ot.attention(q, k, v, at, causal=causal, grad_out=go)
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = cr.packed_attention(*leaves, at, causal=causal)
        for name, got in zip(("gq", "gk", "gv"), torch.autograd.grad(out, leaves, go)):
            within(got, ref[name], 2.0 ** -11 * 1.1 * ref[name + "_slack"] + 2.0 ** -24, name)


@pytest.mark.parametrize("lq,heads,key_heads", [(64, 8, 8), (64, 256, 1), (4, 8, 8), (1, 16, 1)])
def test_attention_of_one_great_weight(gpu, lq, heads, key_heads):
    """A weight that outdoes all others leaves its value, whatever it was rounded to itself: with
    the sum of the rounded weights below it, a weight's error e counts e (v - o), so the output
    is off by its own rounding and 2 u (1 - p) 2 max|v| of the others' share 1 - p."""
    g = rng(gpu, 11)
    lk, dim, u = 300, 64, U[torch.float16]
    q, k = (torch.zeros(n, h, dim, dtype=torch.float16, device=gpu)
            for n, h in ((lq, heads), (lk, key_heads)))
    q[:, :, 0] = 0.9 + 0.1 * torch.rand(lq, heads, generator=g, device=gpu)
    k[:, :, 0] = -8.0
    k[3], k[200] = 0.0, 0.0
    k[200, :, 0] = 7.5  # in a later tile than the first reference, and less than 2^8 above it
    v = randn(g, lk, key_heads, dim).half()
    at_q, at_k = offsets_of([lq], gpu), offsets_of([lk], gpu)
    out = cr.packed_attention(q, k, v, at_q, at_k, scale=math.log(2.0))
    want = ot.attention(q, k, v, at_q, at_k, scale=math.log(2.0))["out"]
    rest = 2.0 ** (7.5 * q[:, :, :1].double())
    rest = 1 - rest / (rest + 1 + 298 * 2.0 ** (-8 * q[:, :, :1].double()))
    assert float(rest.max()) < 0.05
    within(out, want, u * want.abs() + 4 * u * rest * float(v.abs().max()) + 16 * E, "out")


@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("dim", [32, 72, 128])
def test_attention_of_one_key_has_no_score_gradient(gpu, dim, dtype):
    """A query that sees one key: its weight is 1 whatever the score, so its gradient and what it
    adds to the key's are zero, not the difference of two roundings of one sum."""
    for lq, lk, causal in (([1] * 40, None, False), ([1] * 40, None, True), ([70, 3], [1, 1], False),
                           ([70, 3], [1, 1], True), ([300], [1], False)):
        at_q, at_k = offsets_of(lq, gpu), offsets_of(lk or lq, gpu)
        q, k, v, go = attention_inputs(gpu, sum(lq), sum(lk or lq), 4, 2, dim, dtype)
        _, _, gq, gk, gv = check_attention(q, k, v, at_q, at_k, causal=causal, go=go)
        assert bool((gq == 0).all()) and bool((gk == 0).all()) and bool((gv != 0).any())
    # the first query of a causal sequence, and the first that sees a key of fewer keys
    for lq, lk, first in (([130, 65], [130, 65], [0, 130]), ([200], [140], [60])):
        at_q, at_k = offsets_of(lq, gpu), offsets_of(lk, gpu)
        q, k, v, go = attention_inputs(gpu, sum(lq), sum(lk), 4, 2, dim, dtype)
        alone = torch.zeros_like(go)
        alone[first] = go[first]
        _, _, gq, gk, gv = check_attention(q, k, v, at_q, at_k, causal=True, go=alone)
        assert bool((gq == 0).all()) and bool((gk == 0).all()) and bool((gv != 0).any())
        _, _, gq, _, _ = check_attention(q, k, v, at_q, at_k, causal=True, go=go)
        assert bool((gq[first] == 0).all()) and bool((gq != 0).any())


def test_attention_float16_query_gradients_keep_their_bits(gpu):
    """Their error is about that of rounding them once; a second rounding of the same size, of
    the score gradients, would make it sqrt(2) times as large."""
    for lengths, heads, dim, causal in (([700], 4, 72, False), ([40] * 30, 4, 64, True)):
        rows = sum(lengths)
        q, k, v, go = attention_inputs(gpu, rows, rows, heads, heads, dim, torch.float16)
        at = offsets_of(lengths, gpu)
        leaves = [t.requires_grad_(True) for t in (q, k, v)]
        out = cr.packed_attention(*leaves, at, causal=causal)
        (gq,) = torch.autograd.grad(out, leaves[:1], go)
        want = ot.attention(q.detach(), k.detach(), v.detach(), at, causal=causal,
                                   grad_out=go)["gq"]
        once = (want.half().double() - want).norm()
        assert float((gq.double() - want).norm() / once) < 1.3


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [64, 72, 128])
def test_attention_gradients_of_short_rows_keep_their_bits(gpu, dim, causal):
    """Score gradients of one tile are not rounded a second time: that would make the error
    sqrt(2) times that of rounding the gradients once, and more with what delta has of its own."""
    lengths = torch.randint(2, 8, (300,), generator=torch.Generator().manual_seed(dim)).tolist()
    rows = sum(lengths)
    q, k, v, go = attention_inputs(gpu, rows, rows, 2, 2, dim, torch.bfloat16)
    at = offsets_of(lengths, gpu)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    got = torch.autograd.grad(cr.packed_attention(*leaves, at, causal=causal), leaves[:2], go)
    ref = ot.attention(q.detach(), k.detach(), v.detach(), at, causal=causal, grad_out=go)
    for grad, name in zip(got, ("gq", "gk")):
        once = (ref[name].bfloat16().double() - ref[name]).norm()
        assert float((grad.double() - ref[name]).norm() / once) < 2 ** 0.5, name


def test_attention_does_not_see_the_masked(gpu):
    """NaN and infinity in keys and values after a query change nothing before them."""
    for dtype in TYPES[1:]:
        q, k, v, _ = attention_inputs(gpu, 300, 300, 4, 2, 64, dtype)
        at = offsets_of([300], gpu)
        clean = cr.packed_attention(q, k, v, at, causal=True)
        slack = ot.attention(q, k, v, at, causal=True)["out_slack"]
        for row, value in ((299, math.nan), (150, math.inf), (70, math.nan), (1, -math.inf)):
            k2, v2 = k.clone(), v.clone()
            k2[row:, :, 3], v2[row:, :, 5] = value, value
            got = cr.packed_attention(q, k2, v2, at, causal=True)
            within(got[:row], clean[:row].double(), 2 * U[dtype] * slack[:row], (dtype, row))
            assert not bool(torch.isfinite(got[row:]).all())


@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("lq,lk", [(300, 300), (1, 1), (3, 5000), (300, 3000)])
def test_attention_of_queries_that_are_nan(gpu, dtype, lq, lk):
    """A NaN in a query makes its output, log-sum and gradient NaN, and no other's; so does one
    in the only key of a sequence.  (Rows in tiles, few rows, and keys in splits.)"""
    q, k, v, go = attention_inputs(gpu, lq, lk, 4, 2, 64, dtype)
    oq, ok = offsets_of([lq], gpu), offsets_of([lk], gpu)
    row = lq // 2
    clean = cr.packed_attention(q, k, v, oq, ok, return_log_sum=True)
    q2 = q.clone()
    q2[row, :, 7] = math.nan
    leaves = [t.clone().requires_grad_(True) for t in (q2, k, v)]
    out, log_sum = cr.packed_attention(*leaves, oq, ok, return_log_sum=True)
    gq, gk, gv = torch.autograd.grad(out, leaves, go)
    alone = cr.packed_attention(q2, k, v, oq, ok)
    others = torch.arange(lq, device=gpu) != row
    for got, want in ((out, clean[0]), (log_sum, clean[1]), (alone, clean[0])):
        assert bool(torch.isnan(got[row]).all())
        assert torch.equal(got[others], want[others])
    assert bool(torch.isnan(gq[row]).all()) and bool(torch.isfinite(gq[others]).all())
    assert bool(torch.isnan(gk).all()) and bool(torch.isnan(gv).all())
    k2 = k.clone()
    k2[0, :, 7] = math.nan
    one = cr.packed_attention(q, k2, v, oq, ok, torch.ones(1, device=gpu, dtype=torch.int32))
    assert bool(torch.isnan(one).all())


def test_attention_layouts(gpu):
    for dtype in TYPES[1:]:
        for dim in (64, 72):
            q, k, v, go = attention_inputs(gpu, 130, 130, 4, 2, dim, dtype)
            at = offsets_of([70, 60], gpu)
            want = check_attention(q, k, v, at, causal=True, go=go)
            qkv = torch.cat((q, k, v), 1)
            views = qkv[:, :4], qkv[:, 4:6], qkv[:, 6:]
            apart = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v, go)]
            odd = []
            for t in (q, k, v, go):  # 2 bytes off: a copy is taken
                odd.append(torch.empty(t.numel() + 1, dtype=dtype, device=gpu)[1:].view(t.shape))
                odd[-1].copy_(t)
            gaps = [torch.cat((t, t[..., :3]), 2)[..., :dim] for t in (q, k, v, go)]
            for x in ((*views, go), apart, odd, gaps):
                got = check_attention(*x[:3], at, causal=True, go=x[3])
                assert all(torch.equal(a, b) for a, b in zip(want, got))
            # one gradient for all rows and heads, values broadcast over the heads
            check_attention(q, k, v[:, :1].expand(130, 2, dim), at, go=go[:1, :1].expand(130, 4, dim))


def test_attention_offsets_past_32_bits(gpu):
    """A cache whose elements pass 2^31, far rows of it."""
    rows = 70_000
    cache = torch.zeros(rows, 1, 32_768 + 64, dtype=torch.float16, device=gpu)
    q, k, v, go = attention_inputs(gpu, 3, 900, 2, 1, 64, torch.float16)
    kk, vv = cache[..., :64], cache[..., 32_768:]
    kk[rows - 900:], vv[rows - 900:] = k, v
    oq = offsets_of([3], gpu)
    far = torch.tensor([rows - 900, rows], dtype=torch.int32, device=gpu)
    near = offsets_of([900], gpu)
    check_attention(q, k, v, oq, near, causal=True, go=go)
    ref = ot.attention(q, k, v, oq, near, causal=True, grad_out=go)
    leaf = [t.detach().requires_grad_(True) for t in (q, kk, vv)]
    out = cr.packed_attention(*leaf, oq, far, causal=True)
    gq, gk, gv = torch.autograd.grad(out, leaf, go)
    for name, got in (("out", out.detach()), ("gq", gq), ("gk", gk[rows - 900:]),
                      ("gv", gv[rows - 900:])):
        within(got, ref[name], 2 * U[q.dtype] * ref[name + "_slack"] + 2.0 ** -12, name)
    assert bool((gk[:rows - 900] == 0).all()) and bool((gv[:rows - 900] == 0).all())


def test_attention_of_many_sequences(gpu):
    g = torch.Generator().manual_seed(3)
    lengths = torch.randint(0, 9, (300,), generator=g).tolist()
    q, k, v, go = attention_inputs(gpu, sum(lengths), sum(lengths), 2, 1, 32, torch.bfloat16)
    check_attention(q, k, v, offsets_of(lengths, gpu), causal=True, go=go)
    lk = torch.randint(1, 40, (300,), generator=g).tolist()
    q, k, v, go = attention_inputs(gpu, 300, sum(lk), 8, 2, 64, torch.bfloat16)
    check_attention(q, k, v, offsets_of([1] * 300, gpu), offsets_of(lk, gpu), causal=True, go=go)


def test_attention_with_offsets_out_of_range(gpu):
    """Clamped to the tensors: no read past them, and correct sequences are not touched."""
    q, k, v, _ = attention_inputs(gpu, 60, 60, 2, 1, 64, torch.float16)
    good = cr.packed_attention(q, k, v, offsets_of([20, 40], gpu))
    at = torch.tensor([0, 20, 1_000_000], dtype=torch.int32, device=gpu)
    assert torch.equal(cr.packed_attention(q, k, v, at), good)
    at = torch.tensor([-5, 20, 60], dtype=torch.int32, device=gpu)
    assert torch.equal(cr.packed_attention(q, k, v, at), good)


def test_attention_gradient_is_the_difference(gpu):
    """Along one direction, against central differences of the oracle's forward."""
    q, k, v, go = attention_inputs(gpu, 120, 120, 4, 2, 64, torch.bfloat16)
    at = offsets_of([50, 70], gpu)
    _, _, *grads = check_attention(q, k, v, at, causal=True, go=go)
    ref = ot.attention(q, k, v, at, causal=True, grad_out=go)
    g = rng(gpu, 4)
    for i, name in enumerate(("gq", "gk", "gv")):
        xs = [t.double() for t in (q, k, v)]
        d = torch.randn(xs[i].shape, generator=g, device=gpu, dtype=torch.float64)
        ends = []
        for h in (1e-4, -1e-4):
            moved = list(xs)
            moved[i] = xs[i] + h * d
            ends.append((ot.attention(*moved, at, causal=True)["out"] * go.double()).sum())
        want = float(ends[0] - ends[1]) / 2e-4
        tolerance = float((2.0 ** -8 * ref[name + "_slack"] * d.abs()).sum()) + 1e-6 * abs(want)
        assert abs(float((grads[i].double() * d).sum()) - want) <= tolerance


def test_attention_on_another_stream_and_in_a_graph(gpu):
    q, k, v, go = attention_inputs(gpu, 260, 260, 4, 2, 64, torch.bfloat16)
    at = offsets_of([100, 160], gpu)
    want = check_attention(q, k, v, at, causal=True, go=go)
    w, b = torch.ones(64, device=gpu), torch.zeros(64, device=gpu)
    f = cr.axial_frequencies((8, 24), 100.0, gpu)
    pos = torch.zeros(260, 2, dtype=torch.int32, device=gpu)

    def step(leaves):
        # outputs without their autograd nodes: a node that outlives its step would bind the
        # leaves to its stream, and a capture on another one would have to wait for it
        out = cr.packed_attention(*leaves, at, causal=True)
        turned, _ = cr.axial_rotary(cr.layer_norm(out, w, b), None, pos, f, (8, 24))
        return (turned.detach(), *torch.autograd.grad(turned, leaves, go))

    leaves, own = ([t.detach().clone().requires_grad_(True) for t in (q, k, v)] for _ in range(2))
    eager = step(leaves)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(leaves)
        assert torch.equal(cr.packed_attention(q, k, v, at, causal=True), want[0])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(eager, other))
    captured = CapturedStep(lambda: step(own))
    for seed in range(3):  # new values and other lengths in the same buffers
        new = attention_inputs(gpu, 260, 260, 4, 2, 64, torch.bfloat16, seed=seed + 1)
        with torch.no_grad():
            for one, two, t in zip(leaves, own, new):
                one.copy_(t)
                two.copy_(t)
        at.copy_(offsets_of([100 + 20 * seed, 160 - 20 * seed], gpu))
        captured.replay()
        eager = step(leaves)
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(eager, captured.output))


def test_attention_refusals(gpu):
    q, k, v, _ = attention_inputs(gpu, 8, 8, 4, 2, 64, torch.float16)
    at = offsets_of([8], gpu)
    good = dict(q=q, k=k, v=v, offsets_q=at)
    cr.packed_attention(**good)
    for bad in (dict(q=q.float()), dict(k=k.bfloat16()), dict(v=v[:7]), dict(k=k[..., :56]),
                dict(q=q[:, :3]), dict(q=q[0]), dict(offsets_q=at.long()), dict(offsets_q=at.cpu()),
                dict(offsets_q=at[:0]), dict(k=k[:7], v=v[:7]), dict(offsets_k=at[:1]),
                dict(lengths_k=at), dict(q=q[..., :60], k=k[..., :60], v=v[..., :60]),
                dict(q=q.repeat(1, 1, 3), k=k.repeat(1, 1, 3), v=v.repeat(1, 1, 3)),
                dict(q=q[:, :0])):
        with pytest.raises(RuntimeError, match="packed_attention"):
            cr.packed_attention(**{**good, **bad})
    with pytest.raises(ValueError, match="scale"):
        cr.packed_attention(**good, scale=math.inf)
    leaf = q.clone().requires_grad_(True)
    out = cr.packed_attention(leaf, k, v, at)
    with pytest.raises(RuntimeError, match="grad_out"):
        tokens.attention_backward(out.float(), q, k, v, out, out, out[..., 0].float(), at, at, None,
                                  False, 0.125)
