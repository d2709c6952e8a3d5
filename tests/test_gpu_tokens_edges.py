"""GPU parity of the patch-network operators where types, lengths and layouts end: float16's
range, infinities, tiles that a sequence just fills, rows far apart, callers that want part of
the work.

Gradients of attention are held to oracle/tokens.py::attention_gradients, which derives a bound
for every element, and as a whole to 3 u of their length: each element has three roundings of at
most u that matter (its own, its score gradients', delta's), which are independent, so that
their root mean square together is no more than u."""

from __future__ import annotations

import math

import pytest
import torch

import helpers  # noqa: F401
import cuda_rasterizer as cr
from oracle import tokens as ot

pytestmark = pytest.mark.gpu

HALVES = [torch.float16, torch.bfloat16]
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def randn(g, *shape):
    return torch.randn(shape, generator=g, device=g.device)


def offsets_of(lengths, gpu):
    return torch.tensor([0] + lengths, device=gpu).cumsum(0).to(torch.int32)


def inputs(gpu, tq, tk, heads, key_heads, dim, dtype, seed=0):
    g = torch.Generator(device=gpu).manual_seed(11 * tq + tk + dim + seed)
    return ((1.5 * randn(g, tq, heads, dim)).to(dtype), (1.5 * randn(g, tk, key_heads, dim)).to(dtype),
            randn(g, tk, key_heads, dim).to(dtype), randn(g, tq, heads, dim).to(dtype))


def gradients(q, k, v, go, oq, ok=None, lk=None, causal=False, scale=None):
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = cr.packed_attention(*leaves, oq, ok, lk, causal=causal, scale=scale)
    return out.detach(), torch.autograd.grad(out, leaves, go)


def check_gradients(q, k, v, go, oq, ok=None, lk=None, causal=False, scale=None, names="qkv"):
    """Against the oracle, element by element and as a whole; gradients of zeros would fail."""
    ref = ot.attention_gradients(q, k, v, oq, go, ok, lk, causal, scale)
    _, grads = gradients(q, k, v, go, oq, ok, lk, causal, scale)
    for name, grad in zip("qkv", grads):
        if name not in names:
            continue
        want, bound = ref["g" + name], ref[f"g{name}_bound"]
        assert bool(torch.isfinite(grad).all()), name
        off = (grad.double() - want).abs()
        assert float((off - bound).max()) <= 0.0, (name, float(off.max()), float((off - bound).max()))
        length = float(want.norm())
        assert float(off.norm()) <= 3 * U[q.dtype] * length and length > 0.0, (
            name, float(off.norm()) / length)
    return grads


# --------------------------------------------------------------- float16's range
def ranged(gpu, kind, dim):
    """float16 inputs (q, k, v, go, lengths) whose score gradients, or what leads to them, lie near
    the ends of float16, though the gradients do not."""
    g = torch.Generator(device=gpu).manual_seed(dim)
    lengths = [2] * 20 if kind == "two equal weights" else [64, 250, 350]
    n = sum(lengths)
    q, k, v, go = (randn(g, n, 2, dim) for _ in range(4))
    sign = torch.sign(randn(g, n, 2, 1))
    if kind == "two equal weights":  # the difference to the output is as large as the values
        q, k, go = 0.01 * q, 0.25 * k, 1.9 + 0.0 * go
        v = 34.0 * torch.tensor([1.0, -1.0], device=gpu).repeat(n // 2)[:, None, None] + 0.0 * v
    elif kind == "values equal along a row":
        q, k, v, go = 0.3 * q, 0.3 * k, 100.0 * sign + 0.0 * v, 1e-3 * torch.sign(go[..., :1]) + 0.0 * go
    elif kind == "large values":
        q, k, v = 0.3 * q, 0.3 * k, 1000.0 * v
    elif kind == "largest values":
        q, k, v, go = 0.1 * q, 0.1 * k, 30000.0 * sign + 0.0 * v, 0.5 * go
    elif kind == "small values":
        q, k, v = 3.0 * q, 3.0 * k, v / 1024.0
    else:  # "first queries large"
        go = go * torch.where(torch.arange(n, device=gpu) % 64 < 40, 2.0 ** 10, 2.0 ** -7)[:, None, None]
    return *(t.half() for t in (q, k, v, go)), lengths


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [64, 72, 128])
@pytest.mark.parametrize("kind", ["two equal weights", "values equal along a row", "large values",
                                  "largest values", "small values", "first queries large"])
def test_attention_query_gradients_stay_in_float16(gpu, kind, dim, causal):
    q, k, v, go, lengths = ranged(gpu, kind, dim)
    check_gradients(q, k, v, go, offsets_of(lengths, gpu), causal=causal, names="q")


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [64, 72, 128])
@pytest.mark.parametrize("kind", ["two equal weights", "values equal along a row", "large values",
                                  "largest values", "small values", "first queries large"])
def test_attention_key_gradients_stay_in_float16(gpu, kind, dim, causal):
    """Under a causal mask a key's gradient keeps its bits beside rows, however large, that do not
    see it."""
    q, k, v, go, lengths = ranged(gpu, kind, dim)
    check_gradients(q, k, v, go, offsets_of(lengths, gpu), causal=causal, names="kv")


# ------------------------------------------------------------- infinities and NaN
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("dim", [64, 72, 128])
@pytest.mark.parametrize("lq,lk", [(300, 300), (40, 40), (3, 5000), (300, 3000)])
def test_attention_gives_infinities_that_a_query_sees(gpu, lq, lk, dim, dtype):
    """In tiles that all rows see and at a causal edge alike, in rows, few rows and splits: an
    infinity in a value comes out as one, infinities of both signs and NaN as NaN, in the columns
    that hold them and in the rows that see them."""
    q, k, v, _ = inputs(gpu, lq, lk, 4, 2, dim, dtype)
    q, k = q / 5, k / 5  # no weight is rounded to 0
    oq, ok = offsets_of([lq], gpu), offsets_of([lk], gpu)
    first, second = lk - lq // 2 - 1, lk - lq // 4 - 1
    w = v.clone()
    w[first, :, 3], w[second, :, 3] = math.inf, -math.inf
    w[first, :, 20] = -math.inf
    w[second, :, 41] = math.nan
    w[second, 1, 50] = math.inf  # one of two key heads
    for causal in (False, True):
        ref = ot.attention(q, k, v, oq, ok, causal=causal)
        got = cr.packed_attention(q, k, w, oq, ok, causal=causal)
        at = torch.arange(lq, device=gpu) + (lk - lq if causal else lk)
        one, two = (at >= first)[:, None], (at >= second)[:, None]
        want = ref["out"].clone()
        want[..., 3] = torch.where(two, math.nan, torch.where(one, math.inf, want[..., 3]))
        want[..., 20] = torch.where(one, -math.inf, want[..., 20])
        want[..., 41] = torch.where(two, math.nan, want[..., 41])
        want[:, 2:, 50] = torch.where(two, math.inf, want[:, 2:, 50])
        got = got.double()
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(torch.isinf(got) * got.sign(), torch.isinf(want) * want.sign())
        there = torch.isfinite(want)
        off = (got - want)[there].abs() - 1.1 * U[dtype] * ref["out_slack"][there]
        assert float(off.max()) <= 2.0 ** -24


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lq,lk", [([30, 200], [30, 200]), ([2, 3], [700, 5000]), ([40, 300], [600, 3000]),
                                   ([30, 200], [30, 150])])
def test_attention_of_keys_that_all_score_minus_infinity(gpu, lq, lk, causal, dtype):
    """They are seen: weights of 0 / 0 give NaN, with its gradients, where a query that sees no key
    gives 0.  The other sequence does not change."""
    q, k, v, go = inputs(gpu, sum(lq), sum(lk), 4, 2, 64, dtype)
    q[lq[0]:, :, 0] = 1.0
    k[lk[0]:, :, 0] = -math.inf
    oq, ok = offsets_of(lq, gpu), offsets_of(lk, gpu)
    sees = torch.arange(lq[1], device=gpu) + lk[1] - lq[1] >= 0 if causal else torch.ones(
        lq[1], device=gpu, dtype=torch.bool)
    with torch.no_grad():
        alone = cr.packed_attention(q, k, v, oq, ok, causal=causal)
    out, log_sum = cr.packed_attention(q, k, v, oq, ok, causal=causal, return_log_sum=True)
    first = gradients(q[:lq[0]], k[:lk[0]], v[:lk[0]], go[:lq[0]], oq[:2], ok[:2], causal=causal)
    whole = gradients(q, k, v, go, oq, ok, causal=causal)
    for got in (alone, out, whole[0], whole[1][0]):
        second = got[lq[0]:]
        assert bool(torch.isnan(second[sees]).all()) and bool((second[~sees] == 0).all())
    assert bool((log_sum[lq[0]:] == -math.inf).all())
    for grad, one in zip(whole[1], first[1]):
        assert bool(torch.isfinite(grad[:one.shape[0]]).all())
        assert float((grad[:one.shape[0]] - one).float().norm()) <= 4 * U[dtype] * float(one.float().norm())
    for grad in whole[1][1:]:
        assert bool(torch.isnan(grad[lk[0]:]).all())


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("dim", [64, 72, 128])
@pytest.mark.parametrize("row,value", [(40, math.inf), (100, -math.inf), (299, math.inf), (60, math.nan)])
def test_attention_gradients_of_one_infinite_output_gradient(gpu, row, value, dim, dtype):
    """It reaches the value gradients of the keys that its query sees, in its own column only, and
    their key gradients; in tiles that see the query whole and at a causal edge."""
    q, k, v, go = inputs(gpu, 300, 300, 4, 2, dim, dtype)
    q, k = q / 5, k / 5
    at = offsets_of([300], gpu)
    bad, none = go.clone(), go.clone()
    bad[row, 1, 7], none[row, 1, 7] = value, 0.0
    for causal in (False, True):
        ref = ot.attention_gradients(q, k, v, at, none, causal=causal)
        _, (gq, gk, gv) = gradients(q, k, v, bad, at, causal=causal)
        seen = torch.arange(300, device=gpu) <= (row if causal else 299)
        want, bound = ref["gv"].clone(), ref["gv_bound"]
        want[seen, 0, 7] = value
        assert torch.equal(torch.isfinite(gv), torch.isfinite(want))
        assert bool(torch.isnan(gv[seen, 0, 7]).all()) or bool((gv[seen, 0, 7] == value).all())
        assert (value != value) == bool(torch.isnan(gv).any())
        there = torch.isfinite(want)
        assert float(((gv.double() - want)[there].abs() - bound[there]).max()) <= 0.0
        # keys that the query does not see, and the other key head
        assert not bool(torch.isfinite(gk[seen, 0]).any())
        for got, name, rows in ((gk[~seen, 0], "gk", (~seen, 0)), (gk[:, 1], "gk", (slice(None), 1))):
            if got.numel():
                off = (got.double() - ref[name][rows]).abs() - ref[name + "_bound"][rows]
                assert float(off.max()) <= 0.0
        others = torch.ones(300, 4, device=gpu, dtype=torch.bool)
        others[row, 1] = False
        assert not bool(torch.isfinite(gq[row, 1]).any())
        off = (gq.double() - ref["gq"]).abs() - ref["gq_bound"]
        assert float(off[others].max()) <= 0.0


# ------------------------------------------------------ tiles that are just filled
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [64, 72, 128])
@pytest.mark.parametrize("lq,lk", [(64, 64), (63, 64), (64, 60), (7, 64)])
def test_attention_gradients_of_one_full_tile_keep_their_bits(gpu, lq, lk, dim, causal):
    """Score gradients of up to 64 keys and queries are not rounded a second time, the full tile's
    among them: that would make the error sqrt(2) times that of rounding the gradients once."""
    n = 40
    q, k, v, go = inputs(gpu, n * lq, n * lk, 2, 2, dim, torch.bfloat16)
    oq, ok = offsets_of([lq] * n, gpu), offsets_of([lk] * n, gpu)
    ref = ot.attention_gradients(q, k, v, oq, go, ok, causal=causal)
    _, grads = gradients(q, k, v, go, oq, ok, causal=causal)
    for grad, name in zip(grads[:2], ("gq", "gk")):
        once = (ref[name].bfloat16().double() - ref[name]).norm()
        assert float((grad.double() - ref[name]).norm() / once) < 1.3, name


# ------------------------------------------------------------ how callers call them
def operators(gpu):
    """(name, function of its differentiable inputs, these inputs) of each operator."""
    g = torch.Generator(device=gpu).manual_seed(9)
    x, w, b = randn(g, 20, 64), randn(g, 64), randn(g, 64)
    pos = torch.arange(40, device=gpu, dtype=torch.int32).view(20, 2)
    f, at = cr.axial_frequencies((8, 24), 100.0, gpu), offsets_of([12, 8], gpu)
    q, k, v = (randn(g, 20, h, 64) for h in (4, 2, 2))
    return [("layer_norm", lambda x, w, b: cr.layer_norm(x, w, b), (x, w, b)),
            ("axial_rotary", lambda q, k: cr.axial_rotary(q, k, pos, f, (8, 24)), (q, k)),
            ("packed_attention", lambda q, k, v: cr.packed_attention(q, k, v, at, causal=True),
             tuple(t.half() for t in (q, k, v)))]


def test_forward_mode_tangents_are_refused(gpu):
    """In every differentiable input, with and without gradients enabled: no output silently
    without its tangent."""
    with torch.autograd.forward_ad.dual_level():
        for name, run, args in operators(gpu):
            run(*args)
            for i, t in enumerate(args):
                dual = torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))
                for grad in (True, False):
                    with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match=name):
                        run(*args[:i], dual, *args[i + 1:])


def test_traced_calls_compute(gpu):
    """A traced function runs the operator on its new inputs, with gradients enabled or not; it
    does not return what memory holds."""
    for name, run, args in operators(gpu):
        new = tuple(t.flip(0).contiguous() for t in args)
        want = run(*new)
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                traced = torch.jit.trace(run, args, check_trace=False)
            for _ in range(2):
                spoil = [torch.full_like(t, math.nan) for t in args for _ in range(4)]
                del spoil  # an output that is only allocated would hold these
                got = traced(*new)
                for a, b in zip(got if isinstance(got, tuple) else (got,),
                                want if isinstance(want, tuple) else (want,)):
                    assert torch.equal(a, b), (name, grad)


# --------------------------------------------------------------------- layouts
@pytest.mark.parametrize("dim", [64, 72, 88, 128])
def test_attention_of_rows_megabytes_apart(gpu, dim):
    """Values whose rows lie 12 MB apart, so that a tile of keys spans more than 2^31 bytes: what
    lies between them, also at that distance, is not read."""
    stride, rows = 6_000_000, 200
    q, k, v, go = inputs(gpu, rows, rows, 4, 1, dim, torch.bfloat16)
    wide = torch.full((rows * stride,), math.nan, dtype=torch.bfloat16, device=gpu)
    far = wide.as_strided((rows, 1, dim), (stride, dim, 1))
    far.copy_(v)
    at = offsets_of([rows], gpu)
    for causal in (False, True):
        want = gradients(q, k, v, go, at, causal=causal)
        got = gradients(q, k, far, go, at, causal=causal)
        for a, b in zip((want[0], *want[1]), (got[0], *got[1])):
            assert torch.equal(a, b)


# --------------------------------------------------------- part of the gradients
@pytest.mark.parametrize("lq,lk", [([30, 200], [30, 200]), ([3], [20_000]), ([40], [0])])
def test_attention_gradients_that_are_asked_for(gpu, lq, lk):
    """The same values as all together, for every choice of inputs that have one; keys and values
    without a gradient get no memory for it."""
    q, k, v, go = inputs(gpu, sum(lq), sum(lk), 8, 8, 128, torch.bfloat16)
    oq, ok = offsets_of(lq, gpu), offsets_of(lk, gpu)
    whole = gradients(q, k, v, go, oq, ok, causal=True)[1]
    for choice in range(1, 8):
        leaves = [t.clone().requires_grad_(bool(choice >> i & 1)) for i, t in enumerate((q, k, v))]
        out = cr.packed_attention(*leaves, oq, ok, causal=True)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        got = torch.autograd.grad(out, [t for t in leaves if t.requires_grad], go)
        peak = torch.cuda.max_memory_allocated() - before
        for a, b in zip(got, [w for i, w in enumerate(whole) if choice >> i & 1]):
            assert torch.equal(a, b)
        if choice == 1 and sum(lk) > 10_000:
            assert peak < k.numel() * k.element_size()


# ---------------------------------------------- gradients within their derived bounds
@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dim", [40, 64, 72, 88, 96, 128])
@pytest.mark.parametrize("lq,lk", [([700, 5, 100], None), ([257], None), ([128, 129, 64, 65], None),
                                   ([40, 256, 1], [300, 513, 256])])
def test_attention_gradients_within_bounds(gpu, lq, lk, dim, causal, dtype):
    """Blocks of 128 and 256 keys, their remainders and their places among the values."""
    q, k, v, go = inputs(gpu, sum(lq), sum(lk or lq), 4, 2, dim, dtype)
    check_gradients(q, k, v, go, offsets_of(lq, gpu), offsets_of(lk or lq, gpu), causal=causal)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("lq,lk,heads", [([1], [20_001], 4), ([70], [3000], 4), ([1500], [700], 4),
                                         ([3000, 100], [300, 300], 8), ([700], [5000], 2)])
@pytest.mark.parametrize("dim", [64, 72, 96, 128])
def test_attention_gradients_in_splits_within_bounds(gpu, lq, lk, heads, dim, dtype):
    """Few queries over many keys and many queries over few, whose sums are split."""
    q, k, v, go = inputs(gpu, sum(lq), sum(lk), heads, 1, dim, dtype)
    check_gradients(q, k, v, go, offsets_of(lq, gpu), offsets_of(lk, gpu))


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("slab,longs,sequences", [(700, 290, 300), (6400, 5, 127)])
def test_attention_over_more_caches_than_workgroups(gpu, slab, longs, sequences, dtype):
    """More parts of caches than the launch has workgroups, so that one takes several in turn: 2400
    whole caches, and 1056 parts of which some are halves."""
    g = torch.Generator().manual_seed(slab)
    few = torch.randint(1, 64, (sequences,), generator=g)
    many = torch.randint(slab - 100, slab + 1, (sequences,), generator=g)
    lengths = torch.where(torch.randperm(sequences, generator=g) < longs, many, few)
    q, k, v, _ = inputs(gpu, sequences, sequences * slab, 8, 8, 64, dtype)
    oq, ok = offsets_of([1] * sequences, gpu), offsets_of([slab] * sequences, gpu)
    lk = lengths.to(device=gpu, dtype=torch.int32)
    for causal in (False, True):
        out, log_sum = cr.packed_attention(q, k, v, oq, ok, lk, causal=causal, return_log_sum=True)
        ref = ot.attention(q, k, v, oq, ok, lk, causal)
        off = (out.double() - ref["out"]).abs()
        least = 2.0 ** -25 * slab * float(v.abs().max()) if dtype == torch.float16 else 0.0
        assert float((off - 1.1 * U[dtype] * ref["out_slack"]).max()) <= least
        assert float(off.norm()) <= 3 * U[dtype] * float(ref["out"].norm())
        # scores off by (dim + 16) 2^-24 of their largest, and the sum's logarithm rounded
        reach = 64 ** -0.5 * float(q.double().norm(dim=2).max() * k.double().norm(dim=2).max())
        bound = (64 + 16) * 2.0 ** -24 * (reach + ref["log_sum"].abs() + 1)
        assert float(((log_sum - ref["log_sum"]).abs() - bound).max()) <= 0.0


# -------------------------------------------------------------------- positions
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("ptype,sizes", [(torch.int64, (10 ** 12, 10 ** 15, 10 ** 17, 17 * 10 ** 17)),
                                         (torch.float32, (1e12, 1e16, 1e19, 1e22))])
def test_axial_rotary_of_times_in_nanoseconds(gpu, ptype, sizes, interleaved):
    """Positions up to the types' large numbers turn pairs by the angle that float64 holds, to a
    float's accuracy, and keep their length."""
    g = torch.Generator(device=gpu).manual_seed(12)
    rows = 64
    q = randn(g, rows, 2, 32)
    scale = torch.tensor(sizes, dtype=torch.float64).repeat(rows // 4)[:, None]
    part = 1 + torch.rand(rows, 2, generator=torch.Generator().manual_seed(1), dtype=torch.float64)
    positions = (scale * part * torch.tensor([1.0, -1.0])).to(ptype)
    f = cr.axial_frequencies((7, 9), 100.0, "cpu")
    got = cr.axial_rotary(q, None, positions.to(gpu), f.to(gpu), (7, 9), interleaved=interleaved)[0]
    want = ot.rotary(q.cpu(), positions, f, (7, 9), interleaved)
    lo, hi = (slice(0, 32, 2), slice(1, 32, 2)) if interleaved else (slice(0, 16), slice(16, 32))
    length = torch.hypot(q.cpu().double()[..., lo], q.cpu().double()[..., hi])
    for part in (lo, hi):
        off = (got.cpu().double()[..., part] - want[..., part]).abs()
        assert float((off - 9 * 2.0 ** -24 * length).max()) <= 0.0


# --------------------------------------------------------------------- refusals
def test_layer_norm_refuses_channels_past_its_numbers(gpu):
    """More channels than 32-bit numbers hold, which would be taken for their lowest bits."""
    x = torch.zeros(1, 1, device=gpu)
    for channels in (2 ** 30 + 1, 2 ** 31 + 8, 2 ** 32 + 8):
        with pytest.raises(RuntimeError, match="channels"):
            cr.layer_norm(x.expand(1, channels))
