"""Operators of a network that predicts Gaussians from posed images.

Such a network cuts its images into patches, one token each (with 16x16 patches
the rasterizer's own tiles: 2500 for an 800x800 view, 8160 for 1920x1080), runs
blocks of normalisation, attention and matrix products over a scene's tokens, and
ends in Gaussians that render() draws and sends gradients back through.  Beside
the matrix products, its blocks need

- layer_norm(x, weight, bias): normalisation over the last dimension;
- axial_rotary(q, k, positions, frequencies, sections): rotary positions of up to
  four axes (view or time, row, column); axial_frequencies(sections) makes the
  usual frequencies;
- packed_attention(q, k, v, offsets_q, ...): softmax attention over scenes of any
  sizes packed one after another, grouped heads, causal (a stream of views) or
  not, or new queries over a cache of earlier keys and values.

All run on the library's gfx950 kernels on the current HIP stream, without host
synchronisation, and are differentiable once, backwards (packed_attention in q, k and
v; axial_rotary in q and k; layer_norm in all three); forward-mode tangents are refused.  Inputs are float32, float16 or
bfloat16 (packed_attention: float16 or bfloat16); sums and statistics are held in
float32 and each output is rounded once.  Nothing here has a counterpart in the
reference.
"""

from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd.forward_ad import unpack_dual
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import GsAttention, GsRotaryTensor

_TYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_POSITIONS = {torch.int32: 0, torch.int64: 1, torch.float32: 2}
MAX_CHANNELS = 1 << 30
MAX_AXES = 4
MAX_HEAD_DIM = 128
_MAX_STRIDE = 1 << 23  # elements from a row to the next


def _check(what: str, name: str, t, dims: int | None = None, types=_TYPES, device=None):
    if not isinstance(t, torch.Tensor):
        raise RuntimeError(f"{what}: {name} must be a torch.Tensor, got {type(t).__name__}")
    if t.device.type != "cuda":
        raise RuntimeError(f"{what} runs on the GPU only; {name} is on {t.device} "
                           "(there is no CPU fallback)")
    if device is not None and t.device != device:
        raise RuntimeError(f"{what}: {name} is on {t.device}, expected {device}")
    if t.dtype not in types:
        raise RuntimeError(f"{what}: {name} must be one of "
                           f"{', '.join(str(d) for d in types)}, got {t.dtype}")
    if dims is not None and t.dim() != dims:
        raise RuntimeError(f"{what}: {name} must have {dims} dimensions, got {tuple(t.shape)}")


def _ptr(t):
    return None if t is None else t.data_ptr()


def _workspace(query, *args, device):
    size = ctypes.c_size_t(0)
    _lib.check(query(*args, ctypes.byref(size)), query.__name__)
    if size.value == 0:
        return None, 0
    return torch.empty(size.value, dtype=torch.uint8, device=device), size.value


def _differentiable(what: str, *tensors) -> bool:
    """Whether the call has to be an autograd function's: where gradients are recorded, and where
    torch.jit.trace records, which would find only the allocation of the outputs otherwise.  A
    tangent of forward-mode differentiation is refused: the operators have no such rule, and
    their outputs would drop it."""
    grad, found = torch.is_grad_enabled(), torch.jit.is_tracing()
    for t in tensors:
        if isinstance(t, torch.Tensor):
            found = found or (grad and t.requires_grad)
            if unpack_dual(t).tangent is not None:
                raise NotImplementedError(f"{what} has no forward-mode derivative")
    return found


# ------------------------------------------------------------------ layer norm
def _rows_of(t: torch.Tensor) -> torch.Tensor:
    """t as (rows, channels) with contiguous channels, a view where there is one."""
    t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def layer_norm_forward(x, weight=None, bias=None, eps: float = 1e-5, with_stats: bool = True):
    """(y, stats): the normalised rows in x's shape, contiguous, and the float32
    (rows, 2) means and reciprocal deviations that layer_norm_backward reads (None
    without with_stats)."""
    _check("layer_norm", "x", x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise RuntimeError(f"layer_norm: x needs channels in its last dimension, got {tuple(x.shape)}")
    channels = x.shape[-1]
    if channels > MAX_CHANNELS:
        raise RuntimeError(f"layer_norm: at most {MAX_CHANNELS} channels are supported, got {channels}")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        _check("layer_norm", name, t, 1, device=x.device)
        if t.shape[0] != channels:
            raise RuntimeError(f"layer_norm: {name} must have {channels} elements, got {t.shape[0]}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise RuntimeError(f"layer_norm: weight is {weight.dtype} and bias {bias.dtype}; "
                           "they must have one type")
    if not eps >= 0.0:
        raise ValueError(f"layer_norm: eps must be >= 0, got {eps}")
    rows = _rows_of(x)
    n = rows.shape[0]
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    given = weight if weight is not None else bias
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    stats = torch.empty((n, 2), dtype=torch.float32, device=x.device) if with_stats else None
    with _lib.on_device(x.device):
        ev = _lib.timer.record("layer_norm_forward", x.device)
        _lib.check(_lib.load().gs_layer_norm_forward(
            rows.data_ptr(), rows.stride(0), _ptr(weight), _ptr(bias), n, channels, eps,
            _TYPES[x.dtype], _TYPES[x.dtype if given is None else given.dtype], y.data_ptr(),
            _ptr(stats), _lib.stream_of(x.device)), "layer_norm_forward")
        _lib.timer.stop(ev, x.device)
    return y, stats


def layer_norm_backward(grad_y, x, weight, stats, needs=(True, True, True), weight_dtype=None):
    """(grad_x, grad_weight, grad_bias) of layer_norm_forward, None where needs is
    False; the sums over the rows are in weight's type (or weight_dtype)."""
    _check("layer_norm", "grad_y", grad_y, device=x.device)
    if grad_y.dtype != x.dtype or grad_y.shape != x.shape:
        raise RuntimeError(f"layer_norm: grad_y must be {x.dtype} {tuple(x.shape)}, got "
                           f"{grad_y.dtype} {tuple(grad_y.shape)}")
    rows, grads = _rows_of(x), _rows_of(grad_y)
    n, channels = rows.shape
    weight = None if weight is None else weight.contiguous()
    dtype = weight_dtype or (x.dtype if weight is None else weight.dtype)
    dev = x.device
    gx = torch.empty(x.shape, dtype=x.dtype, device=dev) if needs[0] else None
    gw, gb = (torch.empty(channels, dtype=dtype, device=dev) if need else None
              for need in needs[1:])
    lib = _lib.load()
    with _lib.on_device(dev):
        ws, size = (_workspace(lib.gs_layer_norm_backward_workspace_size, n, channels, device=dev)
                    if needs[1] or needs[2] else (None, 0))
        ev = _lib.timer.record("layer_norm_backward", dev)
        _lib.check(lib.gs_layer_norm_backward(
            grads.data_ptr(), grads.stride(0), rows.data_ptr(), rows.stride(0), _ptr(weight),
            stats.data_ptr(), n, channels, _TYPES[x.dtype], _TYPES[dtype], _ptr(gx), _ptr(gw),
            _ptr(gb), _ptr(ws), size, _lib.stream_of(dev)), "layer_norm_backward")
        _lib.timer.stop(ev, dev)
    return gx, gw, gb


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, stats = layer_norm_forward(x, weight, bias, eps)
        ctx.save_for_backward(x, weight, stats)
        ctx.dtype = bias.dtype if weight is None and bias is not None else None
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y):
        x, weight, stats = ctx.saved_tensors
        return (*layer_norm_backward(grad_y, x, weight, stats, ctx.needs_input_grad[:3],
                                     ctx.dtype), None)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None,
               bias: torch.Tensor | None = None, eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over x's last dimension, in x's
    type; weight and bias may have another (float32 weights for bfloat16 x)."""
    if _differentiable("layer_norm", x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, eps)
    return layer_norm_forward(x, weight, bias, eps, with_stats=False)[0]


# ---------------------------------------------------------------------- rotary
def axial_frequencies(sections, base: float = 100.0, device="cuda") -> torch.Tensor:
    """Frequencies for axial_rotary: base ** (-i / n) for the n pairs of each axis."""
    return torch.tensor([base ** (-i / n) for n in sections for i in range(n)],
                        dtype=torch.float32, device=device)


def _rotate(tensors, positions, frequencies, sections, interleaved, inverse):
    first = tensors[0]
    dev = first.device
    tokens, _, dim = first.shape
    out = [torch.empty(t.shape, dtype=t.dtype, device=dev) for t in tensors]
    tensors = [t if t.stride(2) == 1 or dim == 1 else t.contiguous() for t in tensors]
    specs = (GsRotaryTensor * len(out))(*(
        GsRotaryTensor(t.data_ptr(), y.data_ptr(), t.stride(0), t.stride(1), y.stride(0),
                       y.stride(1), t.shape[1]) for t, y in zip(tensors, out)))
    with _lib.on_device(dev):
        ev = _lib.timer.record("axial_rotary", dev)
        _lib.check(_lib.load().gs_axial_rotary(
            specs, len(out), positions.data_ptr(), positions.stride(0),
            _POSITIONS[positions.dtype], frequencies.data_ptr(),
            (ctypes.c_int32 * len(sections))(*sections), len(sections), tokens, dim,
            _TYPES[first.dtype], interleaved, inverse, _lib.stream_of(dev)), "axial_rotary")
        _lib.timer.stop(ev, dev)
    return out


class _AxialRotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, frequencies, sections, interleaved):
        ctx.save_for_backward(positions, frequencies)
        ctx.how = (sections, interleaved)
        ctx.set_materialize_grads(False)
        out = _rotate([t for t in (q, k) if t is not None], positions, frequencies, sections,
                      interleaved, False)
        return out[0], out[1] if k is not None else None

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_q, grad_k):
        grads = [grad_q, grad_k]
        given = [i for i in (0, 1) if grads[i] is not None and ctx.needs_input_grad[i]]
        if given:
            turned = _rotate([grads[i] for i in given], *ctx.saved_tensors, *ctx.how, True)
            for i, t in zip(given, turned):
                grads[i] = t
        return grads[0], grads[1], None, None, None, None


def axial_rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor,
                 frequencies: torch.Tensor, sections, interleaved: bool = False):
    """(q', k'): the (tokens, heads, dim) queries and keys with every head's pairs
    turned by the token's positions, contiguous; k may be None.

    positions is (tokens, axes), int32, int64 or float32; sections says how many
    pairs go to each axis, in order, and frequencies (float32) has one entry a
    pair.  With P pairs in all, pair p is elements (p, p + P) of a head, or
    (2 p, 2 p + 1) when interleaved; elements from 2 P on stay as they are.  Angles
    are products in float64, off by 2^-53 of themselves, and are reduced there, so
    large positions keep their accuracy.  No gradient
    goes to positions or frequencies."""
    _check("axial_rotary", "q", q, 3)
    dev = q.device
    if k is not None:
        _check("axial_rotary", "k", k, 3, (q.dtype,), dev)
        if k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2]:
            raise RuntimeError(f"axial_rotary: q {tuple(q.shape)} and k {tuple(k.shape)} must "
                               "have the same tokens and dimension")
    sections = tuple(int(n) for n in sections)
    if not 1 <= len(sections) <= MAX_AXES or min(sections) < 0:
        raise RuntimeError(f"axial_rotary: 1 to {MAX_AXES} sections of pairs are supported, got "
                           f"{sections}")
    pairs = sum(sections)
    if 2 * pairs > q.shape[2]:
        raise RuntimeError(f"axial_rotary: {pairs} pairs do not fit in heads of {q.shape[2]}")
    _check("axial_rotary", "positions", positions, 2, _POSITIONS, dev)
    if tuple(positions.shape) != (q.shape[0], len(sections)):
        raise RuntimeError(f"axial_rotary: positions must be {(q.shape[0], len(sections))}, got "
                           f"{tuple(positions.shape)}")
    _check("axial_rotary", "frequencies", frequencies, 1, (torch.float32,), dev)
    if frequencies.shape[0] != pairs:
        raise RuntimeError(f"axial_rotary: frequencies must have {pairs} entries, got "
                           f"{frequencies.shape[0]}")
    positions = positions if positions.stride(1) == 1 else positions.contiguous()
    frequencies = frequencies.contiguous()
    if _differentiable("axial_rotary", q, k):
        return _AxialRotary.apply(q, k, positions, frequencies, sections, bool(interleaved))
    out = _rotate([t for t in (q, k) if t is not None], positions, frequencies, sections,
                  bool(interleaved), False)
    return out[0], out[1] if k is not None else None


# ------------------------------------------------------------------- attention
def _laid_out(t: torch.Tensor) -> torch.Tensor:
    """t where the kernels can read its rows in 16-byte pieces, else a contiguous copy."""
    s = t.stride()
    if (s[2] == 1 and s[0] % 8 == 0 and s[1] % 8 == 0 and t.shape[2] <= s[0] <= _MAX_STRIDE
            and t.data_ptr() % 16 == 0):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _problem(q, k, v, offsets_q, offsets_k, lengths_k, causal, scale):
    return GsAttention(q.shape[0], k.shape[0], q.stride(0), q.stride(1), k.stride(0), k.stride(1),
                       v.stride(0), v.stride(1), offsets_q.data_ptr(), offsets_k.data_ptr(),
                       _ptr(lengths_k), offsets_q.shape[0] - 1, q.shape[1], k.shape[1], q.shape[2],
                       _TYPES[q.dtype], causal, scale)


def attention_forward(q, k, v, offsets_q, offsets_k, lengths_k, causal: bool, scale: float,
                      with_log_sum: bool = True, with_rest: bool = True):
    """(out, out_rest, log_sum) of checked inputs (see packed_attention).  out_rest is
    what rounding took from out; attention_backward reads it and log_sum.  None for
    what is not asked for."""
    q, k, v = _laid_out(q), _laid_out(k), _laid_out(v)
    dev = q.device
    out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    rest = torch.empty(q.shape, dtype=q.dtype, device=dev) if with_rest else None
    log_sum = (torch.empty(q.shape[:2], dtype=torch.float32, device=dev) if with_log_sum else None)
    a = _problem(q, k, v, offsets_q, offsets_k, lengths_k, causal, scale)
    lib = _lib.load()
    with _lib.on_device(dev):
        ws, size = _workspace(lib.gs_attention_forward_workspace_size, ctypes.byref(a), device=dev)
        ev = _lib.timer.record("attention_forward", dev)
        _lib.check(lib.gs_attention_forward(
            ctypes.byref(a), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _ptr(rest),
            _ptr(log_sum), _ptr(ws), size, _lib.stream_of(dev)), "attention_forward")
        _lib.timer.stop(ev, dev)
    return out, rest, log_sum


def attention_backward(grad_out, q, k, v, out, out_rest, log_sum, offsets_q, offsets_k, lengths_k,
                       causal: bool, scale: float, needs=(True, True, True)):
    """(grad_q, grad_k, grad_v), contiguous, of attention_forward's out, None where needs is
    False; those of k and v are computed together."""
    _check("packed_attention", "grad_out", grad_out, 3, (q.dtype,), q.device)
    if grad_out.shape != q.shape:
        raise RuntimeError(f"packed_attention: grad_out must be {tuple(q.shape)}, got "
                           f"{tuple(grad_out.shape)}")
    q, k, v, go = _laid_out(q), _laid_out(k), _laid_out(v), _laid_out(grad_out)
    dev = q.device
    wanted = needs[0], needs[1] or needs[2], needs[1] or needs[2]
    gq, gk, gv = (torch.empty(t.shape, dtype=t.dtype, device=dev) if want else None
                  for t, want in zip((q, k, v), wanted))
    a = _problem(q, k, v, offsets_q, offsets_k, lengths_k, causal, scale)
    lib = _lib.load()
    with _lib.on_device(dev):
        ws, size = _workspace(lib.gs_attention_backward_workspace_size, ctypes.byref(a), device=dev)
        ev = _lib.timer.record("attention_backward", dev)
        _lib.check(lib.gs_attention_backward(
            ctypes.byref(a), q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
            out_rest.data_ptr(), log_sum.data_ptr(), go.data_ptr(), go.stride(0), go.stride(1),
            _ptr(gq), _ptr(gk), _ptr(gv), _ptr(ws), size, _lib.stream_of(dev)),
            "attention_backward")
        _lib.timer.stop(ev, dev)
    return gq, gk if needs[1] else None, gv if needs[2] else None


class _PackedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, offsets_q, offsets_k, lengths_k, causal, scale):
        args = offsets_q, offsets_k, lengths_k
        out, rest, log_sum = attention_forward(q, k, v, *args, causal, scale)
        ctx.save_for_backward(q, k, v, out, rest, log_sum, *args)
        ctx.how = (causal, scale)
        ctx.mark_non_differentiable(log_sum)
        return out, log_sum

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out, _):
        return (*attention_backward(grad_out, *ctx.saved_tensors, *ctx.how,
                                    ctx.needs_input_grad[:3]),
                None, None, None, None, None)


def packed_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, offsets_q: torch.Tensor,
                     offsets_k: torch.Tensor | None = None, lengths_k: torch.Tensor | None = None,
                     causal: bool = False, scale: float | None = None,
                     return_log_sum: bool = False):
    """softmax(scale q k^T) v for sequences packed one after another.

    q is (queries, heads, dim), k and v (keys, key_heads, dim), float16 or bfloat16,
    dim a multiple of 8 up to 128, heads a multiple of key_heads (consecutive heads
    share a key head).  offsets_q (int32, on the GPU, sequences + 1 entries, rising)
    says where each sequence's queries begin, offsets_k (default: offsets_q) its
    keys.  lengths_k (int32, one a sequence) limits the keys to the first ones of
    the sequence's range, for a cache that is not full.  causal: with Lq queries and
    Lk keys, query i sees keys j <= i + Lk - Lq, so new queries at a cache's end see
    all before them; else every key.  A query without keys gives 0; a row before the
    first offset or after the last gives 0 and a zero gradient, and so do cache rows
    past a length.  Offsets are not read on the host: values outside the tensors are
    clamped, and nothing is checked about them.

    scale defaults to dim ** -0.5.  With return_log_sum also the float32 (queries,
    heads) natural logarithm of each softmax's denominator (no gradient).  Scores
    and sums are float32; probabilities are rounded to q's type before they meet v, and in
    the backward they and the score gradients before they meet grad_out, q and k.

    What a query does not see, whatever it is, changes nothing.  An infinity in a value
    that it sees gives that infinity, or NaN where its probability was rounded to 0 or
    both signs meet; keys that all score minus infinity, though it sees them, give NaN.
    """
    _check("packed_attention", "q", q, 3, (torch.float16, torch.bfloat16))
    dev = q.device
    for name, t in (("k", k), ("v", v)):
        _check("packed_attention", name, t, 3, (q.dtype,), dev)
        if t.shape[2] != q.shape[2]:
            raise RuntimeError(f"packed_attention: {name} must have dimension {q.shape[2]}, got "
                               f"{tuple(t.shape)}")
    if k.shape != v.shape:
        raise RuntimeError(f"packed_attention: k {tuple(k.shape)} and v {tuple(v.shape)} differ")
    heads, key_heads, dim = q.shape[1], k.shape[1], q.shape[2]
    if key_heads < 1 or heads < 1 or heads % key_heads:
        raise RuntimeError(f"packed_attention: {heads} heads are no multiple of {key_heads} key heads")
    if dim % 8 or not 8 <= dim <= MAX_HEAD_DIM:
        raise RuntimeError(f"packed_attention: dimension must be a multiple of 8 up to "
                           f"{MAX_HEAD_DIM}, got {dim}")
    if offsets_k is None:
        if k.shape[0] != q.shape[0]:
            raise RuntimeError("packed_attention: offsets_k is needed where q and k have "
                               f"different rows ({q.shape[0]} and {k.shape[0]})")
        offsets_k = offsets_q
    for name, t, n in (("offsets_q", offsets_q, None), ("offsets_k", offsets_k, 0),
                       ("lengths_k", lengths_k, -1)):
        if t is None and n == -1:
            continue
        _check("packed_attention", name, t, 1, (torch.int32,), dev)
        want = None if n is None else offsets_q.shape[0] + n
        if t.shape[0] != want if want is not None else t.shape[0] < 1:
            raise RuntimeError(f"packed_attention: {name} has {t.shape[0]} entries, expected "
                               f"{'at least 1' if want is None else want}")
    offsets_q, offsets_k = offsets_q.contiguous(), offsets_k.contiguous()
    lengths_k = None if lengths_k is None else lengths_k.contiguous()
    scale = dim ** -0.5 if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"packed_attention: scale must be finite, got {scale}")
    args = (q, k, v, offsets_q, offsets_k, lengths_k, bool(causal), scale)
    if _differentiable("packed_attention", q, k, v):
        out, log_sum = _PackedAttention.apply(*args)
    else:
        out, _, log_sum = attention_forward(*args, with_log_sum=return_log_sum, with_rest=False)
    return (out, log_sum) if return_log_sum else out
