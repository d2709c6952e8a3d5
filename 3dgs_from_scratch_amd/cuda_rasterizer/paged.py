"""A paged cache of keys and values, for a network that takes its views one by one.

packed_attention reads a cache whose sequences lie in slabs, each as long as the longest
may become.  Scenes are 12 to some ten thousands of tokens long, and a stream of views has
no end; here their keys and values lie in pages of one pool:

    k_pages, v_pages   (pages, page_size, key_heads, dim), float16 or bfloat16
    weights            (pages, page_size, key_heads), float32: the attention that keys got
    tables             (sequences, width), int32: the pages of a sequence, in order
    lengths            (sequences,), int32: the slots that it has filled

Slot i of sequence b is place i % page_size of page tables[b, i // page_size].  Who owns
which page is the caller's to say, and sequences may share pages that nothing is appended to.

- paged_append(k, v, k_pages, v_pages, tables, lengths, offsets, weights): new tokens' keys
  and values into the last slots of their sequences;
- paged_attention(q, k_pages, v_pages, tables, lengths, offsets, ...): the new tokens over
  the slots, themselves among them, and what attention each slot gets on request;
- paged_evict(k_pages, v_pages, weights, tables, lengths, new_tables, keep, recent): the
  slots with the largest weights, and the most recent ones, to other pages.

lengths count the new tokens in all of them.  All run on the library's gfx950 kernels on
the current HIP stream, without host synchronisation; tables, lengths and offsets are not
read on the host, so that a captured step may change them.  They are for prediction: there
are no gradients, and a tensor that requires one is refused while gradients are recorded.
A page number outside the pool (-1, say) stands for slots that are not there: no query
sees them, nothing is written to them.  Nothing here has a counterpart in the reference.
"""

from __future__ import annotations

import ctypes
import functools

import torch
from torch.autograd import forward_ad

from . import _lib
from ._lib import GsPagedQueries, GsPages
from .tokens import (_MAX_STRIDE, _TYPES, MAX_HEAD_DIM, _check, _laid_out, _ptr, _scale_of,
                     _workspace)

_HALVES = (torch.float16, torch.bfloat16)
MAX_SLOTS = (1 << 31) - 1 - 65536  # of a sequence


def _no_gradient(what: str, *tensors) -> None:
    """The operators have no derivatives, and a trace would record their outputs as constants."""
    if torch.jit.is_tracing():
        raise RuntimeError(f"{what} cannot be traced")
    grad = torch.is_grad_enabled()
    # (outside of every dual level, -1, there are no tangents)
    dual = getattr(forward_ad, "_current_level", 0) >= 0
    if not grad and not dual:
        return
    for t in tensors:
        if isinstance(t, torch.Tensor):
            if grad and t.requires_grad:
                raise RuntimeError(f"{what} has no gradient; call it under torch.no_grad()")
            if dual and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError(f"{what} has no forward-mode derivative")


def _written(*tensors) -> None:
    """Tells autograd that the tensors' values have changed."""
    torch.autograd.graph.increment_version([t for t in tensors
                                            if t is not None and not t.is_inference()])


def _apart(shape, strides, inner: int) -> bool:
    """Whether no two of the blocks of `inner` elements that the dimensions number overlap."""
    extent = inner
    for stride, size in sorted(zip(strides, shape)):
        if size > 1:
            if stride < extent:
                return False
            extent += (size - 1) * stride
    return True


# What follows from sizes alone is remembered by them.
@functools.lru_cache(maxsize=256)
def _pool_strides(shape, strides):
    """Strides of pages, slots and heads, 0 where there is but one (and of slots dim); None where
    the kernels cannot read or write such a pool."""
    *shape, dim = shape
    strides, last = [s if n > 1 else 0 for n, s in zip(shape, strides)], strides[3]
    apart = _apart(shape, strides, dim)
    if shape[1] == 1:
        strides[1] = dim
    if (last != 1 or any(s % 8 or s >= 1 << 31 for s in strides) or strides[1] > _MAX_STRIDE
            or not apart):
        return None
    return tuple(strides)


@functools.lru_cache(maxsize=256)
def _weight_strides(shape, strides):
    strides = tuple(s if n > 1 else 0 for n, s in zip(shape, strides))
    return strides if max(strides) < 1 << 31 and _apart(shape, strides, 1) else None


@functools.lru_cache(maxsize=256)
def _layout(what: str, shape, k_strides, v_shape, v_strides, w_shape, w_strides, tables, lengths):
    """The numbers of a cache's description between its pointers, for sizes that go together."""
    pages, page_size, heads, dim = shape
    if v_shape != shape:
        raise RuntimeError(f"{what}: k_pages {tuple(shape)} and v_pages {tuple(v_shape)} must have "
                           "the same shape")
    if page_size < 1 or heads < 1:
        raise RuntimeError(f"{what}: k_pages {tuple(shape)} has pages of nothing")
    if dim % 8 or not 8 <= dim <= MAX_HEAD_DIM:
        raise RuntimeError(f"{what}: dimension must be a multiple of 8 up to {MAX_HEAD_DIM}, got {dim}")
    strides = _pool_strides(shape, k_strides)
    if strides is None or strides != _pool_strides(shape, v_strides):
        raise RuntimeError(f"{what}: k_pages and v_pages must have the same strides, "
                           "with neighbouring elements in the last dimension, other strides that are "
                           "multiples of 8 below 2^31, that of a page's slots at most 2^23, and rows that "
                           f"do not overlap; got {k_strides} and {v_strides}")
    sums = (0, 0, 0)
    if w_shape is not None:
        if w_shape != shape[:3]:
            raise RuntimeError(f"{what}: weights must be {tuple(shape[:3])}, got {tuple(w_shape)}")
        sums = _weight_strides(w_shape, w_strides)
        if sums is None:
            raise RuntimeError(f"{what}: weights overlap in memory or have strides of 2^31 or more, "
                               f"got {w_strides}")
    sequences, width = tables
    if lengths[0] != sequences:
        raise RuntimeError(f"{what}: lengths must have {sequences} entries, got {lengths[0]}")
    if max(sequences, page_size, heads) > MAX_SLOTS:
        raise RuntimeError(f"{what}: {sequences} sequences and {heads} heads in pages of {page_size} are "
                           "too many")
    if width * page_size > MAX_SLOTS:
        raise RuntimeError(f"{what}: at most {MAX_SLOTS} slots a sequence are supported, got "
                           f"{width} pages of {page_size}")
    return (pages, *strides, *sums), (width, sequences, page_size, heads, dim)


def _pages(what: str, k_pages, v_pages, weights, tables, lengths) -> GsPages:
    """The checked description of a cache."""
    if not (_on(k_pages, v_pages, tables, lengths) and (weights is None or (
            isinstance(weights, torch.Tensor) and weights.dtype is torch.float32
            and weights.get_device() == k_pages.get_device() and weights.dim() == 3))):
        _check(what, "k_pages", k_pages, 4, _HALVES)
        dev = k_pages.device
        _check(what, "v_pages", v_pages, 4, (k_pages.dtype,), dev)
        if weights is not None:
            _check(what, "weights", weights, 3, (torch.float32,), dev)
        _check(what, "tables", tables, 2, (torch.int32,), dev)
        _check(what, "lengths", lengths, 1, (torch.int32,), dev)
    w = (None, None) if weights is None else (weights.shape, weights.stride())
    first, last = _layout(what, k_pages.shape, k_pages.stride(), v_pages.shape, v_pages.stride(), *w,
                          tables.shape, lengths.shape)
    if (k_pages.data_ptr() | v_pages.data_ptr()) % 16:
        raise RuntimeError(f"{what}: k_pages and v_pages must begin on 16 bytes")
    return GsPages(*first, tables.data_ptr(), lengths.data_ptr(), tables.stride(0), *last,
                   _TYPES[k_pages.dtype])


# The checks find nothing where these are true, at less of the host's time.
def _on(k_pages, v_pages, tables, lengths) -> bool:
    try:
        device, dtype = k_pages.get_device(), k_pages.dtype
        return (device >= 0 and dtype in _HALVES and v_pages.dtype is dtype
                and tables.dtype is torch.int32 and lengths.dtype is torch.int32
                and device == v_pages.get_device() == tables.get_device() == lengths.get_device()
                and k_pages.dim() == v_pages.dim() == 4 and tables.dim() == 2 and lengths.dim() == 1)
    except AttributeError:  # no tensor
        return False


def _heads_on(t, k_pages) -> bool:
    return (isinstance(t, torch.Tensor) and t.dtype is k_pages.dtype and t.dim() == 3
            and t.get_device() == k_pages.get_device())


def _rows(t):
    """t with neighbouring entries in its last dimension (what is no tensor is refused later)."""
    return t.contiguous() if isinstance(t, torch.Tensor) and t.dim() and t.stride(-1) != 1 else t


def _offsets(what: str, offsets, tables) -> None:
    if not (isinstance(offsets, torch.Tensor) and offsets.dtype is torch.int32 and offsets.dim() == 1
            and offsets.get_device() == tables.get_device()):
        _check(what, "offsets", offsets, 1, (torch.int32,), tables.device)
    if offsets.shape[0] != tables.shape[0] + 1:
        raise RuntimeError(f"{what}: offsets must have {tables.shape[0] + 1} entries, got "
                           f"{offsets.shape[0]}")


def paged_append(k: torch.Tensor, v: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 tables: torch.Tensor, lengths: torch.Tensor, offsets: torch.Tensor,
                 weights: torch.Tensor | None = None) -> None:
    """Writes new keys and values into their sequences' last slots, in place.

    k and v are (tokens, key_heads, dim) in the pool's type.  offsets (int32, on the GPU,
    sequences + 1 entries, rising) says where each sequence's tokens begin; with Ln of them,
    token i goes to slot lengths[b] - Ln + i, so lengths already count them.  The slots'
    weights become 0 where weights is given.  Rows before the first offset or after the last,
    and tokens whose slot is below 0, past the table or on no page, go nowhere, so that no
    earlier token is lost; offsets are clamped to the tokens.  Two tokens on one place of a
    page (a page that two tables have) leave a mixture of both."""
    what = "paged_append"
    _no_gradient(what, k, v, k_pages, v_pages, weights)
    tables, lengths, offsets = _rows(tables), _rows(lengths), _rows(offsets)
    p = _pages(what, k_pages, v_pages, weights, tables, lengths)
    dev = k_pages.device
    for name, t in (("k", k), ("v", v)):
        if not _heads_on(t, k_pages):
            _check(what, name, t, 3, (k_pages.dtype,), dev)
        if t.shape[1] != p.heads or t.shape[2] != p.dim:
            raise RuntimeError(f"{what}: {name} must have {p.heads} heads of {p.dim}, got "
                               f"{tuple(t.shape)}")
    if k.shape != v.shape:
        raise RuntimeError(f"{what}: k {tuple(k.shape)} and v {tuple(v.shape)} differ")
    _offsets(what, offsets, tables)
    k, v = _laid_out(k), _laid_out(v)
    with _lib.on_device(dev):
        ev = _lib.timer.record(what, dev)
        _lib.check(_lib.load().gs_paged_append(
            ctypes.byref(p), k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0),
            v.stride(1), k.shape[0], offsets.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
            _ptr(weights), _lib.stream_of(dev)), what)
        _lib.timer.stop(ev, dev)
    _written(k_pages, v_pages, weights)


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                    tables: torch.Tensor, lengths: torch.Tensor, offsets: torch.Tensor,
                    causal: bool = False, scale: float | None = None,
                    weights: torch.Tensor | None = None, return_log_sum: bool = False):
    """softmax(scale q k^T) v of queries over their sequences' filled slots, (queries, heads,
    dim), contiguous.

    q is (queries, heads, dim) in the pool's type, heads a multiple of key_heads (consecutive
    heads share a key head), and offsets (int32, on the GPU, sequences + 1 entries, rising)
    says where each sequence's queries begin: one token each, or chunks of any sizes.  causal:
    of Lq queries, query i sees slots j <= i + lengths[b] - Lq, so that new tokens, appended
    before, see all before them; else every filled slot.  A query that sees no slot, and a row
    of no sequence, gives 0.  lengths are clamped to the tables, as if a longer sequence ended
    there, offsets to the queries.

    With weights also adds to each slot's weight the probabilities that it gets, summed over
    the sequence's queries and the heads that share its key head, in float32 and in an order
    that depends on the sizes and tables alone.  A page that the tables hold several times, such
    as one that sequences share, gets those of all its places there, in any order: only there
    may the last bits of repeated calls differ.  With weights, sequences times key heads
    times the slots that a table's row covers are below 2^38 - 2^23.

    scale defaults to dim ** -0.5.  With return_log_sum also the float32 (queries, heads)
    natural logarithm of each softmax's denominator.  Types, rounding and what is not finite
    are as packed_attention's; queries with a log-sum of -infinity add no weights."""
    what = "paged_attention"
    _no_gradient(what, q, k_pages, v_pages, weights)
    tables, lengths, offsets = _rows(tables), _rows(lengths), _rows(offsets)
    p = _pages(what, k_pages, v_pages, weights, tables, lengths)
    dev = k_pages.device
    if not _heads_on(q, k_pages):
        _check(what, "q", q, 3, (k_pages.dtype,), dev)
    heads = q.shape[1]
    if q.shape[2] != p.dim:
        raise RuntimeError(f"{what}: q must have dimension {p.dim}, got {tuple(q.shape)}")
    if heads < 1 or heads % p.heads:
        raise RuntimeError(f"{what}: {heads} heads are no multiple of {p.heads} key heads")
    _offsets(what, offsets, tables)
    scale = _scale_of(what, scale, p.dim)
    q = _laid_out(q)
    a = GsPagedQueries(q.shape[0], q.stride(0), q.stride(1), offsets.data_ptr(), heads,
                       bool(causal), scale)
    out = torch.empty(q.shape, dtype=q.dtype, device=dev)
    log_sum = (torch.empty(q.shape[:2], dtype=torch.float32, device=dev)
               if return_log_sum or weights is not None else None)
    lib = _lib.load()
    with _lib.on_device(dev):
        ws, size = _workspace(lib.gs_paged_attention_workspace_size, ctypes.byref(p),
                              ctypes.byref(a), weights is not None, device=dev)
        ev = _lib.timer.record(what, dev)
        _lib.check(lib.gs_paged_attention(
            ctypes.byref(p), ctypes.byref(a), q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
            out.data_ptr(), _ptr(log_sum), _ptr(weights), _ptr(ws), size, _lib.stream_of(dev)), what)
        _lib.timer.stop(ev, dev)
    if weights is not None:
        _written(weights)
    return (out, log_sum) if return_log_sum else out


def paged_evict(k_pages: torch.Tensor, v_pages: torch.Tensor, weights: torch.Tensor,
                tables: torch.Tensor, lengths: torch.Tensor, new_tables: torch.Tensor, keep: int,
                recent: int = 0):
    """(new_lengths, kept): copies the `keep` slots that matter of every sequence and key head,
    keys, values and weights, to slots 0, 1, ... of the pages in new_tables, in their order.

    Those are the last `recent` filled slots, and of the others those with the largest weights
    (the lower slot where they are equal; NaN counts as the largest); all where there are no
    more than `keep`.  Slots on no page do not count.  Each key head keeps its own: positions
    lie in the keys (axial_rotary), and attention does not ask for a slot's number beyond the
    order of the newest.  new_tables is int32 (sequences, at least keep / page_size); a page in
    it must be in no table that is read here and in one row only.  The old pages stay as they
    are, for other sequences that share them or for the caller to use again.

    new_lengths (int32, sequences) is how many stayed, the same for all heads, and kept (int32,
    (sequences, key_heads, keep)) which, rising, -1 behind the last."""
    what = "paged_evict"
    _no_gradient(what, k_pages, v_pages, weights)
    given = tables, new_tables
    tables, lengths, new_tables = _rows(tables), _rows(lengths), _rows(new_tables)
    if weights is None:
        raise RuntimeError(f"{what}: weights must be a torch.Tensor, got NoneType")
    p = _pages(what, k_pages, v_pages, weights, tables, lengths)
    dev = k_pages.device
    _check(what, "new_tables", new_tables, 2, (torch.int32,), dev)
    keep, recent = int(keep), int(recent)
    if keep < 1 or not 0 <= recent <= keep:
        raise ValueError(f"{what}: keep must be at least 1 and recent from 0 to keep, got {keep} "
                         f"and {recent}")
    if keep > MAX_SLOTS:
        raise ValueError(f"{what}: at most {MAX_SLOTS} slots a sequence are supported, keep is {keep}")
    if new_tables.shape[0] != p.sequences or new_tables.shape[1] * p.page_size < keep:
        raise RuntimeError(f"{what}: new_tables must have {p.sequences} rows of "
                           f"{-(-keep // p.page_size)} pages at least, got {tuple(new_tables.shape)}")
    if given[0].data_ptr() == given[1].data_ptr() and tables.numel():  # (_rows may have copied them)
        raise ValueError(f"{what}: new_tables are the tables that are read; slots move to other pages")
    new_lengths = torch.empty(p.sequences, dtype=torch.int32, device=dev)
    kept = torch.empty((p.sequences, p.heads, keep), dtype=torch.int32, device=dev)
    with _lib.on_device(dev):
        ev = _lib.timer.record(what, dev)
        _lib.check(_lib.load().gs_paged_evict(
            ctypes.byref(p), k_pages.data_ptr(), v_pages.data_ptr(), weights.data_ptr(),
            new_tables.data_ptr(), new_tables.stride(0), new_tables.shape[1], keep, recent,
            new_lengths.data_ptr(), kept.data_ptr(), _lib.stream_of(dev)), what)
        _lib.timer.stop(ev, dev)
    _written(k_pages, v_pages, weights)
    return new_lengths, kept
