"""The bounds that gradients of attention are held to (oracle/tokens.py::attention_gradients):
the same gradients as the formulas', bounds that a rounding implementation keeps, and that zeros
do not; and a host check of layer norm's entry points (no GPU)."""

from __future__ import annotations

import ctypes

import pytest
import torch

import helpers  # noqa: F401
from cuda_rasterizer import _lib
from oracle import tokens as ot

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def inputs(lq, lk, dtype, dim=64, size=1.5):
    g = torch.Generator().manual_seed(sum(lq) + 3 * sum(lk))
    q, go = (torch.randn(sum(lq), 4, dim, generator=g) for _ in range(2))
    k, v = (torch.randn(sum(lk), 2, dim, generator=g) for _ in range(2))
    at = [torch.tensor([0] + n).cumsum(0) for n in (lq, lk)]
    return *((size * t).to(dtype) for t in (q, k)), v.to(dtype), go.to(dtype), *at


def rounding(q, k, v, oq, ok, causal, go):
    """One sequence's gradients in float64, but weights, score gradients and results rounded to
    q's type, and delta from an output of rounded weights."""
    dtype, group, scale = q.dtype, q.shape[1] // k.shape[1], q.shape[2] ** -0.5
    got = [torch.zeros_like(t, dtype=torch.float64) for t in (q, k, v)]
    for q0, q1, k0, k1 in ot.spans(oq, ok, None, q.shape[0], k.shape[0]):
        for h in range(q.shape[1]):
            kv = slice(k0, k1), h // group
            qh, kh, vh, g = (t.double() for t in (q[q0:q1, h], k[kv], v[kv], go[q0:q1, h]))
            s = scale * qh @ kh.T
            if causal:
                s = s.masked_fill(torch.ones_like(s, dtype=torch.bool).triu(k1 - k0 - q1 + q0 + 1),
                                  -torch.inf)
            p = torch.exp(s - torch.logsumexp(s, 1, keepdim=True))
            w = (p / p.amax(1, keepdim=True)).to(dtype).double()
            o = w @ vh / w.sum(1, keepdim=True)
            ds = p * (g @ vh.T - (g * o).sum(1, keepdim=True))
            top = ds.abs().amax(0, keepdim=True) / 512
            rounded = (ds / top).to(dtype).double() * top
            got[0][q0:q1, h] = scale * (ds if dtype == torch.float16 else ds.to(dtype).double()) @ kh
            got[1][kv] += scale * rounded.T @ qh
            got[2][kv] += (p * 1024).to(dtype).double().T @ g / 1024
    return [t.to(dtype) for t in got]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lq,lk,causal", [([700, 5, 100], [700, 5, 100], True), ([1], [20_001], False),
                                          ([70], [3000], True), ([257], [257], False)])
def test_bounds_let_roundings_pass_and_zeros_fail(lq, lk, causal, dtype):
    q, k, v, go, oq, ok = inputs(lq, lk, dtype)
    ref = ot.attention_gradients(q, k, v, oq, go, ok, causal=causal)
    same = ot.attention(q, k, v, oq, ok, causal=causal, grad_out=go)
    for name, got in zip(("gq", "gk", "gv"), rounding(q, k, v, oq, ok, causal, go)):
        want, bound = ref[name], ref[name + "_bound"]
        assert float((want - same[name]).abs().max()) <= 1e-12 * float(want.abs().max())
        off = (got.double() - want).abs()
        assert bool((off <= bound).all()) and float(off.norm()) <= 3 * U[dtype] * float(want.norm())
        assert float(want.norm()) > 0.0  # so that zeros are not within 3 u of it
        if dtype == torch.float16:  # and element by element, where the type has the bits
            assert float((want.abs() > bound).double().mean()) > 0.6, name


def test_layer_norm_entry_points_refuse_too_many_channels():
    lib, size = _lib.load(), ctypes.c_size_t(0)
    some, many = ctypes.c_void_p(4096), 2 ** 30 + 1  # rejected before anything is read
    assert lib.gs_layer_norm_forward(some, many, None, None, 1, many, 1e-5, 0, 0, some, None, None) == -4
    assert lib.gs_layer_norm_backward_workspace_size(1, many, ctypes.byref(size)) == -4
    assert lib.gs_layer_norm_backward(some, many, some, many, None, some, 1, many, 0, 0, some, None,
                                      None, None, 0, None) == -4
