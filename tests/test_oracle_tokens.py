"""The float64 oracle of the patch-network operators (oracle/tokens.py): its gradients
from the formulas against central differences of its forward, and hand-made cases;
and the host checks of the operators' entry points (no GPU)."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import helpers  # noqa: F401
import cuda_rasterizer as cr
from cuda_rasterizer import _lib, tokens
from oracle import tokens as ot


def _difference(f, x, d, h=1e-5):
    return float((f(x + h * d) - f(x - h * d)) / (2 * h))


def _agree(got, want):
    assert abs(got - want) <= 1e-7 * max(1.0, abs(want)), (got, want)


def test_layer_norm_gradients_are_the_differences():
    g = torch.Generator().manual_seed(1)
    x, w, b, gy = (torch.randn(s, generator=g, dtype=torch.float64)
                   for s in ((5, 7), (7,), (7,), (5, 7)))
    gx, gw, gb, _, _ = ot.layer_norm_backward(gy, x, w)
    for t, grad, f in ((x, gx, lambda t: (ot.layer_norm(t, w, b) * gy).sum()),
                       (w, gw, lambda t: (ot.layer_norm(x, t, b) * gy).sum()),
                       (b, gb, lambda t: (ot.layer_norm(x, w, t) * gy).sum())):
        d = torch.randn(t.shape, generator=g, dtype=torch.float64)
        _agree(float((grad * d).sum()), _difference(f, t, d))


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_turns_pairs_and_back(interleaved):
    g = torch.Generator().manual_seed(2)
    x = torch.randn(4, 2, 10, generator=g, dtype=torch.float64)
    pos = torch.tensor([[0, 0], [1, 5], [3, 0], [100, 7]])
    f = torch.tensor([1.0, 0.5, 0.25, 2.0])
    y = ot.rotary(x, pos, f, (1, 3), interleaved)
    assert torch.equal(y[0], x[0]) and torch.equal(y[..., 8:], x[..., 8:])
    back = ot.rotary(y, pos, f, (1, 3), interleaved, inverse=True)
    assert float((back - x).abs().max()) < 1e-13
    # the second pair of token 1 turns by position 5 on axis 1 times frequency 0.5
    a, b = (2, 3) if interleaved else (1, 5)
    z = torch.complex(x[1, 0, a], x[1, 0, b]) * complex(math.cos(2.5), math.sin(2.5))
    assert abs(float(y[1, 0, a] - z.real)) < 1e-14 and abs(float(y[1, 0, b] - z.imag)) < 1e-14


@pytest.mark.parametrize("causal", [False, True])
def test_attention_gradients_are_the_differences(causal):
    g = torch.Generator().manual_seed(3)
    oq, ok = torch.tensor([0, 3, 3, 9, 10]), torch.tensor([0, 5, 7, 11, 11])
    q, go = (torch.randn(10, 4, 8, generator=g, dtype=torch.float64) for _ in range(2))
    k, v = (torch.randn(11, 2, 8, generator=g, dtype=torch.float64) for _ in range(2))
    ref = ot.attention(q, k, v, oq, ok, None, causal, grad_out=go)

    def loss(q, k, v):
        return (ot.attention(q, k, v, oq, ok, None, causal)["out"] * go).sum()

    for t, name, f in ((q, "gq", lambda t: loss(t, k, v)), (k, "gk", lambda t: loss(q, t, v)),
                       (v, "gv", lambda t: loss(q, k, t))):
        d = torch.randn(t.shape, generator=g, dtype=torch.float64)
        _agree(float((ref[name] * d).sum()), _difference(f, t, d))
    # the third sequence has 6 queries and 4 keys, the last one key but no query sees it
    assert bool((ref["out"][9] == 0).all()) and bool(torch.isinf(ref["log_sum"][9]).all())
    first = ref["out"][3:5]  # its first two queries come before all its keys
    assert bool((first == 0).all()) == causal


def _attention_problem(**changes):
    fake = 4096  # never dereferenced: every call here is rejected first or has no rows
    fields = dict(rows_q=4, rows_k=4, q_row=64, q_head=64, k_row=64, k_head=64, v_row=64,
                  v_head=64, offsets_q=fake, offsets_k=fake, lengths_k=None, sequences=1,
                  heads_q=2, heads_k=1, dim=64, type=1, causal=0, scale=0.125)
    fields.update(changes)
    return _lib.GsAttention(*(fields[name] for name, _ in _lib.GsAttention._fields_))


def test_entry_points_reject_on_the_host():
    lib = _lib.load()
    some, odd, size = ctypes.c_void_p(4096), ctypes.c_void_p(4104), ctypes.c_size_t(0)
    # layer norm
    norm = (lib.gs_layer_norm_forward, lib.gs_layer_norm_backward)
    assert norm[0](some, 8, None, None, -1, 8, 1e-5, 0, 0, some, None, None) == -1
    assert norm[0](some, 8, None, None, 4, 0, 1e-5, 0, 0, some, None, None) == -1
    assert norm[0](some, 8, None, None, 4, 8, 1e-5, 3, 0, some, None, None) == -1  # type
    assert norm[0](some, 8, None, None, 4, 8, float("nan"), 0, 0, some, None, None) == -1
    assert norm[0](None, 8, None, None, 4, 8, 1e-5, 0, 0, some, None, None) == -1
    assert norm[0](None, 8, None, None, 0, 8, 1e-5, 0, 0, None, None, None) == 0
    assert lib.gs_layer_norm_backward_workspace_size(100, 64, ctypes.byref(size)) == 0
    assert size.value > 0
    assert lib.gs_layer_norm_backward_workspace_size(-1, 64, ctypes.byref(size)) == -1
    assert norm[1](some, 8, some, 8, None, some, 100, 8, 0, 0, some, some, some, some, 1,
                   None) == -2
    assert norm[1](some, 8, some, 8, None, None, 4, 8, 0, 0, some, None, None, None, 0, None) == -1
    # rotary
    t = _lib.GsRotaryTensor(4096, 4096, 64, 32, 64, 32, 2)
    one, sections = ctypes.byref(t), (ctypes.c_int32 * 2)(8, 8)
    rotary = lib.gs_axial_rotary
    assert rotary(one, 1, some, 2, 0, some, sections, 2, 10, 31, 0, 0, 0, None) == -1  # 16 pairs
    assert rotary(one, 1, some, 2, 3, some, sections, 2, 10, 32, 0, 0, 0, None) == -1
    assert rotary(one, 1, some, 2, 0, some, sections, 5, 10, 32, 0, 0, 0, None) == -1
    assert rotary(one, 0, some, 2, 0, some, sections, 2, 10, 32, 0, 0, 0, None) == -1
    assert rotary(one, 1, None, 2, 0, some, sections, 2, 10, 32, 0, 0, 0, None) == -1
    assert rotary(one, 1, some, 2, 0, some, sections, 2, 0, 32, 0, 0, 0, None) == 0
    sections[0] = -1
    assert rotary(one, 1, some, 2, 0, some, sections, 2, 10, 32, 0, 0, 0, None) == -1
    # attention
    forward_size = lib.gs_attention_forward_workspace_size
    assert forward_size(ctypes.byref(_attention_problem()), ctypes.byref(size)) == 0
    for changes, status in (
            (dict(rows_q=-1), -1), (dict(heads_q=3, heads_k=2), -1), (dict(heads_k=0), -1),
            (dict(sequences=-1), -1), (dict(offsets_q=None), -1), (dict(scale=math.nan), -1),
            (dict(type=7), -1), (dict(q_row=-8), -1), (dict(type=0), -4), (dict(dim=60), -4),
            (dict(dim=136), -4), (dict(k_row=60), -4), (dict(rows_k=2**31), -4)):
        a = ctypes.byref(_attention_problem(**changes))
        assert forward_size(a, ctypes.byref(size)) == status, changes
        assert lib.gs_attention_forward(a, some, some, some, some, None, None, None, 0,
                                        None) == status
        assert lib.gs_attention_backward(a, *([some] * 7), 64, 64, some, some, some, some, 1 << 40,
                                         None) == status
    a = ctypes.byref(_attention_problem())
    assert lib.gs_attention_forward(a, None, some, some, some, None, None, None, 0, None) == -1
    assert lib.gs_attention_forward(a, odd, some, some, some, None, None, None, 0, None) == -4
    assert lib.gs_attention_backward_workspace_size(a, ctypes.byref(size)) == 0
    assert lib.gs_attention_backward(a, *([some] * 7), 64, 64, some, some, some, some,
                                     size.value - 1, None) == -2
    assert lib.gs_attention_backward(a, *([some] * 7), 60, 64, some, some, some, some, size.value,
                                     None) == -4
    assert lib.gs_attention_forward(ctypes.byref(_attention_problem(rows_q=0)), None, None, None,
                                    None, None, None, None, 0, None) == 0


def test_python_layer_refuses_cpu_tensors_and_other_things():
    x = torch.zeros(4, 2, 64, dtype=torch.float16)
    at = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU only"):
        cr.packed_attention(x, x, x, at)
    with pytest.raises(RuntimeError, match="GPU only"):
        cr.layer_norm(x)
    with pytest.raises(RuntimeError, match="GPU only"):
        cr.axial_rotary(x, None, torch.zeros(4, 1, dtype=torch.int32), torch.ones(2), (2,))
    with pytest.raises(RuntimeError, match="torch.Tensor"):
        cr.layer_norm([1.0])
    f = cr.axial_frequencies((2, 4), 16.0, "cpu")
    assert torch.allclose(f, torch.tensor([1.0, 0.25, 1.0, 0.5, 0.25, 0.125]))
    assert tokens.MAX_HEAD_DIM == 128
