"""Calls of the linear-attention operators that would write over what they read, or lose what they were given: refused on the
host, no GPU is needed."""

import ctypes

import pytest
import torch

from anna_amd import _lib
from anna_amd import linear_attention as la

BF = torch.bfloat16


def test_norm_refuses_its_residual_as_output_by_any_name():
    x, w = torch.zeros(3, 16), torch.zeros(16)
    for residual, out in [(x, x), (x.view(3, 16), x), (x, x.view(3, 16))]:  # the sum would be lost behind the norm
        with pytest.raises(ValueError, match="out must not overlap residual"):
            la.rms_norm(x, w, residual=residual, out=out)
    gate = torch.zeros(3, 16)
    with pytest.raises(ValueError, match="out must not overlap residual"):
        la.rms_norm(x, w, gate=gate, residual=gate, out=gate)
    with pytest.raises(ValueError, match="out must not overlap weight"):
        la.rms_norm(w, w, out=w)
    for kw in (dict(out=x), dict(gate=gate, out=gate), dict(gate=x, out=x), dict(residual=torch.zeros(3, 16), out=x)):
        with pytest.raises(RuntimeError, match="ROCm"):  # nothing but the device
            la.rms_norm(x, w, **kw)


def norm_args(**over):
    t = dict(dtype=_lib.BF16, rows=3, cols=16, x=1 << 20, x_stride=16, weight=1 << 21, out=1 << 22, out_stride=16, eps=1e-6)
    t.update(over)
    return _lib.RmsNormArgs(**t)


@pytest.mark.parametrize("over", [
    dict(residual=1 << 22, residual_stride=16), dict(residual=(1 << 22) + 64, residual_stride=16),
    dict(x=1 << 22, residual=1 << 22, residual_stride=16), dict(residual=(1 << 22) + 16, residual_stride=48, out_stride=48),
    dict(residual=(1 << 22) + 40, residual_stride=16, out_format=1, group=16, scales=1 << 23),
])
def test_the_c_entry_refuses_an_output_over_the_residual(over):
    assert _lib.load().anna_mi_rms_norm(ctypes.byref(norm_args(**over)), None) == 1
    assert b"out overlaps the residual" in _lib.load().anna_mi_last_error()


def conv(**over):
    store = torch.zeros(6, 64, dtype=BF)
    t = dict(x=torch.zeros(5, 8, dtype=BF), weight=torch.zeros(8, 4, dtype=BF), bias=torch.zeros(8, dtype=BF), state=torch.zeros(3, 3, 8, dtype=BF), span=None)
    t.update({n: f(store) for n, f in over.items()})
    return t


def slots(store, rows=3):  # states in the first 24 columns of a matrix
    return store[:rows].as_strided((rows, 3, 8), (64, 8, 1))


@pytest.mark.parametrize("over,name", [
    (dict(state=slots, x=lambda s: s[1:6, :8]), "x"),  # the same columns
    (dict(state=slots, x=lambda s: s[:5, 20:28]), "x"),
    (dict(state=slots, x=lambda s: s[:5, 60:].as_strided((5, 8), (64, 1))), "x"),  # over a row's end into the next slot
    (dict(state=slots, x=lambda s: s.view(-1)[24:64].view(5, 8), weight=lambda s: s[1, 8:40].view(8, 4)), "weight"),
    (dict(state=slots, x=lambda s: s.view(-1)[32:72].view(5, 8)), "x"),
    (dict(state=slots, x=lambda s: s.view(-1)[24:].as_strided((5, 8), (10, 1)), bias=lambda s: s[2, 23:31]), "x"),
    (dict(state=slots, bias=lambda s: s[2, 23:31]), "bias"),
    (dict(state=lambda s: s.view(-1)[:72].view(3, 3, 8), x=lambda s: s.view(-1)[70:110].view(5, 8)), "x"),
])
def test_conv_refuses_a_state_over_its_inputs(over, name):
    with pytest.raises(ValueError, match=f"state must not overlap {name}"):
        la.causal_conv1d(**conv(**over))


@pytest.mark.parametrize("over", [
    dict(state=slots, x=lambda s: s[:5, 24:32]), dict(state=slots, x=lambda s: s[1:6, 56:]), dict(state=slots, x=lambda s: s[4:, :8].repeat(3, 1)[:5]),
    dict(state=slots, x=lambda s: s.view(-1)[24:64].view(5, 8)),  # all in the gap behind a slot
    dict(state=slots, bias=lambda s: s[1, 24:32]), dict(state=lambda s: s.view(-1)[:72].view(3, 3, 8), x=lambda s: s.view(-1)[72:112].view(5, 8)),
    dict(state=slots, x=lambda s: s[:0, :8]), dict(state=lambda s: s[2:2].as_strided((0, 3, 8), (24, 8, 1)), x=lambda s: s[:5, :8]),
    dict(state=lambda s: s.view(-1)[:24].view(1, 3, 8), x=lambda s: s.view(-1)[24:64].view(5, 8)),
])
def test_conv_takes_a_state_beside_its_inputs(over):
    with pytest.raises(RuntimeError, match="ROCm device tensors"):
        la.causal_conv1d(**conv(**over))


@pytest.mark.parametrize("name", ["query", "key", "value", "decay", "beta", "a_log", "dt_bias"])
def test_delta_refuses_a_state_over_its_inputs(name):
    store = torch.zeros(3 * 4 * 64 * 32 + 640)
    t = dict(query=torch.zeros(5, 2, 64, dtype=BF), key=torch.zeros(5, 2, 64, dtype=BF), value=torch.zeros(5, 4, 32, dtype=BF),
             decay=torch.zeros(5, 4), beta=torch.zeros(5, 4), a_log=torch.zeros(4), dt_bias=torch.zeros(4),
             state=store[:3 * 4 * 64 * 32].view(3, 4, 64, 32), span=None, scaling=0.1)
    for first, refused in ((3 * 4 * 64 * 32 - 4, True), (3 * 4 * 64 * 32, False)):
        flat = store[first:first + t[name].numel() * t[name].element_size() // 4]
        over = flat.view(t[name].dtype).view(t[name].shape)
        with pytest.raises(ValueError if refused else RuntimeError, match=f"state must not overlap {name}" if refused else "ROCm device tensors"):
            la.gated_delta_rule(**{**t, name: over})


def test_the_c_entries_refuse_a_state_over_their_inputs():
    lib = _lib.load()
    span = _lib.StateSpan(1, 5, 9, 1, 0, 0, 0, 0, 1 << 40, 1 << 30)
    mb = 1 << 20
    assert lib.anna_mi_causal_conv1d(mb, _lib.BF16, 8, 8, 2 * mb, 4, None, mb + 64, 1, 24, 1, ctypes.byref(span), 3 * mb, 8, None) == 1
    assert b"the state overlaps x" in lib.anna_mi_last_error()
    assert lib.anna_mi_causal_conv1d(mb, _lib.BF16, 8, 8, 2 * mb, 4, 4 * mb, 4 * mb, 1, 24, 1, ctypes.byref(span), 3 * mb, 8, None) == 1
    assert b"the state overlaps bias" in lib.anna_mi_last_error()
    fields = dict(dtype=_lib.BF16, gates_dtype=_lib.F32, key_heads=1, value_heads=1, key_dim=64, value_dim=32, scaling=1.0, slots=1, state_stride_slot=2048,
                  query_stride_token=64, key_stride_token=64, value_stride_token=32, decay_stride=1, beta_stride=1, state=mb, out=9 * mb,
                  query=2 * mb, key=3 * mb, value=4 * mb, decay=5 * mb, beta=6 * mb, a_log=7 * mb, dt_bias=8 * mb)
    for name in ("query", "key", "value", "decay", "beta", "a_log", "dt_bias"):
        args = _lib.GatedDeltaArgs(**{**fields, name: mb + 16})
        assert lib.anna_mi_gated_delta(ctypes.byref(args), ctypes.byref(span), None) == 1
        assert b"the state overlaps " + name.encode() in lib.anna_mi_last_error()
    assert span.least_slots == 1 << 40  # a refused call leaves no trace


def test_dual_tensors_are_refused():
    """Their tangents would be lost without a word, under no_grad too."""
    x = torch.zeros(3, 16)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones(3, 16))
        with torch.no_grad(), pytest.raises(RuntimeError, match="gate has a tangent"):
            la._on(torch.device("cpu"), x=x, weight=None, gate=dual)
        la._on(torch.device("cpu"), x=x)
    la._on(torch.device("cpu"), x=x)


def refilled(monkeypatch, meanwhile):
    """A span of two sequences whose layout is made again, with `meanwhile` run as a call of another thread would be."""
    monkeypatch.setattr(torch.cuda, "is_available", lambda: False)  # nothing here is captured
    span = object.__new__(la.StateSpan)
    span._counts, span._c = None, _lib.StateSpan()
    span._ref = ctypes.byref(span._c)
    span._lay_out([0, 1], [1, 1], None)
    real = _lib.call

    def call(name, *args):
        real(name, *args)
        if name == "anna_mi_state_span_fill":
            meanwhile(span._c)

    monkeypatch.setattr(_lib, "call", call)
    return span


def test_a_refill_keeps_what_a_call_beside_it_found_out(monkeypatch):
    def small_pool(c):
        c.least_slots = 4

    span = refilled(monkeypatch, small_pool)
    span._lay_out([3, 1], [1, 1], None)
    assert span._c.least_slots == 4 and span._c.max_slot == 3
    with pytest.raises(RuntimeError, match="slot 4: the span was used with states of 4 slots"):
        span._lay_out([2, 4], [1, 1], None)
    assert span._c.max_slot == 3 and span.slots == [3, 1]


def test_a_refill_behind_the_pool_of_a_call_beside_it_is_refused(monkeypatch):
    def small_pool(c):
        c.least_slots = 4

    span = refilled(monkeypatch, small_pool)
    with pytest.raises(RuntimeError, match="slot 9: the span was used with states of 4 slots"):
        span._lay_out([9, 1], [1, 1], None)
    assert span._c.max_slot == 1 and span.slots == [0, 1]


def test_the_c_refill_refuses():
    lib = _lib.load()
    span, plan = _lib.StateSpan(2, 2, 18, 2, 0, 0, 0, 1, 4, None), _lib.StateSpan(2, 2, 18, 2, 0, 0, 0, 4, 1 << 40, None)
    assert lib.anna_mi_state_span_refill(ctypes.byref(span), ctypes.byref(plan)) == 1
    assert b"slot 4: the span was used with states of 4 slots" in lib.anna_mi_last_error() and span.max_slot == 1
    plan.max_slot = 3
    assert lib.anna_mi_state_span_refill(ctypes.byref(span), ctypes.byref(plan)) == 0
    assert (span.max_slot, span.least_slots) == (3, 4)
    plan.tokens = 3
    assert lib.anna_mi_state_span_refill(ctypes.byref(span), ctypes.byref(plan)) == 1
    assert b"other counts" in lib.anna_mi_last_error()
    assert lib.anna_mi_state_span_refill(None, ctypes.byref(plan)) == 1
