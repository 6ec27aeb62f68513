"""Layout of packed sequences, and what the linear-attention calls refuse, on the host: no GPU is needed."""

import ctypes

import pytest
import torch

from anna_amd import _lib
from anna_amd import linear_attention as la

BF = torch.bfloat16


def plan(slots, counts, fresh=None):
    n = len(slots)
    s, c = (ctypes.c_int32 * n)(*slots), (ctypes.c_int64 * n)(*counts)
    f = None if fresh is None else (ctypes.c_int32 * n)(*fresh)
    span = _lib.StateSpan()
    _lib.call("anna_mi_state_span_plan", n, s, c, f, ctypes.byref(span))
    words = (ctypes.c_int32 * span.words)()
    _lib.call("anna_mi_state_span_fill", n, s, c, f, ctypes.byref(span), words)
    return span, list(words)


def test_struct_sizes():
    lib = _lib.load()
    assert lib.anna_mi_sizeof_state_span() == ctypes.sizeof(_lib.StateSpan)
    assert lib.anna_mi_sizeof_gated_delta_args() == ctypes.sizeof(_lib.GatedDeltaArgs)
    assert lib.anna_mi_sizeof_rms_norm_args() == ctypes.sizeof(_lib.RmsNormArgs)


def test_layout():
    span, words = plan([5, -1, 0, 9, 2], [1, 12, 0, 13, 129], [0, 1, 0, 0, 7])
    assert (span.sequences, span.tokens, span.steps, span.chains, span.chunks, span.longest, span.max_slot) == (5, 155, 2, 2, 4, 3, 9)
    assert words[:20] == [5, 0, 1, 0, -1, 1, 12, 1, 0, 13, 0, 0, 9, 13, 13, 0, 2, 26, 129, 1]
    assert words[20:28] == [5, 0, 1, 0, -1, 1, 12, 1]
    assert words[28:44] == [2, 26, 129, 1, 1, 0, 0, 0, 9, 13, 13, 0, 0, 0, 0, 0]
    assert words[44:60] == [9, 13, 13, 0, 2, 26, 64, 0, 2, 90, 64, 0, 2, 154, 1, 0]
    assert words[60:] == [0] + [1] * 12 + [3] * 13 + [4] * 129
    span, words = plan([], [])
    assert (span.sequences, span.tokens, span.words, span.max_slot) == (0, 0, 1, -1)


@pytest.mark.parametrize("slots,counts,msg", [
    ([1, 2, 1], [1, 1, 1], "slot 1 is named twice"),
    ([-2], [1], "slot -2"),
    ([0], [-1], "of -1 tokens"),
    ([0], [1 << 31], "tokens"),
    ([0, 1], [(1 << 31) - 1, 1], "more than 2"),
])
def test_layout_refuses(slots, counts, msg):
    with pytest.raises(RuntimeError, match=msg):
        plan(slots, counts)


def test_padding_slots_may_repeat():
    span, _ = plan([-1, 3, -1], [1, 1, 1])
    assert span.max_slot == 3


def test_fill_refuses_other_counts():
    span, _ = plan([0, 1], [1, 20])
    s, c, words = (ctypes.c_int32 * 2)(0, 1), (ctypes.c_int64 * 2)(1, 200), (ctypes.c_int32 * 100)()
    with pytest.raises(RuntimeError, match="other counts"):
        _lib.call("anna_mi_state_span_fill", 2, s, c, None, ctypes.byref(span), words)


def test_span_needs_the_device():
    with pytest.raises(RuntimeError, match="ROCm device"):
        la.StateSpan([0], device="cpu")


def delta_inputs(**over):
    t = dict(query=torch.zeros(5, 2, 64, dtype=BF), key=torch.zeros(5, 2, 64, dtype=BF), value=torch.zeros(5, 4, 32, dtype=BF),
             decay=torch.zeros(5, 4), beta=torch.zeros(5, 4), state=torch.zeros(3, 4, 64, 32), span=None, scaling=0.1)
    t.update(over)
    return t


def test_delta_reaches_the_device_check():
    with pytest.raises(RuntimeError, match="ROCm device tensors"):
        la.gated_delta_rule(**delta_inputs())


@pytest.mark.parametrize("over,msg", [
    (dict(query=torch.zeros(5, 2, 64)), "bfloat16 or float16"),
    (dict(query=torch.zeros(5, 128, dtype=BF)), "tokens, heads, dim"),
    (dict(query=torch.zeros(5, 2, 32, dtype=BF), key=torch.zeros(5, 2, 32, dtype=BF)), "key_dim 32"),
    (dict(key=torch.zeros(5, 1, 64, dtype=BF)), "key must be"),
    (dict(key=torch.zeros(4, 2, 64, dtype=BF)), "key must be"),
    (dict(key=torch.zeros(5, 2, 64, dtype=torch.float16)), "key must be"),
    (dict(value=torch.zeros(5, 4, 48, dtype=BF)), "value_dim 48"),
    (dict(value=torch.zeros(5, 4, 288, dtype=BF)), "value_dim 288"),
    (dict(value=torch.zeros(5, 3, 32, dtype=BF)), "multiple of key_heads"),
    (dict(decay=torch.zeros(5, 2)), "decay must be"),
    (dict(beta=torch.zeros(5, 4, dtype=BF)), "beta must be"),
    (dict(decay=torch.zeros(5, 4, dtype=torch.float64), beta=torch.zeros(5, 4, dtype=torch.float64)), "decay must be"),
    (dict(a_log=torch.zeros(4)), "go together"),
    (dict(a_log=torch.zeros(4, dtype=BF), dt_bias=torch.zeros(4)), "a_log must be float32"),
    (dict(a_log=torch.zeros(4), dt_bias=torch.zeros(2)), "dt_bias must be float32"),
    (dict(scaling=float("inf")), "scaling must be finite"),
    (dict(scaling=float("nan")), "scaling must be finite"),
    (dict(state=torch.zeros(3, 4, 32, 64)), "state must be"),
    (dict(state=torch.zeros(3, 4, 64, 32, dtype=BF)), "state must be"),
    (dict(state=torch.zeros(3, 4, 32, 64).transpose(2, 3)), "contiguous in each slot"),
    (dict(state=torch.zeros(1, 4, 64, 32).expand(3, 4, 64, 32)), "slots overlap"),
    (dict(state=torch.zeros(3 * 4 * 64 * 32 + 1)[1:].view(3, 4, 64, 32)), "16-byte aligned"),
])
def test_delta_refuses(over, msg):
    with pytest.raises(ValueError, match=msg):
        la.gated_delta_rule(**delta_inputs(**over))


def conv_inputs(**over):
    t = dict(x=torch.zeros(5, 24, dtype=BF), weight=torch.zeros(24, 4, dtype=BF), bias=None,
             state=torch.zeros(3, 3, 24, dtype=BF), span=None)
    t.update(over)
    return t


def test_conv_reaches_the_device_check():
    with pytest.raises(RuntimeError, match="ROCm device tensors"):
        la.causal_conv1d(**conv_inputs())


@pytest.mark.parametrize("over,msg", [
    (dict(x=torch.zeros(5, 24, dtype=torch.float64)), "x must be"),
    (dict(x=torch.zeros(1, 5, 24, dtype=BF)), "x must be"),
    (dict(weight=torch.zeros(24, 4)), "weight must be"),
    (dict(weight=torch.zeros(24, 9, dtype=BF)), "weight must be"),
    (dict(weight=torch.zeros(24, 1, dtype=BF)), "weight must be"),
    (dict(weight=torch.zeros(4, 24, dtype=BF)), "weight must be"),
    (dict(bias=torch.zeros(23, dtype=BF)), "bias must be"),
    (dict(state=torch.zeros(3, 24, 3, dtype=BF)), "state must be"),
    (dict(state=torch.zeros(3, 24, 3, dtype=BF).transpose(1, 2)), "contiguous in each slot"),
    (dict(activation="gelu"), "activation must be"),
])
def test_conv_refuses(over, msg):
    with pytest.raises(ValueError, match=msg):
        la.causal_conv1d(**conv_inputs(**over))


@pytest.mark.parametrize("kw,msg", [
    (dict(x=torch.zeros(3, 16, dtype=torch.float64), weight=torch.zeros(16)), "x must be"),
    (dict(x=torch.zeros(3, 16), weight=torch.zeros(8)), "weight must be"),
    (dict(x=torch.zeros(3, 16), weight=torch.zeros(16, dtype=BF)), "weight must be"),
    (dict(x=torch.zeros(3, 16), weight=torch.zeros(16), eps=-1.0), "eps must be"),
    (dict(x=torch.zeros(3, 16), weight=torch.zeros(16), eps=float("nan")), "eps must be"),
    (dict(x=torch.zeros(3, 16), weight=torch.zeros(16), out=torch.zeros(16, 3)), "out must be"),
    (dict(x=torch.zeros(3, 16), weight=torch.zeros(16), out=torch.zeros(3, 16, dtype=BF)), "out must be"),
])
def test_norm_refuses(kw, msg):
    with pytest.raises(ValueError, match=msg):
        la.rms_norm(**kw)


def test_norm_refuses_a_residual_over_other_rows():
    wide = torch.zeros(4, 64)
    x, w = wide[:3, :16], torch.zeros(16)
    for residual, kw, name in [(wide[1:, :16], {}, "x"), (wide[:3, 8:24], {}, "x"), (wide.view(-1)[4:52].view(3, 16), {}, "x"),
                               (wide[:3, 16:32], dict(gate=wide[:3, 31:47]), "gate"), (wide[:3, 16:32], dict(gate=wide[:3, 16:32]), "gate")]:
        with pytest.raises(ValueError, match=f"residual must not overlap {name}"):
            la.rms_norm(x, w, residual=residual, **kw)
        with pytest.raises(ValueError, match=f"residual must not overlap {name}"):
            la.rms_norm_e4m3(x, w, residual=residual, **kw)
    with pytest.raises(ValueError, match="residual must not overlap weight"):
        la.rms_norm(x, wide[1, 24:40], residual=wide[:3, 16:32])
    for residual in (x, wide[:3, 16:32], wide[:3, 48:], wide[3:, 16:64].view(3, 16)):
        with pytest.raises(RuntimeError, match="ROCm"):  # nothing but the device
            la.rms_norm(x, w, residual=residual)


def test_norm_refuses_an_output_over_another_row():
    x = torch.zeros(64)
    with pytest.raises(ValueError, match="must not overlap x"):
        la.rms_norm(x[:48].view(3, 16), torch.zeros(16), out=x[16:].view(3, 16))
    with pytest.raises(ValueError, match="must not overlap residual"):
        r = torch.zeros(3, 16)
        la.rms_norm(torch.zeros(3, 16), torch.zeros(16), residual=r, out=r)


@pytest.mark.parametrize("cols,group", [(96, 64), (128, 16), (200, 128), (64, 0)])
def test_e4m3_refuses_groups(cols, group):
    with pytest.raises(ValueError, match="group_size"):
        la.rms_norm_e4m3(torch.zeros(2, cols), torch.zeros(cols), group_size=group)


def test_c_entries_refuse():
    lib = _lib.load()
    span = _lib.StateSpan(1, 1, 9, 1, 0, 0, 0, 0, 1 << 40, None)
    args = _lib.GatedDeltaArgs(dtype=_lib.F32)
    assert lib.anna_mi_gated_delta(None, ctypes.byref(span), None) == 1
    assert lib.anna_mi_gated_delta(ctypes.byref(args), ctypes.byref(span), None) == 1
    assert b"dtype" in lib.anna_mi_last_error()
    args = _lib.GatedDeltaArgs(dtype=_lib.BF16, gates_dtype=_lib.F32, key_heads=2, value_heads=4, key_dim=128, value_dim=128, slots=0)
    assert lib.anna_mi_gated_delta(ctypes.byref(args), ctypes.byref(span), None) == 1
    assert b"slot 0 of a state of 0" in lib.anna_mi_last_error()
    assert lib.anna_mi_causal_conv1d(None, _lib.BF16, 8, 8, None, 4, None, None, 1, 24, 1, ctypes.byref(span), None, 8, None) == 1
    assert b"null pointer" in lib.anna_mi_last_error()
    norm = _lib.RmsNormArgs(dtype=_lib.BF16, out_format=0, rows=1 << 24, cols=8192, x=16, x_stride=8192, weight=16, out=16, out_stride=8192)
    assert lib.anna_mi_rms_norm(ctypes.byref(norm), None) == 1
    assert b"too many for a launch" in lib.anna_mi_last_error()
