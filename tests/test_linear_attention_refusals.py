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
