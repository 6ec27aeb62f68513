"""What the linear-attention operators refuse of tensors on the device, through the host module and the general way."""

import pytest
import torch

from anna_amd import linear_attention as la

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def test_dual_tensors_are_refused(gpu):
    def zeros(*shape, dtype=BF):
        return torch.zeros(shape, dtype=dtype, device=gpu)

    span = la.StateSpan([0], [3], device=gpu)
    calls = {
        "norm": (la.rms_norm, dict(x=zeros(3, 16), weight=zeros(16), residual=zeros(3, 16), gate=zeros(3, 16)), {}),
        "codes": (la.rms_norm_e4m3, dict(x=zeros(3, 16), weight=zeros(16), residual=zeros(3, 16), gate=zeros(3, 16)), {}),
        "conv": (la.causal_conv1d, dict(x=zeros(3, 8), weight=zeros(8, 4), bias=zeros(8), state=zeros(1, 3, 8)), dict(span=span)),
        "delta": (la.gated_delta_rule, dict(query=zeros(3, 1, 64), key=zeros(3, 1, 64), value=zeros(3, 1, 32), decay=zeros(3, 1), beta=zeros(3, 1),
                                            state=zeros(1, 1, 64, 32, dtype=torch.float32), a_log=zeros(1, dtype=torch.float32),
                                            dt_bias=zeros(1, dtype=torch.float32)), dict(span=span, scaling=1.0)),
    }
    with torch.autograd.forward_ad.dual_level(), torch.no_grad():
        for call, tensors, more in calls.values():
            call(**tensors, **more)
            for name, t in tensors.items():
                dual = torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))
                with pytest.raises(RuntimeError, match=f"{name} has a tangent"):
                    call(**{**tensors, name: dual}, **more)


@pytest.mark.parametrize("general", [False, True])
def test_autograd_sees_what_is_written(gpu, general, monkeypatch):
    """A tensor that another operation keeps for its backward pass, and that a call writes: the pass refuses it."""
    if general:
        monkeypatch.setattr(la, "_host", type("Nothing", (), {"__getattr__": lambda self, name: lambda *a: None}))

    def zeros(*shape, dtype=BF):
        return torch.zeros(shape, dtype=dtype, device=gpu)

    span = la.StateSpan([0], [3], device=gpu)
    conv_state, state, stream, out = zeros(1, 3, 8), zeros(1, 1, 64, 32, dtype=torch.float32), zeros(3, 16), zeros(3, 16)
    for written, call in [(stream, lambda: la.rms_norm(zeros(3, 16), zeros(16), residual=stream)),
                          (stream, lambda: la.rms_norm_e4m3(zeros(3, 16), zeros(16), residual=stream)),
                          (out, lambda: la.rms_norm(zeros(3, 16), zeros(16), out=out)),
                          (conv_state, lambda: la.causal_conv1d(zeros(3, 8), zeros(8, 4), None, conv_state, span)),
                          (state, lambda: la.gated_delta_rule(zeros(3, 1, 64), zeros(3, 1, 64), zeros(3, 1, 32), zeros(3, 1), zeros(3, 1), state, span,
                                                              scaling=1.0))]:
        w = torch.ones_like(written, requires_grad=True)
        kept = (w * written).float().sum()
        call()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            kept.backward()


def test_inference_tensors_are_written_as_before(gpu):
    with torch.inference_mode():
        stream, state = torch.ones(3, 16, device=gpu), torch.zeros(1, 3, 8, device=gpu)
        la.rms_norm(torch.ones(3, 16, device=gpu), torch.ones(16, device=gpu), residual=stream)
    with torch.no_grad():
        la.rms_norm(torch.ones(3, 16, device=gpu), torch.ones(16, device=gpu), residual=stream)
        la.causal_conv1d(torch.ones(2, 8, device=gpu), torch.ones(8, 4, device=gpu), None, state, la.StateSpan([0], [2], device=gpu))
    assert (stream == 3).all() and (state[0, 1:] == 1).all() and (state[0, 0] == 0).all()
