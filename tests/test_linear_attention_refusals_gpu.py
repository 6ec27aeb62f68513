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
