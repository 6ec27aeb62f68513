"""The codes of rms_norm_e4m3 are the quotients of the values and the scales, rounded once to fp32 and once to e4m3."""

import pytest
import torch

from anna_amd import linear_attention as la

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cols,group", [(64, 32), (128, 128), (448, None), (4096, 128), (4104, None), (12288, 64), (8200 * 2, None)])
def test_codes_are_quotients(gpu, cols, group):
    """Whole numbers up to 112 in rows whose largest is 112: four times each is a quotient, up to what fp32 rounded before, and many
    lie halfway between two codes.  fp32's norm gives the values before the division; all of it has to be equal.  The oracle
    divides on the CPU, tensor by tensor: torch may take a division by a number as a product."""
    gen = torch.Generator().manual_seed(cols)
    x = torch.randint(-112, 113, (300, cols), generator=gen).float()
    x.view(300, -1, group or cols)[..., 0] = 112
    x = x * torch.rand((300, 1), generator=gen).exp()  # other sums of squares
    x, weight = x.to(gpu), torch.ones(cols, device=gpu)
    values = la.rms_norm(x, weight).view(300, -1, group or cols).cpu()
    codes, scales = (t.cpu() for t in la.rms_norm_e4m3(x, weight, group_size=group))
    assert torch.equal(scales, torch.div(values.abs().amax(-1), torch.full_like(scales, 448.0)))
    want = (values / scales[..., None]).to(torch.float8_e4m3fn).flatten(1)
    assert torch.equal(codes.float(), want.float())


def test_codes_of_what_is_not_finite(gpu):
    x = torch.ones(4, 64, device=gpu)
    weight = torch.ones(64, device=gpu)
    weight[5] = float("inf")
    codes, scales = la.rms_norm_e4m3(x, weight, group_size=32)
    assert torch.isinf(scales[:, 0]).all() and torch.isfinite(scales[:, 1]).all()
    first = codes[:, :32].float()
    assert torch.isnan(first[:, 5]).all() and (first[:, [c for c in range(32) if c != 5]] == 0).all()
    assert (codes[:, 32:].float() == 448).all()
    weight[5] = float("nan")
    codes, scales = la.rms_norm_e4m3(x, weight, group_size=32)
    assert torch.isnan(scales[:, 0]).all() and torch.isnan(codes[:, :32].float()).all() and (codes[:, 32:].float() == 448).all()
