"""The gated delta rule in chunks where an operand's size, or what is left of a sum, is far from its neighbours': against the
64-bit counterpart (tests/_linear.py)."""

import pytest
import torch

import _linear as plain
from anna_amd import linear_attention as la

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def randn(seed, *shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed))


def run(gpu, q, k, v, g, beta, state, scaling, normalize=True):
    """One sequence of one key head on the device -> (out, state)."""
    pool = state[None].to(gpu)
    out = la.gated_delta_rule(q.to(gpu), k.to(gpu), v.to(gpu), g.to(gpu), beta.to(gpu), pool, la.StateSpan([0], [len(q)], device=gpu),
                              scaling=scaling, normalize=normalize)
    return out.cpu(), pool[0].cpu()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("DV", [32, 128])
@pytest.mark.parametrize("heads", [2, 320])
def test_outputs_whose_terms_cancel(gpu, heads, DV, dtype):
    """A query sees pairs of rows of the state (even heads), or pairs of the chunk's own updates (odd ones), that cancel to
    2^-8 of their size.  The operands enter the products with 22 bits, off by 2^-22 of themselves at most and two of them in a
    product of the chunk's own; a sum has 32 products an instruction and up to 12 instructions in a row, 44 roundings of
    2^-24 of a partial sum: 2^-21 + 44 * 2^-24 < 2^-18 of the sum of the terms' sizes, beside the type's own rounding.
    320 heads go with more than one group of columns a workgroup."""
    DK, n = 64, 64
    r, left = randn(1, DK // 2, heads, DV), 2.0 ** -8 * randn(2, DK // 2, heads, DV)
    state = torch.zeros(heads, DK, DV)
    state[0::2, 0::2], state[0::2, 1::2] = r[:, 0::2].movedim(1, 0), (left - r)[:, 0::2].movedim(1, 0)
    k, v = torch.zeros(n, heads, DK), torch.zeros(n, heads, DV)
    beta, g = torch.zeros(n, heads), torch.zeros(n, heads)
    for t in range(32):  # odd heads: token t writes row t
        k[t, 1::2, t] = 1
    v[0:32:2, 1::2], v[1:32:2, 1::2] = r[:16, 1::2], (left - r)[:16, 1::2]
    beta[:32] = 0.7  # updates have more bits than the type
    q = randn(3, n, heads, DK // 2).abs().repeat_interleave(2, 2)
    q, k, v = q.to(dtype), k.to(dtype), v.to(dtype)
    out, after = run(gpu, q, k, v, g, beta, state, 1.0)
    want, S, sums, *_ = plain.delta_rule(q, k, v, g.double(), beta.double(), state, 1.0)
    assert float((want[32:].abs() / sums[32:]).median()) < 2.0 ** -6  # they do cancel
    u = torch.finfo(dtype).eps / 2
    tol = u * want.abs() + (1 + u) * 2.0 ** -18 * sums + torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    off = (out.double() - want).abs()
    assert (off <= tol).all(), float((off / tol).max())
    assert ((after.double() - S).norm(dim=1) <= 2.0 ** -18 * S.norm(dim=1)).all()


def check(out, state, q, k, v, g, beta, S0, scaling, normalize=True):
    """The bounds of tests/_linear.py for the chunks' form, without its allowance for outputs of fewer bits."""
    want, S, sums, errors, E, c = plain.delta_rule(q, k, v, g.double(), beta.double(), S0, scaling, normalize, chunked=True)
    size = 1.0 if normalize else float(q.double().norm(dim=-1).max())
    tol = plain.delta_tolerance(want, sums, errors, c, out.dtype, scaling * size, False)
    off = (out.double() - want).abs()
    assert torch.isfinite(out).all() and (off <= tol).all(), float((off / tol).max())
    off = (state.double() - S).norm(dim=1)
    assert torch.isfinite(state).all() and (off <= E).all(), float((off / E).max())


def sequence(seed, n, heads, DK, DV, dtype=BF):
    q, k, v = randn(seed, n, heads, DK).to(dtype), randn(seed + 1, n, heads, DK).to(dtype), randn(seed + 2, n, heads, DV).to(dtype)
    g, beta = -0.4 * torch.rand((n, heads), generator=torch.Generator().manual_seed(seed + 3)), torch.sigmoid(randn(seed + 4, n, heads))
    return q, k, v, g, beta, 0.5 * randn(seed + 5, heads, DK, DV)


# heads of 4 groups of columns a workgroup from 256 on, at 64 columns
@pytest.mark.parametrize("heads", [2, 320])
@pytest.mark.parametrize("power", [104, 110, 118])
def test_values_that_no_unit_brings_into_fp16s_range(gpu, power, heads):
    """Every chunk's products overflow; the state is finite all the time."""
    q, k, v, g, beta, S = sequence(11, 260, heads, 64, 64)
    v, S = (v.float() * 2.0 ** power).to(BF), S * 2.0 ** power
    out, after = run(gpu, q, k, v, g, beta, S, 0.125)
    check(out, after, q, k, v, g, beta, S, 0.125)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("heads", [2, 320])
@pytest.mark.parametrize("length,beta", [(2.0 ** -5, 900.0), (2.0 ** -10, 2.0 ** 19)])
def test_updates_beyond_fp16s_range(gpu, length, beta, heads, dtype):
    """Short keys with a large beta, beta |k|^2 < 1: an update is of a thousand times the values' size, its part of the state is
    not.  With k' = k / length, beta' = beta length^2 and v' = v / length the states are the same and keys are (nearly) unit ones,
    so the bounds hold in these terms."""
    q, k, v, g, _, S = sequence(31, 200, heads, 64, 64, dtype)
    k = (k.float() / k.float().norm(dim=-1, keepdim=True) * length * 0.98).to(dtype)
    q = (q.float() / 8).to(dtype)
    beta = torch.full_like(g, beta)
    out, after = run(gpu, q, k, v, g, beta, S, 1.0, normalize=False)
    for h in range(0, heads, 16):  # the same rule in unit keys' terms
        at = slice(h, h + 16)
        want, end, sums, errors, E, c = plain.delta_rule(q[:, at], k[:, at].double() / length, v[:, at].double() / length,
                                                         g[:, at].double(), beta[:, at].double() * length ** 2, S[at], 1.0, False, chunked=True)
        tol = plain.delta_tolerance(want, sums, errors, c, dtype, float(q.double().norm(dim=-1).max()), False)
        assert torch.isfinite(out[:, at]).all() and ((out[:, at].double() - want).abs() <= tol).all()
        assert ((after[at].double() - end).norm(dim=1) <= E).all()
