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


# what: (powers of two, how the inputs get them)
def outlier(c, p):  # a value that comes late: the tokens in front of it do not know it
    c["S"][:] = 0
    c["v"][50, :, 3] = 2.0 ** p
    c["v"][90, :, 5] = -(2.0 ** p)


def outlier_on_a_state(c, p):
    c["v"][50, 0, 3] = 2.0 ** p
    c["g"][:] = c["g"] * 20  # nothing of the state is left at the chunk's end


def forgotten_state(c, p):
    c["S"][:, :, 3] *= 2.0 ** p
    c["g"][4] = -100.0


def forgotten_value(c, p):
    c["v"][20, :, 3] = 2.0 ** p
    c["g"][25] = -70.0
    c["g"][100] = float("-inf")


def faint_state(c, p):
    c["S"][:] *= 2.0 ** -p
    c["v"][:40] = 0
    c["v"][70:100] = 0


def small_betas(c, p):
    c["S"][:] = 0
    c["beta"][:40] *= 2.0 ** -p
    c["beta"][70:] *= 2.0 ** -p


def small_columns(c, p):  # in front of, and beside others
    c["S"][:, :, ::2] *= 2.0 ** -p
    c["v"][:, :, ::2] *= 2.0 ** -p
    c["v"][:, :, 1::2] *= 2.0 ** (p // 4)


RANGES = [outlier, outlier_on_a_state, forgotten_state, forgotten_value, faint_state, small_betas, small_columns]


@pytest.mark.parametrize("heads,DK,DV", [(2, 64, 64), (1, 128, 96), (160, 128, 64)])
@pytest.mark.parametrize("power", [8, 14, 18, 22, 26, 34, 48, 90, 110])
@pytest.mark.parametrize("what", RANGES, ids=lambda f: f.__name__)
def test_sizes_far_apart_in_a_column(gpu, what, power, heads, DK, DV):
    """A token's answer is as exact as what it sees allows, whatever else its chunk holds.  (160 heads go with four groups
    of columns a workgroup.)"""
    q, k, v, g, beta, S = sequence(100 + power, 150, heads, DK, DV)
    c = dict(v=v.float(), g=g, beta=beta, S=S)
    what(c, power)
    v = c["v"].to(BF)
    out, after = run(gpu, q, k, v, g, beta, S, 0.1)
    check(out, after, q, k, v, g, beta, S, 0.1)


@pytest.mark.parametrize("power", [6, 10, 13])
def test_sizes_far_apart_in_fp16(gpu, power):
    q, k, v, g, beta, S = sequence(200 + power, 150, 2, 128, 64, HF)
    v[:] = (v.float() * 2.0 ** -12).to(HF)
    S[:] = 0
    v[50, :, 3] = 2.0 ** power
    v[100, 1, ::2] = -(2.0 ** power)
    g[::30] = -25
    out, after = run(gpu, q, k, v, g, beta, S, 0.1)
    check(out, after, q, k, v, g, beta, S, 0.1)


@pytest.mark.parametrize("heads", [2, 320])
@pytest.mark.parametrize("length,beta", [(3000.0, 0.5), (2.0 ** 40, 0.9), (2.0 ** -40, 0.5), (2.0 ** 12, 2.0 ** -30)])
def test_keys_of_any_length(gpu, length, beta, heads):
    """beta |k|^2 below 1, and each of them far from 1: the bounds hold in the terms of unit keys (v' = v / length)."""
    q, k, v, g, _, S = sequence(41, 200, heads, 64, 64)
    k = (k.float() / k.float().norm(dim=-1, keepdim=True) * length * 0.98).to(BF)
    v, q = (v.float() * length ** 0.5).to(BF), (q.float() / 8).to(BF)
    beta = torch.full_like(g, beta / length ** 2)
    out, after = run(gpu, q, k, v, g, beta, S, 1.0, normalize=False)
    want, end, sums, errors, E, c = plain.delta_rule(q, k.double() / length, v.double() / length, g.double(), beta.double() * length ** 2, S, 1.0, False,
                                                     chunked=True)
    tol = plain.delta_tolerance(want, sums, errors, c, BF, float(q.double().norm(dim=-1).max()), False)
    assert torch.isfinite(out).all() and ((out.double() - want).abs() <= tol).all()
    assert ((after.double() - end).norm(dim=1) <= E).all()


@pytest.mark.parametrize("heads", [2, 320])
def test_a_state_that_grows(gpu, heads):
    """The same key again and again with beta 2.5: the state turns round and grows by 1.5 a token, 2^117 in all.  What a token
    adds to the error, in the state's terms of then, is some 16 roundings of 2^-24 of the key's and beta's factors and those
    of a product with the state, 2^-18 of the column's 2-norm at most; all of it grows on by 1.5 a token: after t tokens
    t 2^-18 of 1.5^t of the first state's 2-norm."""
    n = 200
    q, k, v, g, _, S = sequence(51, n, heads, 64, 64)
    k[:] = k[:1]
    q[:] = k  # what grows
    v[:], g[:] = 0, 0
    beta = torch.full_like(g, 2.5)
    out, after = run(gpu, q, k, v, g, beta, S, 1.0)
    want, end, *_ = plain.delta_rule(q, k, v, g.double(), beta.double(), S, 1.0, chunked=True)
    assert torch.isfinite(out).all() and torch.isfinite(after).all()
    t = torch.arange(1, n + 1)[:, None, None].double()
    grown = S.double().norm(dim=1) * 1.5 ** t
    assert ((out.double() - want).abs() <= 2.0 ** -8 * want.abs() + t * 2.0 ** -18 * grown).all()
    assert ((after.double() - end).norm(dim=1) <= n * 2.0 ** -18 * grown[-1]).all()


@pytest.mark.parametrize("DK,dtype,power", [(64, BF, 14), (64, BF, 22), (64, BF, 34), (128, BF, 14), (128, BF, 22), (128, BF, 34), (128, HF, 14)])
@pytest.mark.parametrize("what", RANGES, ids=lambda f: f.__name__)
def test_sizes_far_apart_with_two_groups_of_columns(gpu, what, DK, dtype, power):
    """The forms that take columns that four groups do not divide."""
    q, k, v, g, beta, S = sequence(300 + power, 140, 100, DK, 96, dtype)
    c = dict(v=v.float(), g=g, beta=beta, S=S)
    what(c, power)
    v = c["v"].to(dtype)
    out, after = run(gpu, q, k, v, g, beta, S, 0.1)
    check(out, after, q, k, v, g, beta, S, 0.1)


@pytest.mark.parametrize("DV", [32, 128])
def test_a_chunk_by_tokens_between_others(gpu, DV):
    """Chunks go token by token and in products in turn, of ragged sequences in one call, one of them of nobody: what is beside
    them, and the next chunk, is as without."""
    counts, DK, heads = [200, 13, 64, 65, 300], 128, 4
    n = sum(counts)
    q, k, v, g, beta, _ = sequence(61, n, heads, DK, DV)
    S = 0.5 * randn(66, len(counts) + 1, heads, DK, DV)
    first = [sum(counts[:i]) for i in range(len(counts))]
    for at, p in ((first[0] + 70, 40), (first[2] + 5, 30), (first[3] + 64, 60), (first[4] + 130, 25)):
        v[at, 1, 7] = 2.0 ** p
        g[at + 1:at + 2, 1] = -80.0
    slots = [3, 0, 5, -1, 2]
    pool = S.to(gpu)
    out = la.gated_delta_rule(*(t.to(gpu) for t in (q, k, v, g, beta)), pool, la.StateSpan(slots, counts, fresh=[False, True, False, False, True], device=gpu),
                              scaling=0.1).cpu()
    for slot, at, m, fresh in zip(slots, first, counts, [False, True, False, False, True]):
        rows = slice(at, at + m)
        if slot < 0:
            assert (out[rows] == 0).all()
            continue
        start = torch.zeros_like(S[slot]) if fresh else S[slot]
        check(out[rows], pool[slot].cpu(), q[rows], k[rows], v[rows], g[rows], beta[rows], start, 0.1)
    for slot in (1, 4):
        assert torch.equal(pool[slot].cpu(), S[slot])
