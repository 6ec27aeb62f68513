"""Plain 64-bit counterparts of the linear-attention operators, on the CPU, with what their kernels may be off by."""

from __future__ import annotations

import torch

EPS = 1e-6


def unit(x: torch.Tensor) -> torch.Tensor:
    return x / torch.sqrt((x * x).sum(-1, keepdim=True) + EPS)


def gates(decay, beta, a_log=None, dt_bias=None):
    decay, beta = decay.double(), beta.double()
    if a_log is None:
        return decay, beta
    x = decay + dt_bias.double()
    return -a_log.double().exp() * torch.logaddexp(x, torch.zeros_like(x)), torch.sigmoid(beta)


def delta_rule(q, k, v, g, beta, state, scaling, normalize=True, chunked=False):
    """One sequence: q, k [tokens, key_heads, dk], v [tokens, value_heads, dv], g and beta [tokens, value_heads] (as
    `gates` gives them), state [value_heads, dk, dv] -> (out, state, tolerance of out, of the state's columns' 2-norm).

    With unit keys, 0 <= beta <= 1 and g <= 0 a token's map of the state, e^g (1 - beta k k^T), makes no column longer, so an
    error's norm only ever decays, and a token adds at most c (|S| + |u| + beta |v|) of its column: c counts the fp32
    roundings (2^-24 each) of the products of a state's column with k and of the update: token by token at most 12 in
    a row for a sum, 2 for the update and some 16 of the factors' functions, c = 2^-19; in chunks sums of up to 192
    products, one after the other at worst, c = 2^-16.
    An output's error is scaling times its column's, its rounding to the type, c of the sum of its terms' sizes, and in
    chunks with bf16 outputs the roundings of one fp16 value an operand: two of 2^-11 of that sum."""
    q, k, v = q.double(), k.double(), v.double()
    if normalize:
        q, k = unit(q), unit(k)
    q = q * scaling
    HV = v.shape[1]
    q, k = (x.repeat_interleave(HV // x.shape[1], 1) for x in (q, k))
    S, out, c = state.double().clone(), torch.empty_like(v), 2.0 ** (-16 if chunked else -19)
    E, size = torch.zeros_like(S[:, 0]), S.abs()
    sums, errors = torch.zeros_like(out), torch.zeros_like(out)
    for t in range(v.shape[0]):
        e = torch.exp(g[t])[:, None]
        before = (S * e[..., None]).norm(dim=1)
        S = S * e[..., None]
        u = beta[t][:, None] * (v[t] - torch.einsum("hdn,hd->hn", S, k[t]))
        S = S + k[t][..., None] * u[:, None]
        out[t] = torch.einsum("hdn,hd->hn", S, q[t])
        E = E * e + c * (before + u.abs() + beta[t][:, None] * v[t].abs())
        size = size * e[..., None] + k[t].abs()[..., None] * u.abs()[:, None]
        sums[t], errors[t] = torch.einsum("hdn,hd->hn", size, q[t].abs()), E
    return out, S, sums, errors, E, c


def delta_tolerance(out, sums, errors, c, dtype, scaling, chunked):
    u = torch.finfo(dtype).eps / 2
    kappa = c + (2.0 ** -10 if chunked and dtype == torch.bfloat16 else 0.0)
    step = torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    return u * out.abs() + (1 + u) * (kappa * sums + scaling * errors) + step


def conv(x, weight, bias, state, silu):
    """One sequence: x [tokens, channels], state [width - 1, channels] -> (out, new state, sums of the terms' sizes)."""
    W, n = weight.shape[1], x.shape[0]
    rows = torch.cat((state, x))
    wide, w = rows.double(), weight.double()
    y = sum(wide[j:j + n] * w[:, j] for j in range(W))
    size = sum((wide[j:j + n] * w[:, j]).abs() for j in range(W))
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    return y * torch.sigmoid(y) if silu else y, rows[n:], size


def norm(x, weight, eps, offset, residual=None, gate=None):
    """-> (values, new residual)"""
    if residual is not None:
        residual = (x.float() + residual.float()).to(x.dtype)
        x = residual
    h = x.double()
    y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * (weight.double() + offset)
    if gate is not None:
        y = y * gate.double() * torch.sigmoid(gate.double())
    return y, residual
