"""Plain 64-bit counterparts of the paged 4-bit cache, on the CPU."""

from __future__ import annotations

import math

import torch

GROUP = 64


def held(keys: torch.Tensor, values: torch.Tensor):
    """(keys, values, key scales, value scales) in float64 as the cache holds [..., head_dim]; scales [..., groups]."""
    out = []
    for x in (keys, values):
        g = x.double().unflatten(-1, (-1, GROUP))
        low, high = g.amin(-1), g.amax(-1)
        size = torch.maximum((high - low) / 15, torch.maximum(low.abs(), high.abs()) / 120).float()
        scale = torch.where(size >= 2.0 ** -100, size, 0.0).bfloat16().double()
        step = torch.where(scale > 0, scale, 1.0)
        zero = torch.where(scale > 0, (low / step).round(), 0.0)
        code = ((g / step[..., None]).round() - zero[..., None]).clamp(0, 15)
        out += [((code + zero[..., None]) * scale[..., None]).flatten(-2), scale]
    (k, ks), (v, vs) = out[:2], out[2:]
    lost = ~(torch.isfinite(keys).all(-1) & torch.isfinite(values).all(-1))[..., None]
    return torch.where(lost, math.nan, k), torch.where(lost, 0.0, v), torch.where(lost, 0.0, ks), torch.where(lost, 0.0, vs)


def attention(query, keys, values, key_scale, value_scale, start, scaling, dtype, gate=None):
    """(out, tolerance), float64 [tokens, q_heads, head_dim]: query [tokens, q_heads, head_dim] at positions
    start.. over keys/values [length, kv_heads, head_dim] (float64, as held) with scales [length, kv_heads, groups].

    The tolerance counts the kernels' roundings, with u = half a step of the type and A = sum_t p_t |v_t|:
    - the output's own:  u |out|
    - probabilities (times the values' scales) and values rounded to the type for the second product:  2 u A
    - scores: keys rounded to the type in the tiles' form, each product q_d k_d off by u |q_d k_d| at most; the
      roundings are independent, so their sum stays within 4 u sqrt(sum (q_d k_d)^2) but for one case in 10^4
      (uniform errors: a deviation of u / sqrt(3) each, so this is 7 deviations), and the fp32 sums of whole codes,
      at most 16 roundings one after another of partial sums below 143 scale sum |q_d|; an error of e in
      scores moves every probability by less than 2 e of itself, and the output by 2 e A each way
    - the second product's fp32 sums, of whole codes below 143 times p scale, and of the offsets (below 256) that
      are taken off them: one rounding for every 16 tokens and 16 more to join the shares, of partial sums
      below 399 sum_t p_t scale_t (a value that is 0 is the difference of two such sums)
    - below the type's normal values a rounding is half a step of the subnormal ones: of the output, and of values
      rounded to the type, p of which sum to 1"""
    T, HQ, D = query.shape
    L, H, _ = keys.shape
    u, step = torch.finfo(dtype).eps / 2, torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    q = query.double()
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    for h in range(HQ):
        k, v = keys[:, h * H // HQ], values[:, h * H // HQ]
        score = scaling * (q[:, h] @ k.T)
        unseen = torch.arange(L)[None, :] > (start + torch.arange(T))[:, None]
        p = torch.softmax(score.masked_fill(unseen, -math.inf), -1)
        out[:, h] = p @ v
        size = p @ v.abs()
        e = scaling * (4 * u * torch.sqrt((q[:, h] ** 2) @ (k.T ** 2)).nan_to_num(0).masked_fill(unseen, 0).amax(-1)
                       + 16 * 2.0 ** -24 * 143 * float(key_scale.max() if key_scale.numel() else 0) * q[:, h].abs().sum(-1))
        sums = p @ value_scale[:, h * H // HQ].repeat_interleave(GROUP, -1)
        tol[:, h] = u * out[:, h].abs() + (2 * u + 4 * e[:, None]) * size + (16 + L / 16) * 2.0 ** -24 * 399 * sums + step
    if gate is not None:
        s = torch.sigmoid(gate.double())
        # fp32 sigmoid: far below half a step of the 16-bit types
        out, tol = out * s, tol * s + u * (out * s).abs() * 2.0 ** -4 + step
    return out, tol


class Mirror:
    """What every sequence holds, as dense float64 rows per layer."""

    def __init__(self):
        self.rows = {}  # seq -> [keys, values, key scales, value scales] of [length, kv_heads, ...]

    def store(self, seq, start, keys, values):
        new = held(keys, values)
        old = self.rows.get(seq)
        self.rows[seq] = list(new) if old is None or start == 0 else [torch.cat((o[:start], n)) for o, n in zip(old, new)]
