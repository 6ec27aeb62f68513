"""What is timed of the linear-attention operators (anna_amd.linear_attention), and their plain forms.

Kinds of case
  delta  the gated delta rule over ragged sequences that continue their states: single tokens, drafted
         tokens, prompts, prompts of long documents
  conv   the short causal convolution in front of it, with the last inputs kept in a state
  norm   the root-mean-square norms around it: with the residual's addition, with a gate, with an
         output in e4m3 and its scales

With q^ = scaling q / sqrt(|q|^2 + 1e-6), k^ = k / sqrt(|k|^2 + 1e-6), a state S [key_dim, value_dim] of
every value head takes a token by
  u = beta (v - e^g S^T k^),   S <- e^g S + k^ u^T,   out = S^T q^
where g = -exp(a_log) softplus(a + dt_bias) and beta = sigmoid(b), or both are given.

`own` chooses between the plain form (elementary torch operations in 32 bits, the sums of logarithms of
decays in 64) and the framework's calls.  Head counts are 16 key and 32 value heads of 128 and generic
ones, hidden sizes 2048 and 4096 as in this repository's benchmark and tests; draw() takes the ranges
around them.
"""

import math
import random

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-6
E4M3_MAX = 448.0


def listed():
    return [
        # the smallest call: one sequence's next token, where latency counts
        dict(name="delta_one", kind="delta", batch=1, key_heads=16, value_heads=32, key_dim=128, value_dim=128,
             dtype="bf16", min_len=1, max_len=1, fresh=False, gates="raw", ragged=0),
        # a decode step of a large batch
        dict(name="delta_batch", kind="delta", batch=64, key_heads=16, value_heads=32, key_dim=128, value_dim=128,
             dtype="bf16", min_len=1, max_len=1, fresh=False, gates="raw", ragged=1),
        # one to six drafted tokens a sequence, small heads, decays and betas given
        dict(name="delta_draft", kind="delta", batch=24, key_heads=8, value_heads=16, key_dim=64, value_dim=128,
             dtype="fp16", min_len=1, max_len=6, fresh=False, gates="given", ragged=2),
        # short prompts of ragged length, one token among them, with new states
        dict(name="delta_prompts", kind="delta", batch=5, key_heads=16, value_heads=32, key_dim=128, value_dim=128,
             dtype="bf16", min_len=1, max_len=1500, fresh=True, gates="raw", ragged=3),
        # a long document of one sequence: the chain of states counts
        dict(name="delta_long", kind="delta", batch=1, key_heads=16, value_heads=32, key_dim=128, value_dim=128,
             dtype="bf16", min_len=16384, max_len=16384, fresh=True, gates="raw", ragged=4),
        # a batch of prompts' chunks that go on from earlier ones
        dict(name="delta_chunks", kind="delta", batch=8, key_heads=16, value_heads=32, key_dim=128, value_dim=128,
             dtype="fp16", min_len=1024, max_len=4096, fresh=False, gates="given", ragged=5),
        # the decode step's tokens through the convolution
        dict(name="conv_step", kind="conv", batch=64, channels=8192, width=4, dtype="bf16", bias=False, silu=True,
             min_len=1, max_len=1, fresh=False, ragged=6),
        # ragged prompts through it
        dict(name="conv_prompts", kind="conv", batch=6, channels=8192, width=4, dtype="bf16", bias=True, silu=True,
             min_len=1, max_len=4000, fresh=True, ragged=7),
        # a decode step's hidden states, added to the residual stream and normalised
        dict(name="norm_step", kind="norm", rows=64, cols=2048, dtype="bf16", residual=True, gate=False, offset=1.0,
             group=0),
        # a prompt's, leaving as e4m3 with a scale for every 128 columns
        dict(name="norm_prompt_e4m3", kind="norm", rows=8192, cols=4096, dtype="bf16", residual=True, gate=False,
             offset=1.0, group=128),
        # the same for a few rows, one scale a row
        dict(name="norm_step_e4m3", kind="norm", rows=7, cols=4096, dtype="fp16", residual=False, gate=False, offset=0.0,
             group=4096),
        # the heads' outputs of a prompt, gated
        dict(name="norm_gated", kind="norm", rows=8192 * 32, cols=128, dtype="bf16", residual=False, gate=True, offset=0.0,
             group=0),
    ]


# ---------------------------------------------------------------- draw


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


HEADS = ((16, 32), (16, 32), (16, 16), (8, 32), (4, 12), (2, 2), (1, 3))


def draw(rng):
    kind = rng.choice(("delta", "delta", "delta", "conv", "norm"))
    c = dict(kind=kind, dtype=rng.choice(("bf16", "bf16", "fp16")), ragged=rng.randrange(1 << 30))
    if kind == "delta":
        c["key_heads"], c["value_heads"] = rng.choice(HEADS)
        c.update(key_dim=rng.choice((64, 128, 128)), value_dim=rng.choice((32, 64, 96, 128, 128, 256)),
                 fresh=rng.random() < 0.5, gates=rng.choice(("raw", "given")))
        form = rng.choice(("step", "draft", "prompt", "prompt"))
        c["max_len"] = {"step": 1, "draft": rng.randint(2, 12), "prompt": _log(rng, 13, 16384)}[form]
        c["min_len"] = 1 if form == "step" else rng.randint(1, c["max_len"])
        most = min(128, (1 << 31) // (c["value_heads"] * c["key_dim"] * c["value_dim"]),
                   (1 << 33) // (c["max_len"] * c["value_heads"] * c["key_dim"] * c["value_dim"]))
        c["batch"] = _log(rng, 1, max(1, most))
    elif kind == "conv":
        c.update(channels=8 * _log(rng, 8, 1536), width=rng.choice((2, 3, 4, 4)), bias=rng.random() < 0.5,
                 silu=rng.random() < 0.8, fresh=rng.random() < 0.5, max_len=_log(rng, 1, 8192))
        c["min_len"] = rng.randint(1, c["max_len"])
        c["batch"] = _log(rng, 1, max(1, min(128, (1 << 26) // (c["max_len"] * c["channels"]))))
    else:
        gate = rng.random() < 0.4
        cols = rng.choice((64, 128, 256)) if gate else 8 * _log(rng, 16, 1536)
        c.update(cols=cols, rows=_log(rng, 1, min(1 << 18, (1 << 25) // cols)), gate=gate, residual=not gate and rng.random() < 0.6,
                 offset=rng.choice((0.0, 1.0)), group=0 if gate else rng.choice((0, 0, cols, 128)))
        c["dtype"] = rng.choice(("bf16", "bf16", "fp16", "fp32"))
        if c["group"] == 128:
            c["cols"] = 128 * max(1, cols // 128)
    return c


# ---------------------------------------------------------------- shapes and work


def _lengths(case):
    r = random.Random(case["ragged"])
    lens = [r.randint(case["min_len"], case["max_len"]) for _ in range(case["batch"])]
    lens[0] = case["max_len"]
    if case["batch"] > 1:
        lens[-1] = case["min_len"]
    return lens


def _slots(case):
    """The states' rows of the sequences: some of a larger pool, in no order."""
    return random.Random(case["ragged"] + 1).sample(range(case["batch"] + 3), case["batch"])


def work(case):
    size = SIZES[case["dtype"]]
    if case["kind"] == "norm":
        n = case["rows"] * case["cols"]
        out = n * size if not case["group"] else n + 4 * case["rows"] * (case["cols"] // case["group"])
        return {"bytes": n * size * (1 + 2 * case["residual"] + case["gate"]) + out + case["cols"] * size, "flops": 0}
    tokens = sum(_lengths(case))
    if case["kind"] == "conv":
        kept = case["batch"] * (case["width"] - 1) * case["channels"] * size
        return {"bytes": 2 * tokens * case["channels"] * size + kept * (1 if case["fresh"] else 2)
                + case["channels"] * (case["width"] + case["bias"]) * size,
                "flops": 2 * tokens * case["channels"] * case["width"]}
    HK, HV, DK, DV = (case[x] for x in ("key_heads", "value_heads", "key_dim", "value_dim"))
    gates = 4 if case["gates"] == "given" else size
    return {"bytes": tokens * (2 * HK * DK * size + 2 * HV * DV * size + 2 * HV * gates)
            + case["batch"] * HV * DK * DV * 4 * (1 if case["fresh"] else 2),
            "flops": 6 * tokens * HV * DK * DV}


# ---------------------------------------------------------------- inputs


def _draw_inputs(case, gen):
    """The tensors that a program has in hand before the call."""
    def normal(*shape):
        return torch.randn(shape, device=DEVICE, generator=gen)

    dtype = DTYPES[case["dtype"]]
    if case["kind"] == "norm":
        rows, cols = case["rows"], case["cols"]
        wide = torch.where(torch.rand(cols, device=DEVICE, generator=gen) < 0.01, 8.0, 1.0)  # a few large channels
        return dict(x=(normal(rows, cols) * wide).to(dtype),
                    weight=(0.2 * normal(cols) + 1 - case["offset"]).to(dtype),
                    residual=(3 * normal(rows, cols) * wide).to(dtype) if case["residual"] else None,
                    gate=normal(rows, cols).to(dtype) if case["gate"] else None)
    tokens, pool = sum(_lengths(case)), case["batch"] + 3
    if case["kind"] == "conv":
        ch, width = case["channels"], case["width"]
        return dict(x=normal(tokens, ch).to(dtype), weight=(normal(ch, width) * width ** -0.5).to(dtype),
                    bias=(0.1 * normal(ch)).to(dtype) if case["bias"] else None,
                    state=normal(pool, width - 1, ch).to(dtype))
    HK, HV, DK, DV = (case[x] for x in ("key_heads", "value_heads", "key_dim", "value_dim"))
    # what leaves the convolution: one row of queries, keys and values a token
    mixed = torch.nn.functional.silu(normal(tokens, 2 * HK * DK + HV * DV)).to(dtype)
    s = dict(mixed=mixed, state=0.3 * normal(pool, HV, DK, DV), scaling=DK ** -0.5)
    a, b = normal(tokens, HV), normal(tokens, HV)
    a_log = torch.log(1 + 15 * torch.rand(HV, device=DEVICE, generator=gen))
    dt = torch.exp(torch.rand(HV, device=DEVICE, generator=gen) * math.log(100) + math.log(0.001))
    dt_bias = dt + torch.log(-torch.expm1(-dt))  # softplus gives dt
    if case["gates"] == "raw":
        s.update(decay=a.to(dtype), beta=b.to(dtype), a_log=a_log, dt_bias=dt_bias)
    else:
        s.update(decay=-torch.exp(a_log) * torch.nn.functional.softplus(a + dt_bias), beta=torch.sigmoid(b),
                 a_log=None, dt_bias=None)
    return s


def _heads(case, mixed):
    HK, HV, DK, DV = (case[x] for x in ("key_heads", "value_heads", "key_dim", "value_dim"))
    q, k, v = mixed.split((HK * DK, HK * DK, HV * DV), -1)
    return q.unflatten(-1, (HK, DK)), k.unflatten(-1, (HK, DK)), v.unflatten(-1, (HV, DV))


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    s = dict(case=case, **_draw_inputs(case, gen))
    if case["kind"] == "norm":
        return s
    lens, slots = _lengths(case), _slots(case)
    if own:
        from anna_amd.linear_attention import StateSpan

        s["span"] = StateSpan(slots, lens, fresh=[case["fresh"]] * len(lens), device=DEVICE)
        return s
    s["slots"] = torch.tensor(slots, device=DEVICE)
    length, start = (torch.tensor(x, device=DEVICE) for x in (lens, [sum(lens[:i]) for i in range(len(lens))]))
    seq = torch.repeat_interleave(torch.arange(len(lens), device=DEVICE), length)
    position = torch.arange(sum(lens), device=DEVICE) - start[seq]
    if case["kind"] == "conv":
        # rows of (states, inputs): of every output's taps, and of the inputs that the states keep
        W, B = case["width"], len(lens)
        tap = torch.arange(W - 1, -1, -1, device=DEVICE)

        def rows(seq, back):
            return torch.where(back >= 0, B * (W - 1) + start[seq] + back, seq * (W - 1) + (W - 1) + back)

        s["taps"] = rows(seq[:, None], position[:, None] - tap)
        s["kept"] = rows(torch.arange(B, device=DEVICE)[:, None], length[:, None] - tap[:-1])
        return s
    # the padded batch's places of the tokens
    s["chunk"] = min(64, 1 << (max(lens) - 1).bit_length())
    s["padded"] = -(-max(lens) // s["chunk"]) * s["chunk"]
    s["at"] = seq * s["padded"] + position
    return s


# ---------------------------------------------------------------- the plain forms


def _plain_norm(s):
    case, x = s["case"], s["x"].float()
    if s["residual"] is not None:
        s["residual"].copy_(x + s["residual"].float())
        x = s["residual"].float()
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * (s["weight"].float() + case["offset"])
    if s["gate"] is not None:
        gate = s["gate"].float()
        y = y * (gate * torch.sigmoid(gate))
    out = {} if s["residual"] is None else {"residual": s["residual"]}
    if not case["group"]:
        return {"out": y.to(s["x"].dtype), **out}
    y = y.unflatten(-1, (-1, case["group"]))
    scale = y.abs().amax(-1) / E4M3_MAX
    codes = (y / torch.where(scale > 0, scale, 1.0)[..., None]).clamp(-E4M3_MAX, E4M3_MAX)
    return {"out": codes.flatten(-2).to(torch.float8_e4m3fn), "scales": scale, **out}


def _plain_conv(s):
    state = s["state"][s["slots"]]
    if s["case"]["fresh"]:
        state = torch.zeros_like(state)
    rows = torch.cat((state.flatten(0, 1), s["x"]))
    y = (rows[s["taps"]].float() * s["weight"].float().T).sum(1)
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if s["case"]["silu"]:
        y = y * torch.sigmoid(y)
    s["state"][s["slots"]] = rows[s["kept"]]
    return {"out": y.to(s["x"].dtype), "state": s["state"]}


def _plain_inverse(A):
    """(1 + A)^-1 of strictly lower triangular A [..., C, C], from its diagonal blocks to ever larger ones."""
    C = A.shape[-1]
    T = torch.zeros_like(A)
    T.diagonal(0, -2, -1).fill_(1.0)
    half = 1
    while half < C:
        shape = (C // (2 * half), 2 * half, C // (2 * half), 2 * half)
        a, t = (x.unflatten(-1, shape[2:]).unflatten(-3, shape[:2]).diagonal(0, -4, -2).movedim(-1, -3) for x in (A, T))
        low, high = t[..., :half, :half].contiguous(), t[..., half:, half:].contiguous()
        t[..., half:, :half] = -torch.matmul(torch.matmul(high, a[..., half:, :half].contiguous()), low)
        half *= 2
    return T


def _plain_delta(s):
    case, B, L, C = s["case"], s["case"]["batch"], s["padded"], s["chunk"]
    HK, HV = case["key_heads"], case["value_heads"]
    q, k, v = (x.float() for x in _heads(case, s["mixed"]))
    q, k = (x * torch.rsqrt(x.square().sum(-1, keepdim=True) + EPS) for x in (q, k))
    g, beta = s["decay"].float(), s["beta"].float()
    if s["a_log"] is not None:
        x = g + s["dt_bias"]
        g = -torch.exp(s["a_log"]) * (x.clamp(min=0) + torch.log1p(torch.exp(-x.abs())))
        beta = torch.sigmoid(beta)

    def batch(x):  # [tokens, heads, ...] -> [chunks, batch, value heads, C, ...], zeros where there is no token
        p = x.new_zeros((B * L, *x.shape[1:])).index_copy_(0, s["at"], x).unflatten(0, (B, L // C, C))
        p = p.movedim(0, 1).movedim(3, 2)
        return p.repeat_interleave(HV // p.shape[2], 2) if p.shape[2] != HV else p

    q, k, v, beta = batch(q * s["scaling"]), batch(k), batch(v), batch(beta)[..., None]
    a = batch(g.double()).cumsum(-1)
    later = torch.ones((C, C), dtype=torch.bool, device=DEVICE).triu(1)
    decay = torch.exp((a[..., :, None] - a[..., None, :]).masked_fill_(later, -math.inf)).float()
    kt = k.transpose(-1, -2).contiguous()
    seen = torch.matmul(q, kt) * decay
    T = _plain_inverse((torch.matmul(k, kt) * decay * beta).tril_(-1))
    first, last = torch.exp(a)[..., None].float(), torch.exp(a[..., -1:] - a)[..., None].float()
    kt, end = (k * last).transpose(-1, -2).contiguous(), first[..., -1:, :]
    S = s["state"][s["slots"]]
    if case["fresh"]:
        S = torch.zeros_like(S)
    out = torch.empty_like(v)
    for n in range(L // C):
        U = torch.matmul(T[n], beta[n] * (v[n] - first[n] * torch.matmul(k[n], S)))
        out[n] = first[n] * torch.matmul(q[n], S) + torch.matmul(seen[n], U)
        S = end[n] * S + torch.matmul(kt[n], U)
    s["state"][s["slots"]] = S
    out = out.movedim(2, 3).movedim(1, 0).flatten(0, 2)[s["at"]]
    return {"out": out.to(s["mixed"].dtype), "state": s["state"]}


# ---------------------------------------------------------------- run


def run(s):
    if not own:
        return {"norm": _plain_norm, "conv": _plain_conv, "delta": _plain_delta}[s["case"]["kind"]](s)
    from anna_amd import linear_attention as la

    case = s["case"]
    if case["kind"] == "norm":
        more = {} if s["residual"] is None else {"residual": s["residual"]}
        if case["group"]:
            out, scales = la.rms_norm_e4m3(s["x"], s["weight"], eps=EPS, weight_offset=case["offset"],
                                           residual=s["residual"], group_size=case["group"])
            return {"out": out, "scales": scales, **more}
        return {"out": la.rms_norm(s["x"], s["weight"], eps=EPS, weight_offset=case["offset"], residual=s["residual"],
                                   gate=s["gate"]), **more}
    if case["kind"] == "conv":
        out = la.causal_conv1d(s["x"], s["weight"], s["bias"], s["state"], s["span"],
                               activation="silu" if case["silu"] else None)
    else:
        q, k, v = _heads(case, s["mixed"])
        out = la.gated_delta_rule(q, k, v, s["decay"], s["beta"], s["state"], s["span"], scaling=s["scaling"],
                                  a_log=s["a_log"], dt_bias=s["dt_bias"])
    return {"out": out, "state": s["state"]}


# ---------------------------------------------------------------- the definitions in 64 bits


def exact(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    s = {n: t.double() if isinstance(t, torch.Tensor) and n != "mixed" else t for n, t in _draw_inputs(case, gen).items()}
    if case["kind"] == "norm":
        h, out = s["x"], {}
        if case["residual"]:
            h = (h + s["residual"]).to(DTYPES[case["dtype"]]).double()
            out["residual"] = h
        y = h / (h.pow(2).sum(-1, keepdim=True) / case["cols"] + EPS).sqrt() * (s["weight"] + case["offset"])
        if case["gate"]:
            y = y * s["gate"] / (1 + torch.exp(-s["gate"]))
        if case["group"]:
            parts = y.view(case["rows"], -1, case["group"])
            out["scales"] = parts.abs().max(-1)[0] / E4M3_MAX
            y = (parts / out["scales"][..., None]).view_as(y)
        return {"out": y, **out}
    lens, slots = _lengths(case), _slots(case)
    if case["kind"] == "conv":
        W, start, state = case["width"], 0, s["state"].clone()
        out = torch.empty_like(s["x"])
        for n, slot in zip(lens, slots):
            old = torch.zeros_like(state[slot]) if case["fresh"] else state[slot]
            x = torch.cat((old, s["x"][start:start + n]))
            y = sum(x[j:j + n] * s["weight"][:, j] for j in range(W))
            if case["bias"]:
                y = y + s["bias"]
            out[start:start + n] = y / (1 + torch.exp(-y)) if case["silu"] else y
            state[slot] = x[n:]
            start += n
        return {"out": out, "state": state}
    B, HV, most = case["batch"], case["value_heads"], max(lens)
    q, k, v = (x.double() for x in _heads(case, s["mixed"]))
    q, k = (x / (x.pow(2).sum(-1, keepdim=True) + EPS).sqrt() for x in (q, k))
    q, k = ((x * f).repeat_interleave(HV // case["key_heads"], 1) for x, f in ((q, s["scaling"]), (k, 1.0)))
    g, beta = s["decay"], s["beta"]
    if case["gates"] == "raw":
        x = g + s["dt_bias"]
        g, beta = -s["a_log"].exp() * torch.logaddexp(x, torch.zeros_like(x)), 1 / (1 + torch.exp(-beta))
    state = s["state"].clone()
    S = torch.zeros_like(state[slots]) if case["fresh"] else state[slots]
    out = torch.empty_like(v)
    order = sorted(range(B), key=lambda b: -lens[b])  # those that still have tokens come first
    S = S[order].contiguous()
    first = torch.tensor([sum(lens[:b]) for b in order], device=DEVICE)
    going = B
    for t in range(most):
        while lens[order[going - 1]] <= t:
            going -= 1
        row, P = first[:going] + t, S[:going]
        kt = k[row].unsqueeze(-1)
        P.mul_(g[row].exp()[..., None, None])
        P.add_(kt * (beta[row].unsqueeze(-1) * (v[row] - (P * kt).sum(-2))).unsqueeze(-2))
        out[row] = (P * q[row].unsqueeze(-1)).sum(-2)
    state[torch.tensor([slots[b] for b in order], device=DEVICE)] = S
    return {"out": out, "state": state}
