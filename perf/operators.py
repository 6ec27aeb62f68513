"""What is timed of the paged 4-bit KV cache (anna_amd.paged_cache.PagedInt4Cache), and its plain form.

Kinds of case
  attend  attention of new tokens over the cached pages: single tokens, drafted tokens, prompts, prompt chunks
  store   new tokens of ragged sequences quantized into their pages, and read back dense
  fork    sequences that share their parents' pages, their partly filled last pages copied when they grow
  resize  the live pages of a fragmented pool gathered at the front of a new one

The cache holds groups of 64 values of one token and head as 4-bit codes:
  scale = bf16(max((max - min) / 15, max|x| / 120)),  zero = rint(min / scale),
  code = clamp(rint(x / scale) - zero, 0, 15),        value = (code + zero) * scale
and groups below 2^-100 as zeros.  A page holds 64 tokens of every KV head of a layer.

`own` chooses between the plain form (elementary torch operations in 32 bits, in 64 for the
quotients that are rounded to few bits) and the framework's calls.  Head counts and head sizes
are those of this repository's benchmark and tests (16 query heads on 2 key/value heads with
head_dim 128 and 256, batches of 8, contexts of 1024 to 16384) and generic ones; draw() takes the
ranges around them.
"""

import math
import random

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
PAGE, GROUP = 64, 64
TINY = 2.0 ** -100


def listed():
    return [
        # the smallest call: one sequence's next token, where latency counts
        dict(name="attend_one", kind="attend", batch=1, q_heads=16, kv_heads=2, head_dim=256, dtype="bf16",
             min_len=1000, max_len=1000, min_new=1, max_new=1, gate=False, ragged=0),
        # a decode step of the benchmark's batch: long, unequal sequences, gated output
        dict(name="attend_batch", kind="attend", batch=8, q_heads=16, kv_heads=2, head_dim=256, dtype="bf16",
             min_len=1024, max_len=16384, min_new=1, max_new=1, gate=True, ragged=1),
        # a decode step over very long documents
        dict(name="attend_long", kind="attend", batch=4, q_heads=32, kv_heads=8, head_dim=128, dtype="bf16",
             min_len=100000, max_len=131072, min_new=1, max_new=1, gate=False, ragged=2),
        # verification of one to eight drafted tokens a sequence, seven query heads on each key/value head
        dict(name="attend_draft", kind="attend", batch=24, q_heads=28, kv_heads=4, head_dim=128, dtype="fp16",
             min_len=500, max_len=6000, min_new=1, max_new=8, gate=False, ragged=3),
        # short prompts of ragged length, one token among them, with nothing cached before
        dict(name="attend_prompts", kind="attend", batch=5, q_heads=16, kv_heads=2, head_dim=256, dtype="fp16",
             min_len=1, max_len=1500, min_new=0, max_new=0, gate=True, ragged=4),
        # a prompt's chunk at the end of a long context
        dict(name="attend_chunk", kind="attend", batch=1, q_heads=32, kv_heads=8, head_dim=128, dtype="bf16",
             min_len=32768, max_len=32768, min_new=2048, max_new=2048, gate=False, ragged=5),
        # a decode step's tokens of a large batch enter the cache
        dict(name="store_step", kind="store", batch=64, kv_heads=8, head_dim=128, dtype="bf16",
             min_len=300, max_len=3000, min_new=1, max_new=1, ragged=6),
        # ragged prompts enter the cache, some in the middle of a page
        dict(name="store_prompts", kind="store", batch=6, kv_heads=8, head_dim=128, dtype="fp16",
             min_len=700, max_len=5000, min_new=600, max_new=4000, ragged=7),
        # one prompt answered eight times: its last page is copied for every answer
        dict(name="fork_samples", kind="fork", layers=24, batch=1, copies=8, kv_heads=2, head_dim=256,
             min_len=1000, max_len=1000, ragged=8),
        # every beam of a batch goes on twice
        dict(name="fork_beams", kind="fork", layers=32, batch=48, copies=2, kv_heads=8, head_dim=128,
             min_len=200, max_len=700, ragged=9),
        # a small pool gives memory back after its sequences ended
        dict(name="resize_small", kind="resize", layers=6, batch=7, kv_heads=2, head_dim=64,
             min_len=1, max_len=500, ragged=10),
        # a large fragmented pool
        dict(name="resize_large", kind="resize", layers=32, batch=40, kv_heads=8, head_dim=128,
             min_len=100, max_len=2500, ragged=11),
    ]


# ---------------------------------------------------------------- draw


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


HEADS = ((16, 2), (32, 8), (28, 4), (16, 16), (8, 1), (24, 2))


def draw(rng):
    kind = rng.choice(("attend", "attend", "attend", "attend", "store", "fork", "resize"))
    q_heads, kv_heads = rng.choice(HEADS)
    c = dict(kind=kind, kv_heads=kv_heads, head_dim=rng.choice((64, 128, 256)), ragged=rng.randrange(1 << 30))
    page = kv_heads * _page_bytes(c["head_dim"])
    if kind == "attend":
        c.update(q_heads=q_heads, dtype=rng.choice(("bf16", "fp16")), gate=rng.random() < 0.3)
        form = rng.choice(("decode", "decode", "draft", "chunk", "prompt"))
        c["max_len"] = _log(rng, 2, 131072 if form == "decode" else 32768 if form == "chunk" else 8192)
        c["min_len"] = rng.randint(1, c["max_len"])
        new = {"decode": 1, "draft": rng.randint(2, 16), "chunk": _log(rng, 17, 2048), "prompt": 0}[form]
        c.update(min_new=min(1, new) if form == "draft" else new, max_new=new)
        most = min(64, (1 << 29) // (c["max_len"] * kv_heads * c["head_dim"]),
                   (1 << 31) // (q_heads * (new or c["max_len"]) * c["max_len"]))
        c["batch"] = _log(rng, 1, max(1, most))
    elif kind == "store":
        c.update(dtype=rng.choice(("bf16", "fp16")), max_len=_log(rng, 1, 16384))
        c["min_len"] = rng.randint(1, c["max_len"])
        new = 1 if rng.random() < 0.4 else _log(rng, 1, c["max_len"])
        c.update(min_new=rng.randint(1, new), max_new=new)
        c["batch"] = _log(rng, 1, max(1, min(128, (1 << 26) // (c["max_len"] * kv_heads * c["head_dim"]))))
    elif kind == "fork":
        c.update(max_len=_log(rng, 2, 4000), copies=rng.randint(1, 8))
        c["min_len"] = rng.randint(1, c["max_len"])
        pages = (1 << 30) // page
        c["batch"] = _log(rng, 1, max(1, min(48, pages // (c["max_len"] // PAGE + 1 + c["copies"]))))
        c["layers"] = rng.randint(1, max(1, min(32, pages // (c["batch"] * (c["max_len"] // PAGE + 1 + c["copies"])))))
    else:
        c.update(max_len=_log(rng, 2, 8000))
        c["min_len"] = rng.randint(1, c["max_len"])
        pages = (1 << 30) // page
        c["batch"] = _log(rng, 2, max(2, min(64, pages // (c["max_len"] // PAGE + 1))))
        c["layers"] = rng.randint(1, max(1, min(32, pages // (c["batch"] * (c["max_len"] // PAGE + 1)))))
    return c


# ---------------------------------------------------------------- shapes and work


def _page_bytes(head_dim):
    """Bytes of a page of one KV head: codes of K and V, and a scale and a zero (2 bytes each) of every group."""
    return PAGE * (head_dim + 8 * (head_dim // GROUP))


def _lengths(case):
    """(length, new tokens among them) of every sequence."""
    r = random.Random(case["ragged"])
    lens = [r.randint(case["min_len"], case["max_len"]) for _ in range(case["batch"])]
    lens[0] = case["max_len"]
    if case["batch"] > 1:
        lens[-1] = case["min_len"]
    if case["kind"] in ("fork", "resize"):
        return [(n, 0) for n in lens]
    return [(n, min(n, r.randint(case["min_new"], case["max_new"]) or n)) for n in lens]


def _pages(n):
    return -(-n // PAGE)


def work(case):
    lens = _lengths(case)
    H, D = case["kv_heads"], case["head_dim"]
    if case["kind"] == "attend":
        rows = sum(t for _, t in lens) * case["q_heads"] * D
        pairs = sum(t * n - t * (t - 1) // 2 for n, t in lens)
        return {"bytes": sum(n for n, _ in lens) * H * _page_bytes(D) // PAGE + 2 * rows * (3 if case["gate"] else 2),
                "flops": 4 * case["q_heads"] * D * pairs}
    if case["kind"] == "store":
        n = sum(t for _, t in lens) * H
        return {"bytes": n * (2 * 2 * 2 * D + _page_bytes(D) // PAGE), "flops": 0}
    page = case["layers"] * H * _page_bytes(D)
    if case["kind"] == "fork":
        copied = case["copies"] * sum(n % PAGE != 0 for n, _ in lens)
        return {"bytes": max(1, copied) * 2 * page, "flops": 0}
    live = sum(_pages(n) for n, _ in _live(case))
    return {"bytes": 2 * live * page, "flops": 0}


def _live(case):
    """The sequences that remain: every second one has ended."""
    return _lengths(case)[::2]


# ---------------------------------------------------------------- inputs


def _rows(shape, gen):
    """Normal values with one channel in a hundred eight times as large, as keys and values have."""
    x = torch.randn(shape, device=DEVICE, generator=gen)
    wide = torch.rand(shape[-1], device=DEVICE, generator=gen) < 0.01
    return x.mul_(torch.where(wide, 8.0, 1.0))


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    lens = _lengths(case)
    s = dict(kind=case["kind"], case=case, lens=lens)
    if case["kind"] in ("fork", "resize"):
        return _prepare_pages(s, case, lens, gen)
    dtype, H, D = DTYPES[case["dtype"]], case["kv_heads"], case["head_dim"]
    total, new = sum(n for n, _ in lens), sum(t for _, t in lens)
    if case["kind"] == "attend":
        keys, values = (_rows((total, H, D), gen).to(dtype) for _ in range(2))
        s.update(query=torch.randn((new, case["q_heads"], D), device=DEVICE, generator=gen).to(dtype),
                 gate=torch.randn((new, case["q_heads"], D), device=DEVICE, generator=gen).to(dtype) if case["gate"] else None,
                 scaling=D ** -0.5)
        if own:
            s["cache"], seqs = _cache(case, [n for n, _ in lens], dtype)
            s["cache"].store(0, s["cache"].span(seqs, [0] * len(lens), [n for n, _ in lens]), keys, values)
            s["span"] = s["cache"].span(seqs, [n - t for n, t in lens], [t for _, t in lens])
        else:  # the cache as a padded batch: codes, zeros, scales; and where each new token stands in it
            L, T = max(n for n, _ in lens), max(t for _, t in lens)
            at = torch.tensor([b * L + i for b, (n, _) in enumerate(lens) for i in range(n)], device=DEVICE)
            s["key"], s["value"] = (tuple(x.new_zeros((len(lens) * L, *x.shape[1:])).index_copy_(0, at, x)
                                          .view(len(lens), L, *x.shape[1:]) for x in part) for part in _quantize(keys, values))
            s["at"] = torch.tensor([b * T + i for b, (_, t) in enumerate(lens) for i in range(t)], device=DEVICE)
            s["position"] = torch.tensor([[n - t + min(i, t - 1) for i in range(T)] for n, t in lens], device=DEVICE)
        return s
    s.update(keys=_rows((new, H, D), gen).to(dtype), values=_rows((new, H, D), gen).to(dtype))
    if own:
        s["cache"], seqs = _cache(case, [n - t for n, t in lens], dtype)
        s["span"] = s["cache"].extend(seqs, [t for _, t in lens])
    return s


def _cache(case, lens, dtype, layers=1, pages=None):
    """The framework's cache with sequences of these lengths, their pages interleaved as growing sequences' are."""
    from anna_amd.paged_cache import PagedInt4Cache

    full = _lengths(case)
    cache = PagedInt4Cache(num_layers=layers, num_pages=pages or sum(_pages(n) for n, _ in full) + 1,
                           kv_heads=case["kv_heads"], q_heads=case.get("q_heads", case["kv_heads"]),
                           head_dim=case["head_dim"], max_sequences=len(lens) * (1 + case.get("copies", 0)),
                           max_length=max(n for n, _ in full) + PAGE, dtype=dtype, device=DEVICE)
    seqs = cache.add(len(lens))
    for part in range(4):
        cache.extend(seqs, [n * (part + 1) // 4 - n * part // 4 for n in lens])
    return cache, seqs


def _prepare_pages(s, case, lens, gen):
    B, H, D = case["batch"], case["kv_heads"], case["head_dim"]
    # the pool's pages in the order in which sequences that grow together take them
    used, grown, columns = 0, [0] * B, [[] for _ in range(B)]
    for part in range(4):
        for b, (n, _) in enumerate(lens):
            more = _pages(n * (part + 1) // 4) - grown[b]
            columns[b] += range(used, used + more)
            used, grown[b] = used + more, grown[b] + more
    pages = used + B * case.get("copies", 0) + 1
    width = _pages(max(n for n, _ in lens) + PAGE)
    s["pages"] = sum(_pages(n) for n, _ in _live(case)) + 1  # of the resized pool
    pool = torch.randint(0, 256, (case["layers"], pages, H, _page_bytes(D)), dtype=torch.uint8, device=DEVICE, generator=gen)
    if own:
        s["cache"], s["seqs"] = _cache(case, [n for n, _ in lens], torch.bfloat16, case["layers"], pages)
        s["cache"].pool.copy_(pool)
        if case["kind"] == "resize":
            s["cache"].free(s["seqs"][1::2])
    else:
        live = range(B) if case["kind"] == "fork" else range(0, B, 2)
        table = [columns[b] + [0] * (width - len(columns[b])) if b in live else [0] * width for b in range(B)]
        s.update(pool=pool, table=torch.tensor(table, dtype=torch.int32, device=DEVICE),
                 length=torch.tensor([lens[b][0] if b in live else 0 for b in range(B)], device=DEVICE),
                 free=torch.arange(used, pages, device=DEVICE))
    return s


# ---------------------------------------------------------------- the plain form


def _quantize(keys, values):
    """(codes, zeros, scales) of keys and of values [tokens, heads, head_dim]."""
    def codes(x, lost):
        x = torch.where(lost[..., None], 0.0, x.double().unflatten(-1, (-1, GROUP)))
        low, high = x.amin(-1), x.amax(-1)
        scale = torch.maximum((high - low) / 15, torch.maximum(low.abs(), high.abs()) / 120).float()
        scale = torch.where(scale < TINY, 0.0, scale).to(torch.bfloat16)
        steps = torch.round(x / torch.where(scale == 0, 1.0, scale.double())[..., None])
        steps = torch.where(scale[..., None] == 0, 0.0, steps)
        zero = steps.amin(-1)
        return (steps - zero[..., None]).clamp(0, 15).to(torch.uint8).flatten(-2), zero.to(torch.int16), scale

    lost = ~(torch.isfinite(keys).all(-1) & torch.isfinite(values).all(-1))[..., None]  # held as NaN keys
    kc, kz, ks = codes(keys, lost)
    return (kc, kz, torch.where(lost, float("nan"), ks)), codes(values, lost)


def _dense(codes, zeros, scales):
    return ((codes.float().unflatten(-1, (-1, GROUP)) + zeros.float()[..., None]) * scales.float()[..., None]).flatten(-2)


def _plain_attend(s):
    query, at, position = s["query"], s["at"], s["position"]
    key, value = (_dense(*s[x]).transpose(1, 2) for x in ("key", "value"))  # [batch, kv_heads, len, head_dim]
    (B, H, L, D), T = key.shape, position.shape[1]
    G = query.shape[1] // H
    q = torch.zeros((B * T, H * G, D), device=DEVICE).index_copy_(0, at, query.float())
    q = q.view(B, T, H, G, D).permute(0, 2, 3, 1, 4).reshape(B, H, G * T, D)
    score = torch.matmul(q, key.transpose(2, 3)).mul_(s["scaling"]).view(B, H, G, T, L)
    seen = torch.arange(L, device=DEVICE) <= position[..., None]  # [batch, new, len]
    score.masked_fill_(~seen[:, None, None], float("-inf"))
    p = score.sub_(score.amax(-1, keepdim=True)).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(B, H, G * T, L), value).view(B, H, G, T, D) / total
    out = out.permute(0, 3, 1, 2, 4).reshape(B * T, H * G, D)[at]
    if s["gate"] is not None:
        out = out * torch.sigmoid(s["gate"].float())
    return out.to(query.dtype)


def _plain_store(s):
    key, value = _quantize(s["keys"], s["values"])
    return {"keys": _dense(*key).to(s["keys"].dtype), "values": _dense(*value).to(s["keys"].dtype)}


def _plain_fork(s):
    copies = s["case"]["copies"]
    table, length = s["table"].repeat_interleave(copies, 0), s["length"].repeat_interleave(copies)
    last, to = length // PAGE, s["free"][:len(length)]
    partly = length % PAGE != 0
    source = table.gather(1, last[:, None])[:, 0].long()
    s["pool"][:, to[partly]] = s["pool"][:, source[partly]]
    return {"pool": s["pool"], "table": table.scatter(1, last[:, None], to[:, None].to(table.dtype))}


def _plain_resize(s):
    table, pool = s["table"], s["pool"]
    used = torch.arange(table.shape[1], device=DEVICE) * PAGE < s["length"][:, None]
    live = table[used].long()
    new = pool.new_zeros((pool.shape[0], s["pages"], *pool.shape[2:]))
    new[:, :len(live)] = pool[:, live]
    number = (used.flatten().cumsum(0) - 1).view_as(table)
    return {"pool": new, "table": torch.where(used, number, 0).to(table.dtype)}


# ---------------------------------------------------------------- run


def run(s):
    if not own:
        return {"attend": _plain_attend, "store": _plain_store, "fork": _plain_fork, "resize": _plain_resize}[s["kind"]](s)
    cache = s["cache"]
    if s["kind"] == "attend":
        return cache.attend(0, s["span"], s["query"], scaling=s["scaling"], gate=s["gate"])
    if s["kind"] == "store":
        cache.store(0, s["span"], s["keys"], s["values"])
        keys, values = cache.read(0, s["span"])
        return {"keys": keys, "values": values}
    if s["kind"] == "fork":
        children = cache.fork([seq for seq in s["seqs"] for _ in range(s["case"]["copies"])])
        span = cache.extend(children)
        table = cache.page_table(span)
        cache.free(children)
        return {"pool": cache.pool, "table": table}
    cache.resize(s["pages"])
    return {"pool": cache.pool, "table": cache.table}


# ---------------------------------------------------------------- the definition in 64 bits


def exact(case, seed):
    if case["kind"] in ("fork", "resize"):
        return None  # whole numbers
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    lens, dtype = _lengths(case), DTYPES[case["dtype"]]
    H, D = case["kv_heads"], case["head_dim"]
    total, new = sum(n for n, _ in lens), sum(t for _, t in lens)

    def held(x):
        """What the cache holds of x [..., head_dim], from the definition."""
        x = x.double()
        out = torch.empty_like(x)
        for g in range(0, D, GROUP):
            part = x[..., g:g + GROUP]
            low, high = part.min(-1, keepdim=True)[0], part.max(-1, keepdim=True)[0]
            scale = torch.maximum((high - low) / 15, part.abs().max(-1, keepdim=True)[0] / 120).bfloat16().double()
            zero = (low / scale).round()
            out[..., g:g + GROUP] = scale * (zero + torch.clamp((part / scale).round() - zero, min=0, max=15))
        return out

    if case["kind"] == "store":
        return {"keys": held(_rows((new, H, D), gen).to(dtype)), "values": held(_rows((new, H, D), gen).to(dtype))}
    keys, values = (_rows((total, H, D), gen).to(dtype) for _ in range(2))
    query = torch.randn((new, case["q_heads"], D), device=DEVICE, generator=gen).to(dtype).double()
    gate = torch.randn((new, case["q_heads"], D), device=DEVICE, generator=gen).to(dtype).double() if case["gate"] else None
    out = torch.empty_like(query)
    G, k0, q0 = case["q_heads"] // H, 0, 0
    for n, t in lens:
        unseen = torch.arange(n, device=DEVICE)[None, :] > torch.arange(n - t, n, device=DEVICE)[:, None]
        for h in range(H):
            k, v = held(keys[k0:k0 + n, h]), held(values[k0:k0 + n, h])
            for g in range(h * G, (h + 1) * G):
                score = (query[q0:q0 + t, g] @ k.T) * D ** -0.5
                out[q0:q0 + t, g] = torch.softmax(score.masked_fill(unseen, -math.inf), dim=-1) @ v
        k0, q0 = k0 + n, q0 + t
    return out if gate is None else out / (1 + torch.exp(-gate))
