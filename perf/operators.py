"""One serving step around the linear layers, operator by operator, over the range of sizes a program makes them at.

A case is a dict of plain values; its "kind" says which operator it is:

  rope      rotary positions of the query heads: pairs side by side or half a head apart, the whole head or part of it,
            frequencies scaled for long contexts
  append    the new tokens of a batch, read from the fused projection: queries and keys rotated, keys and values written to
            their slots of a paged cache
  attend    attention of the new tokens of a batch of sequences over the paged cache: one token each, chunks of prompts,
            both in one batch
  sample    the next token of every row of logits: temperature, top-k, top-p and min-p, from given random numbers

Where `own` is false, the operators are computed in their plain form with elementary torch operations.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one stream's next token: the queries of 32 heads, a few kilobytes; launching is all there is
        {"name": "rope_one_token", "kind": "rope", "dtype": "bf16", "tokens": 1, "heads": 32, "head_dim": 128, "rotated": 128,
         "interleaved": True, "scaling": "none"},
        # a prompt of no round length in f32, a quarter of each head rotated in halves, positions beyond the trained range
        {"name": "rope_prompt_f32", "kind": "rope", "dtype": "f32", "tokens": 4001, "heads": 16, "head_dim": 64, "rotated": 16,
         "interleaved": False, "scaling": "bands"},
        # one token of each of 32 streams goes into the cache
        {"name": "append_32_streams", "kind": "append", "dtype": "bf16", "streams": 32, "query": 1, "context": 3000, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "page": 16, "interleaved": False, "scaling": "bands"},
        # a prompt's chunk with a key head for every query head, pairs side by side
        {"name": "append_chunk_f16", "kind": "append", "dtype": "f16", "streams": 1, "query": 4096, "context": 8000, "heads": 16,
         "kv_heads": 16, "head_dim": 64, "page": 64, "interleaved": True, "scaling": "linear"},
        # one stream, 32 heads each with its own keys: the decoder's shape, alone on the machine
        {"name": "attend_one_token", "kind": "attend", "dtype": "bf16", "streams": 1, "query": 1, "context": 1000, "heads": 32,
         "kv_heads": 32, "head_dim": 128, "page": 16, "mix": "one", "window": 0},
        # a full batch of conversations of all lengths, four query heads to a key head: the cache is what is read
        {"name": "attend_32_streams", "kind": "attend", "dtype": "bf16", "streams": 32, "query": 1, "context": 12000, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "page": 16, "mix": "one", "window": 0},
        # a few very long contexts, heads of 64: the long axis has to be shared out
        {"name": "attend_long_f16", "kind": "attend", "dtype": "f16", "streams": 3, "query": 1, "context": 100001, "heads": 16,
         "kv_heads": 4, "head_dim": 64, "page": 64, "mix": "one", "window": 0},
        # chunks of prompts and single tokens in one batch, as a scheduler forms it
        {"name": "attend_mixed", "kind": "attend", "dtype": "bf16", "streams": 12, "query": 300, "context": 3000, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "page": 16, "mix": "mixed", "window": 0},
        # a chunk of a long prompt on top of what came before: the largest call, all tensor-core work
        {"name": "attend_chunk", "kind": "attend", "dtype": "bf16", "streams": 1, "query": 2048, "context": 16384, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "page": 64, "mix": "chunk", "window": 0},
        # one stream's next token out of a text vocabulary
        {"name": "sample_one_row", "kind": "sample", "dtype": "f32", "rows": 1, "vocab": 32000, "filters": "all"},
        # 64 streams, a large vocabulary of odd size, the nucleus alone
        {"name": "sample_64_rows", "kind": "sample", "dtype": "f32", "rows": 64, "vocab": 128001, "filters": "top_p"},
        # 16-bit logits (many equal ones), every request with settings of its own, greedy ones among them
        {"name": "sample_mixed_bf16", "kind": "sample", "dtype": "bf16", "rows": 24, "vocab": 50000, "filters": "mixed"},
    ]


def _spread(rng, lo: int, hi: int) -> int:
    """A size between lo and hi, evenly over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _draw(rng):
    kind = rng.choice(["rope", "append", "attend", "attend", "attend", "sample"])
    if kind == "sample":
        return {"kind": kind, "dtype": rng.choice(["f32", "f32", "bf16", "f16"]), "rows": _spread(rng, 1, 128),
                "vocab": _spread(rng, 1000, 160000), "filters": rng.choice(["all", "top_k", "top_p", "min_p", "none", "mixed"])}
    head_dim = rng.choice([64, 128, 128])
    if kind == "rope":
        return {"kind": kind, "dtype": rng.choice(["bf16", "f16", "f32"]), "tokens": _spread(rng, 1, 8192),
                "heads": _spread(rng, 1, 32), "head_dim": head_dim, "rotated": rng.choice([head_dim, head_dim, head_dim // 2, 16]),
                "interleaved": rng.random() < 0.5, "scaling": rng.choice(["none", "linear", "base", "bands"])}
    kv_heads = rng.choice([1, 2, 4, 8, 16, 32])
    heads = kv_heads * rng.choice([g for g in (1, 2, 3, 4, 5, 6, 7, 8) if g * kv_heads <= 32])
    common = {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "f16"]), "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
              "page": rng.choice([16, 16, 32, 64, 128])}
    if kind == "append":
        one = rng.random() < 0.5
        context = _spread(rng, 16, 20000)
        return {**common, "streams": _spread(rng, 1, 64) if one else rng.choice([1, 2, 3]),
                "query": 1 if one else _spread(rng, 2, min(2048, context)), "context": context,
                "interleaved": rng.random() < 0.5, "scaling": rng.choice(["none", "linear", "base", "bands"])}
    mix = rng.choice(["one", "one", "chunk", "mixed"])
    if mix == "one":
        streams, query, context = _spread(rng, 1, 64), 1, _spread(rng, 16, 100000)
    else:
        streams, context = _spread(rng, 1, 16), _spread(rng, 64, 16000)
        query = _spread(rng, 2, min(2048, context))
    window = _spread(rng, 16, context) if rng.random() < 0.25 else 0
    return {**common, "streams": streams, "query": query, "context": context, "mix": mix, "window": window}


def draw(rng):
    while True:  # nothing that costs more than the largest listed case, in the plain form either
        c = _draw(rng)
        if c["kind"] == "attend":
            tokens = c["streams"] * c["query"]
            if tokens * c["heads"] * c["context"] > 1.07e9 or c["streams"] * c["kv_heads"] * c["context"] * c["head_dim"] > 4e8:
                continue
        w = work(c)
        if w["bytes"] <= 8e8 and w["flops"] <= 5.2e11:
            return c


def _lengths(c):
    """(new tokens, context with them) of every sequence of a case: a conversation has whatever length it has."""
    rng = random.Random("%(streams)d %(query)d %(context)d" % c)
    mix, out = c.get("mix", "chunk"), []
    for b in range(c["streams"]):
        n = c["query"]
        if mix == "mixed" and b:
            n = 1 if rng.random() < 0.5 else rng.randint(1, c["query"])
        ctx = c["context"] if b == 0 else rng.randint(max(n, c["context"] // 8), c["context"])
        out.append((n, ctx))
    return out


def frequencies(rotated: int, scaling: str):
    """Radians per position of every pair, in 64 bits: base^(-2 i / rotated), scaled to contexts 8 times as long as trained."""
    i = torch.arange(rotated // 2, dtype=torch.float64)
    if scaling == "base":  # a larger base slows the slow pairs down by the factor, the fast ones hardly
        return (10000.0 * 8.0 ** (rotated / max(rotated - 2.0, 1.0))) ** (-2.0 * i / rotated)
    f = 10000.0 ** (-2.0 * i / rotated)
    if scaling == "linear":
        return f / 8.0
    if scaling == "bands":  # pairs of few turns over the trained context slow down, those of many turns stay, a ramp between
        turns = 4096 * f / (2.0 * math.pi)
        keep = torch.clamp((turns - 1.0) / (4.0 - 1.0), 0.0, 1.0)
        return f * (keep + (1.0 - keep) / 8.0)
    return f


def prepare(c, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(int(seed))
    kind = c["kind"]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device=dev) * scale).to(DTYPES[c["dtype"]])

    if kind == "rope":
        first = int(torch.randint(0, 30000, (1,), generator=g, device=dev))
        return {"kind": kind, "x": normal(c["tokens"], c["heads"], c["head_dim"]), "interleaved": c["interleaved"],
                "positions": torch.arange(first, first + c["tokens"], device=dev),
                "freqs": frequencies(c["rotated"], c["scaling"]).to(dev)}
    if kind == "sample":
        rows, vocab, f = c["rows"], c["vocab"], c["filters"]
        # logits of a language model: a few likely tokens above a broad floor, and some that the request forbids
        x = torch.randn(rows, vocab, generator=g, device=dev) * 2.0
        x += 9.0 * torch.exp(-0.02 * torch.rand(rows, vocab, generator=g, device=dev) * vocab)
        x[:, 7::997] = -math.inf
        uniform = torch.rand(rows, generator=g, device=dev)
        pick = torch.rand(4, rows, generator=g, device=dev)
        t = 0.6 + 0.6 * pick[0]
        k = 1 + (pick[1] * 200).to(torch.int32)
        p = 0.8 + 0.19 * pick[2]
        m = 0.1 * pick[3]
        if f == "mixed":
            every = torch.arange(rows, device=dev)
            t = torch.where(every % 4 == 1, torch.zeros_like(t), t)
            k = torch.where(every % 3 == 1, torch.zeros_like(k), k)
            p = torch.where(every % 5 == 2, torch.ones_like(p), p)
            m = torch.where(every % 2 == 0, torch.zeros_like(m), m)
        return {"kind": kind, "logits": x.to(DTYPES[c["dtype"]]), "uniform": uniform, "temperature": t,
                "top_k": k if f in ("all", "top_k", "mixed") else None, "top_p": p if f in ("all", "top_p", "mixed") else None,
                "min_p": m if f in ("all", "min_p", "mixed") else None}

    heads, kv, hd, page = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    lengths = _lengths(c)
    tokens = sum(n for n, _ in lengths)
    per = [-(-ctx // page) for _, ctx in lengths]
    # pages are handed out in no order, and the pool has some that nobody uses
    pages = torch.randperm(sum(per) + 3, generator=g, device=dev).to(torch.int32)
    table = torch.zeros(len(per), max(per), dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = pages[at:at + n]
        at += n
    if kind == "append":
        qkv = normal(tokens, (heads + 2 * kv) * hd).view(tokens, heads + 2 * kv, hd)  # the fused projection's rows
        owner = torch.cat([torch.full((n,), b) for b, (n, _) in enumerate(lengths)]).to(dev)
        pos = torch.cat([torch.arange(ctx - n, ctx) for n, ctx in lengths]).to(dev)
        slots = table[owner, pos // page].long() * page + pos % page
        # the pool as far as this batch writes it, and a little more: a step's cost does not depend on the rest of it
        used = torch.unique(slots // page)
        slots = torch.searchsorted(used, slots // page) * page + slots % page
        return {"kind": kind, "q": qkv[:, :heads], "k": qkv[:, heads:heads + kv], "v": qkv[:, heads + kv:], "positions": pos,
                "freqs": frequencies(hd, c["scaling"]).to(dev), "interleaved": c["interleaved"], "slots": slots,
                "k_pages": normal(len(used) + 3, kv, page, hd), "v_pages": normal(len(used) + 3, kv, page, hd)}
    starts = [0]
    for n, _ in lengths:
        starts.append(starts[-1] + n)
    ints = dict(dtype=torch.int32, device=dev)
    s = {"kind": kind, "q": normal(tokens, heads, hd), "k_pages": normal(sum(per) + 3, kv, page, hd),
         "v_pages": normal(sum(per) + 3, kv, page, hd), "table": table, "context": torch.tensor([ctx for _, ctx in lengths], **ints),
         "starts": torch.tensor(starts, **ints) if c["mix"] != "one" else None, "max_query": max(n for n, _ in lengths),
         "max_context": max(ctx for _, ctx in lengths), "scale": 1.0 / math.sqrt(hd), "window": c["window"]}
    return s


# -- the plain forms --------------------------------------------------------------------------------------------------
def _rotated(x, positions, freqs, interleaved):
    angle = positions.double()[:, None, None] * freqs  # [tokens, 1, pairs]: positions times frequencies need 64 bits
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    n = freqs.numel()
    x32 = x.float()
    a, b = (x32[..., 0:2 * n:2], x32[..., 1:2 * n:2]) if interleaved else (x32[..., :n], x32[..., n:2 * n])
    y0, y1 = a * cos - b * sin, a * sin + b * cos
    y = torch.stack([y0, y1], -1).flatten(-2) if interleaved else torch.cat([y0, y1], -1)
    return torch.cat([y, x32[..., 2 * n:]], -1).to(x.dtype)


def _append(s):
    page = s["k_pages"].shape[2]
    at, off = s["slots"] // page, s["slots"] % page
    s["k_pages"][at, :, off] = _rotated(s["k"], s["positions"], s["freqs"], s["interleaved"])
    s["v_pages"][at, :, off] = s["v"]
    return _rotated(s["q"], s["positions"], s["freqs"], s["interleaved"])


def _attend(s):
    q, table, context, starts = s["q"], s["table"].long(), s["context"].long(), s["starts"]
    batch, (tokens, heads, hd) = table.shape[0], q.shape
    kv, width, most = s["k_pages"].shape[1], s["max_query"], s["max_context"]
    if starts is None:
        starts = torch.arange(batch + 1, device=q.device)
    starts = starts.long()
    n = starts[1:] - starts[:-1]
    row = torch.arange(width, device=q.device)
    token = torch.clamp(starts[:-1, None] + row, max=tokens - 1)  # [batch, width], padded
    real = row < n[:, None]
    k = s["k_pages"][table].transpose(1, 2).flatten(2, 3)[:, :, :most].float()  # [batch, kv, context, hd]
    v = s["v_pages"][table].transpose(1, 2).flatten(2, 3)[:, :, :most].float()
    q32 = q[token].float().unflatten(2, (kv, heads // kv)).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [batch, kv, group * width, hd]
    scores = (q32 @ k.transpose(2, 3)).mul_(s["scale"]).unflatten(2, (heads // kv, width))
    key = torch.arange(most, device=q.device)
    last = (context - n)[:, None] + row  # the last key that a row sees
    seen = key <= last[..., None]
    if s["window"]:
        seen &= key > last[..., None] - s["window"]
    seen = seen[:, None, None]
    scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    v = torch.where((key < context[:, None])[:, None, :, None], v, torch.zeros_like(v))
    out = (p.flatten(2, 3) @ v).unflatten(2, (heads // kv, width)) / torch.where(total == 0, torch.ones_like(total), total)
    return out.permute(0, 3, 1, 2, 4).flatten(2, 3)[real].to(q.dtype)  # [tokens, heads, hd]


def _sample(s):
    x = s["logits"].double()  # the draw falls between sums of many small weights: 64 bits
    rows, vocab = x.shape
    rank = torch.arange(vocab, device=x.device)
    t = s["temperature"].double()[:, None]
    value, order = torch.sort(x, dim=1, descending=True, stable=True)
    top = value[:, :1]
    w = torch.exp((value - top) / torch.where(t > 0, t, torch.ones_like(t)))
    w = torch.where(torch.isinf(value), torch.zeros_like(w), w)
    kept = torch.where(t > 0, rank < vocab, rank < 1)
    if s["top_k"] is not None:
        k = s["top_k"].long()[:, None]
        kept = kept & ((rank < k) | (k <= 0))
    w = torch.where(kept, w, torch.zeros_like(w))
    if s["top_p"] is not None:
        p = s["top_p"].double()[:, None]
        before = torch.cumsum(w, 1) - w
        kept = kept & ((before < p * w.sum(1, keepdim=True)) | (p >= 1) | (rank < 1))
    if s["min_p"] is not None:
        kept = kept & (w >= s["min_p"].double()[:, None])
    w = torch.where(kept, w, torch.zeros_like(w))
    mass = torch.zeros_like(w).scatter_(1, order, w)  # back in the vocabulary's order
    below = torch.cumsum(mass, 1)
    past = below > s["uniform"].double()[:, None] * below[:, -1:]
    return torch.where(past, rank, torch.full_like(rank, vocab)).amin(1)


def run(s):
    kind = s["kind"]
    if own:
        import xn_b200 as xn

        if kind == "rope":
            return xn.rope(s["x"], s["positions"], s["freqs"], interleaved=s["interleaved"])
        if kind == "append":
            q = xn.paged_append_(s["k_pages"], s["v_pages"], s["k"], s["v"], s["slots"], q=s["q"], positions=s["positions"],
                                 freqs=s["freqs"], interleaved=s["interleaved"])
            return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
        if kind == "attend":
            return xn.attention_paged(s["q"], s["k_pages"], s["v_pages"], s["table"], s["context"], s["scale"],
                                      query_starts=s["starts"], max_query=s["max_query"], window=s["window"])
        return xn.sample(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"], min_p=s["min_p"])
    if kind == "rope":
        return _rotated(s["x"], s["positions"], s["freqs"], s["interleaved"])
    if kind == "append":
        return {"q": _append(s), "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    if kind == "attend":
        return _attend(s)
    return _sample(s)


def work(c):
    kind = c["kind"]
    if kind == "sample":
        n = c["rows"] * c["vocab"]
        return {"bytes": n * BYTES[c["dtype"]] + 28 * c["rows"], "flops": 4 * n}
    e = BYTES[c["dtype"]]
    if kind == "rope":
        return {"bytes": c["tokens"] * (2 * c["heads"] * c["head_dim"] * e + 8) + 4 * c["rotated"],
                "flops": 3 * c["tokens"] * c["heads"] * c["rotated"]}
    lengths = _lengths(c)
    tokens = sum(n for n, _ in lengths)
    if kind == "append":
        return {"bytes": tokens * (2 * (c["heads"] + 2 * c["kv_heads"]) * c["head_dim"] * e + 16) + 4 * c["head_dim"],
                "flops": 3 * tokens * (c["heads"] + c["kv_heads"]) * c["head_dim"]}
    keys = pairs = 0
    window = c["window"]
    for n, ctx in lengths:
        first = max(0, ctx - n + 1 - window) if window else 0  # the first key that any row sees
        keys += ctx - first
        if window:
            pairs += sum(min(ctx - n + i + 1, window) for i in range(n))
        else:
            pairs += n * (ctx - n) + n * (n + 1) // 2
    table = 4 * sum(-(-ctx // c["page"]) for _, ctx in lengths)
    return {"bytes": 2 * tokens * c["heads"] * c["head_dim"] * e + 2 * keys * c["kv_heads"] * c["head_dim"] * e + table + 8 * len(lengths),
            "flops": 4 * pairs * c["heads"] * c["head_dim"]}


# -- what run() returns, in 64 bits and from the definitions ------------------------------------------------------------
def _exact_turn(x, positions, freqs, interleaved):
    """Every pair as a complex number, times e^(i position frequency)."""
    n = freqs.numel()
    turn = torch.polar(torch.ones(1, 1, dtype=torch.float64, device=x.device), torch.outer(positions.double(), freqs))[:, None]
    y = x.double().clone()
    if interleaved:
        y[..., :2 * n] = torch.view_as_real(torch.view_as_complex(y[..., :2 * n].unflatten(-1, (n, 2)).contiguous()) * turn).flatten(-2)
    else:
        z = torch.complex(y[..., :n], y[..., n:2 * n]) * turn
        y[..., :n], y[..., n:2 * n] = z.real, z.imag
    return y


def exact(c, seed):
    s = prepare(c, seed)
    kind = c["kind"]
    if kind == "rope":
        return _exact_turn(s["x"], s["positions"], s["freqs"], c["interleaved"])
    if kind == "append":
        page = c["page"]
        k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
        rows = _exact_turn(s["k"], s["positions"], s["freqs"], c["interleaved"])
        flat = k_pages.transpose(1, 2).contiguous().flatten(0, 1)  # a row for every slot
        flat[s["slots"]] = rows
        k_pages = flat.unflatten(0, (-1, page)).transpose(1, 2)
        flat = v_pages.transpose(1, 2).contiguous().flatten(0, 1)
        flat[s["slots"]] = s["v"].double()
        return {"q": _exact_turn(s["q"], s["positions"], s["freqs"], c["interleaved"]), "k_pages": k_pages,
                "v_pages": flat.unflatten(0, (-1, page)).transpose(1, 2)}
    if kind == "attend":
        if work(c)["flops"] > 6e11:
            return None
        group, out, at = c["heads"] // c["kv_heads"], torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device), 0
        for b, (n, ctx) in enumerate(_lengths(c)):
            pages = s["table"][b, :-(-ctx // c["page"])].long()
            last = torch.arange(ctx - n, ctx, device=pages.device)[:, None]
            key = torch.arange(ctx, device=pages.device)
            hidden = key > last
            if c["window"]:
                hidden |= key <= last - c["window"]
            for h in range(c["kv_heads"]):
                k = s["k_pages"][pages, h].flatten(0, 1)[:ctx].double()
                v = s["v_pages"][pages, h].flatten(0, 1)[:ctx].double()
                for j in range(h * group, (h + 1) * group):
                    a = s["q"][at:at + n, j].double() @ k.T * s["scale"]
                    out[at:at + n, j] = torch.softmax(a.masked_fill(hidden, -math.inf), 1) @ v
            at += n
        return out
    tokens = []
    for r in range(c["rows"]):
        x = s["logits"][r].double().cpu().numpy()
        t, u = float(s["temperature"][r]), float(s["uniform"][r])
        if t <= 0:
            tokens.append(int(np.argmax(x)))
            continue
        w = np.exp((x - x.max()) / t)
        best = np.lexsort((np.arange(len(x)), -x))
        if s["top_k"] is not None and int(s["top_k"][r]) > 0:
            best = best[:int(s["top_k"][r])]
        if s["top_p"] is not None and float(s["top_p"][r]) < 1:
            total = np.cumsum(w[best])
            best = best[:max(1, int(np.searchsorted(total, float(s["top_p"][r]) * total[-1])) + 1)]
        if s["min_p"] is not None:
            best = best[w[best] >= float(s["min_p"][r])]
        best = np.sort(best)
        total = np.cumsum(w[best])
        tokens.append(int(best[np.searchsorted(total, u * total[-1], side="right")]))
    return torch.tensor(tokens, device=s["logits"].device)
