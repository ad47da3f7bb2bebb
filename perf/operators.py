"""The attention side of a decoder layer, as cases that can be timed.

Four operators stand around the feed-forward path of this package, in the order a layer calls them:

  norm    block_norm (RMS norm in front of a block) and block_norm_add (RMS norm behind it, with gate, residual, layer scalar
          and, on request, the next block's norm of the result)
  append  kv_append: per-head RMS norms of queries and keys, rotation by position, keys and values into a paged cache
  prompt  prompt_attention: causal attention over whole packed prompts, grouped heads, optional sliding window
  chunk   chunk_attention: new tokens of several sequences against their pages of the cache, one token each when decoding

`run` computes a case in plain torch operations in 32 bits, or, with `own` set, through gevva_b200.attention; `exact` computes it
from the definitions in 64 bits.  Heads of 256 and a window of 1024 stand for the sliding layers of the model that this package
serves, heads of 512 over the whole context for every sixth layer; heads of 64 and 128 are generic.
"""
import math

import torch

own = False
DEVICE = "cuda:0"
EPS = 1e-6


def _norm(rows, width, form, name=None):
    case = {"kind": "norm", "rows": rows, "width": width, "form": form}
    return dict(case, name=name) if name else case


def _append(news, pasts, heads, kv_heads, dim, page, theta, rotated, packed, name=None):
    case = {"kind": "append", "news": news, "pasts": pasts, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "theta": theta, "rotated": rotated, "packed": packed}
    return dict(case, name=name) if name else case


def _prompt(news, heads, kv_heads, dim, window, name=None):
    case = {"kind": "prompt", "news": news, "heads": heads, "kv_heads": kv_heads, "dim": dim, "window": window}
    return dict(case, name=name) if name else case


def _chunk(news, pasts, heads, kv_heads, dim, page, window, name=None):
    case = {"kind": "chunk", "news": news, "pasts": pasts, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "window": window}
    return dict(case, name=name) if name else case


# Lengths of a list are written as text, "17 1 130": a case holds plain values only.
def _ints(text):
    return [int(t) for t in text.split()]


def _text(values):
    return " ".join(str(v) for v in values)


def listed():
    return [
        # behind the attention of a decode step: 64 rows, residual, layer scalar and the feed-forward norm in one pass
        _norm(64, 2816, "next", name="norm_add_next_64"),
        # in front of the attention of a prefill batch
        _norm(4608, 2816, "pre", name="norm_4608"),
        # one decode step of 64 sequences at positions of their own
        _append(_text([1] * 64), _text([(977 * i + 13) % 7919 for i in range(64)]), 16, 8, 256, 16, 1e4, 256, False, name="append_decode_64"),
        # a prefill batch of four prompts, whose rotated keys the prompt attention reads packed
        _append("1500 1 2049 1058", "0 0 0 0", 16, 8, 256, 64, 1e4, 256, True, name="append_prompt_4608"),
        # three short prompts, one of a single token: latency
        _prompt("17 1 130", 8, 8, 64, 0, name="prompt_short_64"),
        # a prefill batch through a sliding layer
        _prompt("1500 1 2049 1058", 16, 8, 256, 1024, name="prompt_window_256"),
        # the same size in one prompt through a layer over the whole context
        _prompt("4608", 16, 2, 512, 0, name="prompt_whole_512"),
        # one long prompt, generic heads in groups of four
        _prompt("8191", 32, 8, 128, 0, name="prompt_long_128"),
        # one chat reply, token by token
        _chunk("1", "700", 16, 8, 256, 16, 0, name="decode_1_256"),
        # a busy decode batch with contexts from nothing to thousands of tokens
        _chunk(_text([1] * 64), _text([(977 * i + 13) % 7919 for i in range(64)]), 16, 8, 256, 16, 0, name="decode_64_256"),
        # drafts of eight sequences verified together in a sliding layer
        _chunk(_text([5] * 8), "3001 40 977 5000 1019 1024 2500 300", 16, 8, 256, 64, 1024, name="verify_8_256"),
        # a chunk of a long document through a layer over the whole context
        _chunk("512", "32000", 16, 2, 512, 128, 0, name="chunk_512_512"),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _lengths(rng, total, most):
    """Up to `most` lengths that add up to `total`, uneven."""
    count = min(_log_int(rng, 1, most), total)
    cuts = sorted(rng.sample(range(1, total), count - 1)) if count > 1 else []
    return [b - a for a, b in zip([0] + cuts, cuts + [total])]


def draw(rng):
    kind = rng.choice(["norm", "append", "prompt", "prompt", "chunk", "chunk"])
    if kind == "norm":
        return _norm(_log_int(rng, 1, 6000), rng.choice([2816, 64, 8 * rng.randint(8, 600), 8 * rng.randint(8, 600)]),
                     rng.choice(["pre", "add", "gate", "next"]))
    dim = rng.choice([64, 128, 256, 512])
    kv_heads = rng.randint(1, 8 if dim < 512 else 4)
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8])
    page = rng.choice([16, 32, 64, 128, 256])
    window = rng.choice([0, 0, 1024, rng.randint(1, 2000)])
    if kind == "append":
        news = _lengths(rng, _log_int(rng, 1, 4000), 64)
        return _append(_text(news), _text([_log_int(rng, 1, 20000) - 1 for _ in news]), heads, kv_heads, dim, page,
                       rng.choice([1e4, 1e6]), rng.choice([dim, dim, dim // 2]), rng.random() < 0.5)
    budget = 4 * 512 * 16 * 512 * 32256 // 2  # half of the largest listed case's operations
    if kind == "prompt":
        total = min(_log_int(rng, 1, 8000), int(math.sqrt(budget / (2 * dim * heads))))
        return _prompt(_text(_lengths(rng, max(1, total), 16)), heads, kv_heads, dim, window)
    if rng.random() < 0.5:  # decoding
        count = _log_int(rng, 1, 64)
        news = [rng.choice([1, 1, 1, 2, 5]) for _ in range(count)]
        pasts = [_log_int(rng, 1, 16000) - 1 for _ in range(count)]
    else:
        count = _log_int(rng, 1, 6)
        news = [_log_int(rng, 1, 700) for _ in range(count)]
        pasts = [_log_int(rng, 1, max(1, min(16000, budget // (4 * dim * heads * n * count)))) - 1 for n in news]
    return _chunk(_text(news), _text(pasts), heads, kv_heads, dim, page, window)


def _randn(gen, *shape, mean=0.0, std=1.0):
    return (torch.randn(*shape, generator=gen, device=DEVICE, dtype=torch.float32) * std + mean).to(torch.bfloat16)


def _offsets(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed * 1000003 + 17)
    st = {"case": case}
    if case["kind"] == "norm":
        rows, width = case["rows"], case["width"]
        st["x"] = _randn(gen, rows, width, std=3.0)
        st["weight"] = _randn(gen, width, mean=1.0, std=0.2)
        st["residual"] = _randn(gen, rows, width, std=2.0)
        st["gate"] = _randn(gen, width, mean=0.7, std=0.3)
        st["scale"] = _randn(gen, 1, mean=0.8, std=0.1)
        st["next_weight"] = _randn(gen, width, mean=1.0, std=0.2)
        return st
    news = _ints(case["news"])
    tokens, heads, kv_heads, dim = sum(news), case["heads"], case["kv_heads"], case["dim"]
    st["offsets"] = torch.tensor(_offsets(news), dtype=torch.int32, device=DEVICE)
    if case["kind"] == "prompt":
        st["q"], st["k"], st["v"] = _randn(gen, tokens, heads, dim), _randn(gen, tokens, kv_heads, dim), _randn(gen, tokens, kv_heads, dim)
        return st
    lengths = [p + n for p, n in zip(_ints(case["pasts"]), news)]
    page = case["page"]
    needed = [-(-n // page) for n in lengths]
    pages = sum(needed) + 3
    order = torch.randperm(pages, generator=gen, device=DEVICE).to(torch.int32)
    table = torch.zeros(len(news), max(needed), dtype=torch.int32, device=DEVICE)
    at = 0
    for s, n in enumerate(needed):
        table[s, :n] = order[at:at + n]
        at += n
    st["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=DEVICE)
    st["table"] = table
    st["k_cache"], st["v_cache"] = _randn(gen, pages, page, kv_heads, dim), _randn(gen, pages, page, kv_heads, dim)
    if case["kind"] == "chunk":
        st["q"] = _randn(gen, tokens, heads, dim)
    else:
        # the rows of one projection, as a layer's product leaves them
        qkv = _randn(gen, tokens, heads + 2 * kv_heads, dim, std=2.0)
        st["q"], st["k"], st["v"] = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
        st["q_weight"], st["k_weight"] = _randn(gen, dim, mean=1.0, std=0.2), _randn(gen, dim, mean=1.0, std=0.2)
        half = case["rotated"] // 2
        st["frequencies"] = case["theta"] ** (-torch.arange(half, dtype=torch.float64, device=DEVICE) / half)
    if own:
        from gevva_b200 import attention
        st["cache"] = attention.KvCache(st["k_cache"], st["v_cache"])
        st["batch"] = attention.PagedBatch(st["offsets"], st["lengths"], st["table"])
    return st


def run(st):
    kind = st["case"]["kind"]
    return {"norm": _run_norm, "append": _run_append, "prompt": _run_prompt, "chunk": _run_chunk}[kind](st)


def _own():
    from gevva_b200 import attention
    return attention


def _rms(x, weight):
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return y if weight is None else y * weight.float()


def _run_norm(st):
    form = st["case"]["form"]
    gate = st["gate"] if form in ("gate", "next") else None
    scale = st["scale"] if form == "next" else None
    next_weight = st["next_weight"] if form == "next" else None
    if own:
        if form == "pre":
            return _own().block_norm(st["x"], st["weight"], eps=EPS)
        return _own().block_norm_add(st["x"], st["weight"], st["residual"], gate=gate, scale=scale, next_weight=next_weight, eps=EPS)
    y = _rms(st["x"].float(), st["weight"])
    if form == "pre":
        return y.to(torch.bfloat16)
    if gate is not None:
        y = y * gate.float()
    out = st["residual"].float() + y
    if scale is not None:
        out = out * scale.float()
    if next_weight is None:
        return out.to(torch.bfloat16)
    return out.to(torch.bfloat16), _rms(out, next_weight).to(torch.bfloat16)


def _slots(st):
    """Position of every new token, and its page and slot."""
    news = (st["offsets"][1:] - st["offsets"][:-1]).long()
    total = st["q"].shape[0]
    sequence = torch.repeat_interleave(torch.arange(len(news), device=DEVICE), news, output_size=total)
    position = torch.arange(total, device=DEVICE) - st["offsets"][:-1].long()[sequence] + (st["lengths"].long() - news)[sequence]
    page = st["case"]["page"]
    return position, st["table"][sequence, position // page].long(), position % page


def _run_append(st):
    packed = st["case"]["packed"]
    if own:
        out = _own().kv_append(st["q"], st["k"], st["v"], st["cache"], st["batch"], st["frequencies"], q_weight=st["q_weight"],
                               k_weight=st["k_weight"], normalize_v=True, eps=EPS, packed=packed)
        out = tuple(out) if packed else (out,)
    else:
        position, page, slot = _slots(st)
        angle = position.double()[:, None] * st["frequencies"]
        cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
        half = st["case"]["rotated"] // 2

        def rotate(x):
            a, b = x[..., :half], x[..., half:2 * half]
            return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]], -1).to(torch.bfloat16)

        q, k = rotate(_rms(st["q"].float(), st["q_weight"])), rotate(_rms(st["k"].float(), st["k_weight"]))
        v = _rms(st["v"].float(), None).to(torch.bfloat16)
        st["k_cache"][page, slot] = k
        st["v_cache"][page, slot] = v
        out = (q, k, v) if packed else (q,)
    return (*out, st["k_cache"], st["v_cache"])


def _scale(st):
    return st["case"]["dim"] ** -0.5


def _plain_attention(q, k, v, past, scale, window):
    """q [n, heads, dim] at positions past.., k and v [length, kv_heads, dim]: one key head after another."""
    n, heads, dim = q.shape
    length, kv_heads, _ = k.shape
    group = heads // kv_heads
    at = torch.arange(n, device=DEVICE)[:, None] + past
    key = torch.arange(length, device=DEVICE)[None]
    hidden = key > at
    if window:
        hidden |= key <= at - window
    out = torch.empty(n, heads, dim, dtype=torch.bfloat16, device=DEVICE)
    for h in range(kv_heads):
        mine = slice(h * group, (h + 1) * group)
        scores = q[:, mine].float().transpose(0, 1) @ k[:, h].float().T * scale
        scores.masked_fill_(hidden, -math.inf)
        p = torch.exp(scores - scores.amax(-1, keepdim=True))
        out[:, mine] = ((p @ v[:, h].float()) / p.sum(-1, keepdim=True)).transpose(0, 1).to(torch.bfloat16)
    return out


def _run_prompt(st):
    window = st["case"]["window"]
    if own:
        return _own().prompt_attention(st["q"], st["k"], st["v"], st["offsets"], _scale(st), window=window)
    at = _offsets(_ints(st["case"]["news"]))
    return torch.cat([_plain_attention(st["q"][a:b], st["k"][a:b], st["v"][a:b], 0, _scale(st), window) for a, b in zip(at, at[1:])])


def _run_chunk(st):
    case = st["case"]
    if own:
        return _own().chunk_attention(st["q"], st["cache"], st["batch"], _scale(st), window=case["window"])
    news, pasts, page = _ints(case["news"]), _ints(case["pasts"]), case["page"]
    at, out = _offsets(news), []
    for s, (n, past) in enumerate(zip(news, pasts)):
        length = past + n
        rows = st["table"][s, :-(-length // page)].long()
        k, v = (c[rows].flatten(0, 1)[:length] for c in (st["k_cache"], st["v_cache"]))
        out.append(_plain_attention(st["q"][at[s]:at[s + 1]], k, v, past, _scale(st), case["window"]))
    return torch.cat(out)


# ---- the definitions in 64 bits ----------------------------------------------------------------

def _normed(x, weight):
    x = x.double()
    size = ((x ** 2).sum(-1) / x.shape[-1] + EPS).sqrt()
    x = x / size.unsqueeze(-1)
    return x if weight is None else x * weight.double()


def _defined_attention(q, k_rows, v_rows, past, window, scale):
    """Blocks of queries against the keys that any of them sees; the rows of a head group stand under one another."""
    n, heads, dim = q.shape
    kv_heads = k_rows.shape[1]
    out = torch.zeros(n, heads, dim, dtype=torch.float64, device=DEVICE)
    step = max(1, min(256, 10 ** 9 // max(1, 8 * heads * k_rows.shape[0])))
    for first in range(0, n, step):
        last = min(n, first + step)
        low = max(0, past + first - window + 1) if window else 0
        high = past + last
        where = torch.arange(low, high, device=DEVICE)
        who = torch.arange(first, last, device=DEVICE) + past
        seen = where[None] <= who[:, None]
        if window:
            seen &= where[None] > who[:, None] - window
        k, v = k_rows[low:high].double(), v_rows[low:high].double()
        rows = q[first:last].double().reshape(last - first, kv_heads, heads // kv_heads, dim)
        score = torch.einsum("qhgd,khd->hgqk", rows, k) * scale
        score = torch.where(seen, score, torch.full((), -math.inf, dtype=torch.float64, device=DEVICE))
        share = torch.softmax(score, -1)
        out[first:last] = torch.einsum("hgqk,khd->qhgd", share, v).reshape(last - first, heads, dim)
    return out


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "norm":
        y = _normed(st["x"], st["weight"])
        if case["form"] == "pre":
            return y
        if case["form"] in ("gate", "next"):
            y = y * st["gate"].double()
        out = st["residual"].double() + y
        if case["form"] != "next":
            return out
        out = out * st["scale"].double()
        return out, _normed(out, st["next_weight"])
    news = _ints(case["news"])
    if case["kind"] == "prompt":
        parts, at = [], 0
        for n in news:
            parts.append(_defined_attention(st["q"][at:at + n], st["k"][at:at + n], st["v"][at:at + n], 0, case["window"], _scale(st)))
            at += n
        return torch.cat(parts)
    pasts, page, table = _ints(case["pasts"]), case["page"], st["table"].cpu().tolist()
    if case["kind"] == "chunk":
        parts, at = [], 0
        for s, (n, past) in enumerate(zip(news, pasts)):
            order = torch.tensor(table[s][:(past + n + page - 1) // page], device=DEVICE)
            k, v = (torch.index_select(c, 0, order).reshape(-1, case["kv_heads"], case["dim"]) for c in (st["k_cache"], st["v_cache"]))
            parts.append(_defined_attention(st["q"][at:at + n], k, v, past, case["window"], _scale(st)))
            at += n
        return torch.cat(parts)
    # append: complex numbers turn by the angle
    half = case["rotated"] // 2
    where = [p + i for n, p in zip(news, pasts) for i in range(n)]
    seq = [s for s, n in enumerate(news) for _ in range(n)]
    angle = torch.outer(torch.tensor(where, dtype=torch.float64, device=DEVICE), st["frequencies"])
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]

    def turned(x):
        z = torch.complex(x[..., :half].contiguous(), x[..., half:2 * half].contiguous()) * turn
        return torch.cat([z.real, z.imag, x[..., 2 * half:]], -1)

    q, k, v = turned(_normed(st["q"], st["q_weight"])), turned(_normed(st["k"], st["k_weight"])), _normed(st["v"], None)
    row = torch.tensor([table[s][p // page] * page + p % page for s, p in zip(seq, where)], device=DEVICE)
    caches = []
    for cache, rows in ((st["k_cache"], k), (st["v_cache"], v)):
        whole = cache.double()
        whole.view(-1, case["kv_heads"], case["dim"])[row] = rows
        caches.append(whole)
    return (q, k, v, *caches) if case["packed"] else (q, *caches)


def _pairs_and_keys(case):
    """Visible (query, key) pairs and, over the sequences, keys that any query sees."""
    pairs = keys = 0
    news = _ints(case["news"])
    pasts = _ints(case["pasts"]) if case["kind"] == "chunk" else [0] * len(news)
    window = case["window"]
    for n, past in zip(news, pasts):
        for i in range(n):
            pairs += min(past + i + 1, window) if window else past + i + 1
        keys += past + n - (max(0, past - window + 1) if window else 0)
    return pairs, keys


def work(case):
    if case["kind"] == "norm":
        reads = {"pre": 1, "add": 2, "gate": 2, "next": 2}[case["form"]]
        writes = 2 if case["form"] == "next" else 1
        vectors = {"pre": 1, "add": 1, "gate": 2, "next": 3}[case["form"]]
        return {"bytes": 2 * case["width"] * (case["rows"] * (reads + writes) + vectors), "flops": 6 * case["rows"] * case["width"] * writes}
    tokens = sum(_ints(case["news"]))
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["kind"] == "append":
        read = heads + 2 * kv_heads
        written = read + (2 * kv_heads if case["packed"] else 0)
        return {"bytes": 2 * dim * tokens * (read + written), "flops": 8 * dim * tokens * read}
    pairs, keys = _pairs_and_keys(case)
    return {"bytes": 2 * dim * (2 * tokens * heads + 2 * keys * kv_heads), "flops": 4 * dim * heads * pairs}
