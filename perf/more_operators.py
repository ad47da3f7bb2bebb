"""What a serving step has around its layers, as cases that can be timed.

Four operators, in the order in which a step calls them:

  plan    plan_step: from the lengths of the requests and their numbers of new tokens the rows of each request, pages for them out of a
          pool, and every token's position and slot in the paged cache
  trim    trim_step: the pages that requests no longer need, as rejected drafts and finished requests leave them, go back to the pool
  place   kv_append_at: per-head RMS norms of queries and keys, rotation by positions of several axes (time, height, width), keys and
          values into the slots that the plan named
  sample  sample_tokens: temperature, top-k, top-p and min-p from given random numbers, over logits that may be capped and masked

`run` computes a case in plain torch operations, or, with `own` set, through gevva_b200.step; `exact` computes it from the definitions.
Shares and sums of a vocabulary are taken in 64 bits everywhere, since a token is chosen where a running sum passes a border.
"""
import math

import numpy as np
import torch

own = False
DEVICE = "cuda:0"
EPS = 1e-6


def _plan(sequences, most_past, news, page, spare, name=None):
    """news: how many new tokens a request has: "1" for decoding, "1-5" for drafts of several lengths, "0-1" where slots are idle, or a list."""
    case = {"kind": "plan", "sequences": sequences, "most_past": most_past, "news": news, "page": page, "spare": spare}
    return dict(case, name=name) if name else case


def _trim(sequences, most_past, form, page, name=None):
    case = {"kind": "trim", "sequences": sequences, "most_past": most_past, "form": form, "page": page}
    return dict(case, name=name) if name else case


def _place(tokens, heads, kv_heads, dim, page, axes, form, packed, name=None):
    case = {"kind": "place", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page, "axes": axes, "form": form,
            "packed": packed}
    return dict(case, name=name) if name else case


def _sample(rows, vocabulary, dtype, form, softcap, masked, name=None):
    case = {"kind": "sample", "rows": rows, "vocabulary": vocabulary, "dtype": dtype, "form": form, "softcap": softcap, "masked": masked}
    return dict(case, name=name) if name else case


def listed():
    return [
        # one decode step of 64 requests at lengths of their own
        _plan(64, 7919, "1", 16, 64, name="plan_decode_64"),
        # four prompts that arrive together
        _plan(4, 0, "1500 1 2049 1058", 64, 512, name="plan_prompt_4608"),
        # a large batch with drafts to verify, slots without a request among them
        _plan(1000, 16000, "0-5", 16, 4096, name="plan_drafts_1000"),
        # drafts of 64 requests, most of which are rejected
        _trim(64, 7919, "drafts", 16, name="trim_drafts_64"),
        # every third request of a large batch has ended
        _trim(1000, 16000, "ended", 16, name="trim_ended_1000"),
        # one decode step of 64 requests with images behind them
        _place(64, 16, 8, 256, 16, 3, "decode", False, name="place_decode_64"),
        # prompts of text and images, whose packed keys the prompt attention reads
        _place(4608, 16, 8, 256, 64, 3, "image", True, name="place_image_4608"),
        # a chunk of video
        _place(16384, 32, 8, 128, 64, 3, "video", False, name="place_video_16384"),
        # one reply, token by token: latency
        _sample(1, 262144, "float32", "mixed", 0.0, False, name="sample_one"),
        # a decode batch, each request with settings of its own, capped logits in the type that a product leaves them in
        _sample(64, 262144, "bfloat16", "mixed", 30.0, True, name="sample_mixed_64"),
        # many rollouts from the distribution as it is, an odd vocabulary
        _sample(256, 50257, "float32", "open", 0.0, False, name="sample_open_256"),
        # many requests that keep the nucleus
        _sample(256, 128000, "float32", "nucleus", 0.0, False, name="sample_nucleus_256"),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["plan", "trim", "place", "sample", "sample"])
    page = rng.choice([16, 32, 64, 128, 256])
    if kind == "plan":
        sequences = _log_int(rng, 1, 1200)
        if sequences <= 16 and rng.random() < 0.6:
            news = " ".join(str(_log_int(rng, 1, 2500)) for _ in range(sequences))
        else:
            news = rng.choice(["1", "0-1", "0-5", "1-5", "0-40"])
        return _plan(sequences, _log_int(rng, 1, 16000), news, page, _log_int(rng, 1, 4096))
    if kind == "trim":
        return _trim(_log_int(rng, 1, 1200), _log_int(rng, 1, 16000), rng.choice(["drafts", "ended", "cut"]), page)
    if kind == "place":
        dim = rng.choice([64, 128, 256, 512])
        kv_heads = rng.randint(1, 8 if dim < 512 else 4)
        heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 7, 8])
        most = 16384 * 48 * 128 // ((heads + 2 * kv_heads) * dim)  # (the bytes of the largest listed case)
        return _place(_log_int(rng, 1, max(1, min(12000, most))), heads, kv_heads, dim, page, rng.choice([1, 2, 3, 3, 4]),
                      rng.choice(["decode", "image", "video"]), rng.random() < 0.5)
    vocabulary = _log_int(rng, 1, 262144)
    return _sample(_log_int(rng, 1, max(1, min(2000, 256 * 128000 // vocabulary))), vocabulary, rng.choice(["float32", "bfloat16"]),
                   rng.choice(["mixed", "mixed", "open", "nucleus", "top", "floor", "greedy"]), rng.choice([0.0, 0.0, 30.0]), rng.random() < 0.4)


# ---- inputs ------------------------------------------------------------------------------------------

def _randn(gen, *shape, mean=0.0, std=1.0):
    return (torch.randn(*shape, generator=gen, device=DEVICE, dtype=torch.float32) * std + mean).to(torch.bfloat16)


def _randint(gen, low, high, *shape):
    """Whole numbers from low to high, both among them."""
    return torch.randint(low, high + 1, shape, generator=gen, device=DEVICE, dtype=torch.int32)


def _rand(gen, *shape):
    return torch.rand(*shape, generator=gen, device=DEVICE, dtype=torch.float32)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed * 1000003 + 29)
    st = {"case": case}
    {"plan": _prepare_pages, "trim": _prepare_pages, "place": _prepare_place, "sample": _prepare_sample}[case["kind"]](st, case, gen)
    return st


def _prepare_pages(st, case, gen):
    """Requests that hold pages out of a pool, in no order, as a server has them after some time."""
    sequences, page = case["sequences"], case["page"]
    # lengths from nothing on, short ones more often
    lengths = (_rand(gen, sequences) ** 2 * (case["most_past"] + 1)).to(torch.int32)
    news = torch.zeros_like(lengths)
    if case["kind"] == "plan":
        low, high = _news(case)
        news = torch.tensor(low, dtype=torch.int32, device=DEVICE) if isinstance(low, list) else _randint(gen, low, high, sequences)
        if case["most_past"] == 0:
            lengths.zero_()
        # (positions of requests with images run behind their numbers of tokens)
        st["shift"] = -_randint(gen, 0, 300, sequences).clamp_(max=lengths)
    else:
        dropped = {"drafts": _randint(gen, 0, 5, sequences), "cut": (_rand(gen, sequences) * (lengths + 1)).to(torch.int32),
                   "ended": torch.where(_randint(gen, 0, 2, sequences) == 0, lengths, 0)}[case["form"]]
        st["keep"] = (lengths - dropped).clamp_(min=0).to(torch.int32)
    held = (lengths + page - 1) // page
    # a table as wide as the longest request may need, a pool as large as the requests together do; rows for the most tokens
    longest = case["most_past"] + (_news(case)[1] if case["kind"] == "plan" else 0)
    width = -(-longest // page) + 1
    taken = int(held.sum())
    pages = sequences * (width if sequences <= 64 else width // 2 + 2) + case.get("spare", 64)
    st["free"] = torch.randperm(pages, generator=gen, device=DEVICE).to(torch.int32)
    # what requests hold is what the pool's list has in front, handed out in another order
    order = st["free"][:taken][torch.randperm(taken, generator=gen, device=DEVICE)]
    table = torch.full((sequences, width), -1, dtype=torch.int32, device=DEVICE)
    table[torch.arange(width, device=DEVICE)[None] < held[:, None]] = order
    st["table"], st["lengths"], st["news"] = table, lengths, news
    st["taken"] = torch.tensor([taken], dtype=torch.int32, device=DEVICE)
    st["tokens"] = _rows(case) if case["kind"] == "plan" else 0
    if own:
        from gevva_b200 import step
        st["pool"] = step.PagePool(st["free"], st["taken"])


def _news(case):
    """(least, most) new tokens of a request, or (list, the longest of it)."""
    text, sequences = case["news"], case["sequences"]
    if "-" in text:
        low, high = (int(t) for t in text.split("-"))
        return low, high
    counts = [int(t) for t in text.split()]
    return (counts, max(counts)) if len(counts) == sequences else (counts[0], counts[0])


def _rows(case):
    """Rows of the step's tensors: those of its tokens, as many as there may be where their number goes by the step."""
    low, high = _news(case)
    return sum(low) if isinstance(low, list) else case["sequences"] * high


def _positions(case, gen):
    """int32 [axes, tokens]: text counts on along all axes, images and frames spread over rows and columns."""
    tokens, axes, form = case["tokens"], case["axes"], case["form"]
    if form == "decode":
        return _randint(gen, 0, 30000, 1, tokens).expand(axes, tokens).contiguous()
    at = torch.arange(tokens, device=DEVICE)
    grid, columns = (1024, 32) if form == "image" else (576, 24)
    block, inside = at // grid, at % grid
    visual = (block % 2 == 1) if form == "image" else torch.ones_like(block, dtype=torch.bool)
    start = 700 + (block * 64 if form == "image" else block)
    along = [start, start + inside // columns, start + inside % columns, start + inside % 7]
    return torch.stack([torch.where(visual, along[a], start + inside) for a in range(axes)]).to(torch.int32)


def _prepare_place(st, case, gen):
    tokens, heads, kv_heads, dim, page, axes = (case[n] for n in ("tokens", "heads", "kv_heads", "dim", "page", "axes"))
    qkv = _randn(gen, tokens, heads + 2 * kv_heads, dim, std=2.0)  # the rows of one projection
    st["q"], st["k"], st["v"] = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
    st["q_weight"], st["k_weight"] = _randn(gen, dim, mean=1.0, std=0.2), _randn(gen, dim, mean=1.0, std=0.2)
    pages = -(-tokens // page) + 3
    st["k_cache"], st["v_cache"] = _randn(gen, pages, page, kv_heads, dim), _randn(gen, pages, page, kv_heads, dim)
    if case["form"] == "decode":  # every token in another request's page
        slots = torch.randperm(pages * page, generator=gen, device=DEVICE)[:tokens]
    else:
        order = torch.randperm(pages, generator=gen, device=DEVICE)
        at = torch.arange(tokens, device=DEVICE) + 5
        slots = order[at // page] * page + at % page
    st["slots"] = slots.to(torch.int32)
    st["positions"] = _positions(case, gen)
    # each pair turns along one axis, the axes in turn
    half = dim // 2
    base = 1e4 ** (-torch.arange(half, dtype=torch.float64, device=DEVICE) / half)
    mine = torch.arange(half, device=DEVICE)[None] % axes == torch.arange(axes, device=DEVICE)[:, None]
    st["frequencies"] = torch.where(mine, base, torch.zeros_like(base))
    if own:
        from gevva_b200 import attention
        st["cache"] = attention.KvCache(st["k_cache"], st["v_cache"])


def _prepare_sample(st, case, gen):
    """Logits with a wide bulk and a few dozen tokens ahead of it, surer in some rows than in others."""
    rows, vocabulary = case["rows"], case["vocabulary"]
    logits = torch.randn(rows, vocabulary, generator=gen, device=DEVICE, dtype=torch.float32)
    logits *= 1.0 + 1.5 * _rand(gen, rows, 1)
    ahead = torch.randint(0, vocabulary, (rows, 40), generator=gen, device=DEVICE)
    logits.scatter_reduce_(1, ahead, 3.0 + 14.0 * _rand(gen, rows, 1) * _rand(gen, rows, 40), "amax")
    if case["masked"]:
        # a grammar leaves some rows a part of the vocabulary, masked by infinity or by the type's lowest value
        kind = torch.arange(rows, device=DEVICE)[:, None] % 4
        out = _rand(gen, rows, vocabulary) < 0.9
        lowest = torch.finfo(getattr(torch, case["dtype"])).min
        logits = torch.where((kind == 1) & out, torch.full_like(logits, -math.inf), logits)
        logits = torch.where((kind == 2) & out, torch.full_like(logits, lowest), logits)
    st["logits"] = logits.to(getattr(torch, case["dtype"]))
    st["uniforms"] = _rand(gen, rows)
    form = case["form"]
    pick = lambda *values: torch.tensor(values, dtype=torch.float32, device=DEVICE)[_randint(gen, 0, len(values) - 1, rows).long()]
    st["temperature"] = {"greedy": pick(0.0), "mixed": pick(0.0, 0.6, 0.8, 1.0, 1.0, 1.3)}.get(form, pick(0.7, 1.0))
    st["top_k"] = {"mixed": pick(0, 1, 20, 50, 64, 100).int(), "top": pick(1, 2, 40, 50, 300, 1000, 5000).int()}.get(form)
    st["top_p"] = {"mixed": pick(0.5, 0.9, 0.95, 1.0, 1.0), "nucleus": pick(0.8, 0.9, 0.95)}.get(form)
    st["min_p"] = {"mixed": pick(0.0, 0.0, 0.05, 0.1), "floor": pick(0.01, 0.05, 0.1)}.get(form)


# ---- one pass ----------------------------------------------------------------------------------------

def run(st):
    return {"plan": _run_plan, "trim": _run_trim, "place": _run_place, "sample": _run_sample}[st["case"]["kind"]](st)


def _step():
    from gevva_b200 import step
    return step


def _run_plan(st):
    page, tokens = st["case"]["page"], st["tokens"]
    if own:
        plan = _step().plan_step(st["lengths"], st["news"], st["table"], st["pool"], page, tokens, shift=st["shift"])
        return plan.token_offsets, plan.lengths, plan.slots, plan.positions, plan.taken, st["table"]
    lengths, news, table = st["lengths"].long(), st["news"].long(), st["table"]
    after = lengths + news
    held, needed = (lengths + page - 1) // page, (after + page - 1) // page
    offsets = torch.cat([torch.zeros_like(news[:1]), news.cumsum(0)])
    more = needed - held
    first = st["taken"].long() + more.cumsum(0) - more  # of a request's new pages in the pool's list
    column = torch.arange(table.shape[1], device=DEVICE)[None]
    fresh = (column >= held[:, None]) & (column < needed[:, None])
    which = (first[:, None] + column - held[:, None]).clamp(0, st["free"].numel() - 1)
    table.copy_(torch.where(fresh, st["free"][which], table))
    row = torch.arange(tokens, device=DEVICE)
    sequence = torch.searchsorted(offsets[1:], row, right=True).clamp_(max=len(news) - 1)
    position = row - offsets[sequence] + lengths[sequence]
    # (rows behind the last request's have no slot)
    some = row < offsets[-1]
    slots = torch.where(some, table[sequence, (position // page).clamp(max=table.shape[1] - 1)].long() * page + position % page, -1)
    position = torch.where(some, position + st["shift"][sequence], 0)
    taken = st["taken"] + more.sum().int()
    return offsets.int(), after.int(), slots.int(), position.int(), taken, table


def _run_trim(st):
    page = st["case"]["page"]
    if own:
        trimmed = _step().trim_step(st["lengths"], st["keep"], st["table"], st["pool"], page)
        return trimmed.lengths, trimmed.taken, st["free"]
    lengths = st["lengths"].long()
    after = torch.minimum(lengths, st["keep"].long().clamp(min=0))
    held, needed = (lengths + page - 1) // page, (after + page - 1) // page
    less = held - needed
    taken = st["taken"] - less.sum().int()
    # request after request, each one's pages in the order in which it held them: as plan_step would hand them out again
    column = torch.arange(st["table"].shape[1], device=DEVICE)[None]
    back = (column >= needed[:, None]) & (column < held[:, None])
    at = taken.long() + (less.cumsum(0) - less)[:, None] + column - needed[:, None]
    # (what does not go back is written to a place behind the list)
    longer = torch.cat([st["free"], st["free"][:1]])
    longer[torch.where(back, at, len(longer) - 1)] = st["table"]
    st["free"].copy_(longer[:-1])
    return after.int(), taken, st["free"]


def _rms(x, weight):
    y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
    return y if weight is None else y * weight.float()


def _run_place(st):
    packed = st["case"]["packed"]
    if own:
        out = _step().kv_append_at(st["q"], st["k"], st["v"], st["cache"], st["slots"], st["positions"], st["frequencies"],
                                   q_weight=st["q_weight"], k_weight=st["k_weight"], normalize_v=True, eps=EPS, packed=packed)
        out = tuple(out) if packed else (out,)
        return (*out, st["k_cache"], st["v_cache"])
    angle = st["positions"].double().T @ st["frequencies"]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    half = cos.shape[-1]

    def rotate(x):
        a, b = x[..., :half], x[..., half:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(torch.bfloat16)

    q, k = rotate(_rms(st["q"].float(), st["q_weight"])), rotate(_rms(st["k"].float(), st["k_weight"]))
    v = _rms(st["v"].float(), None).to(torch.bfloat16)
    slots = st["slots"].long()
    st["k_cache"].flatten(0, 1)[slots] = k
    st["v_cache"].flatten(0, 1)[slots] = v
    out = (q, k, v) if packed else (q,)
    return (*out, st["k_cache"], st["v_cache"])


def _run_sample(st):
    case, logits = st["case"], st["logits"]
    if own:
        return _step().sample_tokens(logits, st["uniforms"], temperature=st["temperature"], top_k=st["top_k"], top_p=st["top_p"],
                                     min_p=st["min_p"], softcap=case["softcap"], probability=True)
    vocabulary = logits.shape[1]
    temperature = st["temperature"].double()[:, None]
    ordered, index = logits.sort(dim=1, descending=True, stable=True)
    y = ordered.double()
    if case["softcap"]:
        y = case["softcap"] * torch.tanh(y / case["softcap"])
    weight = torch.exp((y - y[:, :1]) / torch.where(temperature > 0, temperature, 1.0))
    weight = torch.where(ordered > -math.inf, weight, 0.0)
    rank = torch.arange(vocabulary, device=DEVICE)[None]
    kept = (temperature > 0) | (rank == 0)
    if st["top_k"] is not None:
        top_k = st["top_k"][:, None]
        kept &= (top_k <= 0) | (rank < top_k)
    weight = torch.where(kept, weight, 0.0)
    floor = torch.zeros_like(weight[:, :1]) if st["min_p"] is None else st["min_p"].double()[:, None]
    if st["top_p"] is not None:
        top_p = st["top_p"].double()[:, None]
        upto = weight.cumsum(1)
        kept = (top_p >= 1) | (rank == 0) | (upto - weight < top_p * upto[:, -1:])
        weight = torch.where(kept, weight, 0.0)
    weight = torch.where(weight >= floor, weight, 0.0)
    # the running sum over the vocabulary passes the random number's share of the whole
    weight = torch.zeros_like(weight).scatter_(1, index, weight)
    upto = weight.cumsum(1)
    share = st["uniforms"].double()[:, None] * upto[:, -1:]
    token = torch.searchsorted(upto, share, right=True).clamp_(max=vocabulary - 1)
    probability = weight.gather(1, token) / upto[:, -1:]
    some = upto[:, -1] > 0  # (a row whose mask leaves nothing has no token)
    return torch.where(some, token[:, 0], -1).int(), torch.where(some, probability[:, 0], 0.0).float()


# ---- the definitions ---------------------------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    return {"plan": _exact_plan, "trim": _exact_trim, "place": _exact_place, "sample": _exact_sample}[case["kind"]](st)


def _exact_plan(st):
    """One request and one token after the other, on the host."""
    page = st["case"]["page"]
    lengths, news, shift, free = (st[n].tolist() for n in ("lengths", "news", "shift", "free"))
    table, taken = st["table"].tolist(), int(st["taken"])
    offsets, slots, positions = [0], [], []
    for s, (length, more) in enumerate(zip(lengths, news)):
        for x in range(length, length + more):
            if x % page == 0:
                table[s][x // page] = free[taken]
                taken += 1
            slots.append(table[s][x // page] * page + x % page)
            positions.append(x + shift[s])
        offsets.append(offsets[-1] + more)
    after = [a + b for a, b in zip(lengths, news)]
    behind = st["tokens"] - offsets[-1]
    slots, positions = slots + [-1] * behind, positions + [0] * behind
    return tuple(torch.tensor(x, dtype=torch.int32) for x in (offsets, after, slots, positions, [taken], table))


def _exact_trim(st):
    page = st["case"]["page"]
    lengths, keep, table, free = (st[n].tolist() for n in ("lengths", "keep", "table", "free"))
    taken = int(st["taken"])
    for s in reversed(range(len(lengths))):
        while lengths[s] > max(keep[s], 0):
            lengths[s] -= 1
            if lengths[s] % page == 0:
                taken -= 1
                free[taken] = table[s][lengths[s] // page]
    return tuple(torch.tensor(x, dtype=torch.int32) for x in (lengths, [taken], free))


def _exact_place(st):
    def normed(x, weight):
        x = x.double()
        x = x / ((x ** 2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt()
        return x if weight is None else x * weight.double()

    half = st["frequencies"].shape[1]
    angle = sum(torch.outer(p.double(), f) for p, f in zip(st["positions"], st["frequencies"]))
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]

    def turned(x):
        z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * turn
        return torch.cat([z.real, z.imag], -1)

    q, k, v = turned(normed(st["q"], st["q_weight"])), turned(normed(st["k"], st["k_weight"])), normed(st["v"], None)
    caches = []
    for cache, rows in ((st["k_cache"], k), (st["v_cache"], v)):
        whole = cache.double()
        whole.view(-1, *cache.shape[2:]).index_copy_(0, st["slots"].long(), rows)
        caches.append(whole)
    return (q, k, v, *caches) if st["case"]["packed"] else (q, *caches)


def _exact_sample(st):
    """Row after row on the host: the tokens in front, as many as each rule keeps, and then a walk over the vocabulary."""
    cap = st["case"]["softcap"]
    logits = st["logits"].float().cpu().numpy().astype(np.float64)
    settings = {n: None if st[n] is None else st[n].cpu().numpy().astype(np.float64) for n in ("uniforms", "temperature", "top_k", "top_p", "min_p")}
    tokens, shares = [], []
    for r, row in enumerate(logits):
        one = {n: None if x is None else x[r] for n, x in settings.items()}
        order = np.argsort(-row, kind="stable")
        order = order[row[order] > -np.inf]
        if not len(order):
            tokens.append(-1)
            shares.append(0.0)
            continue
        if one["temperature"] <= 0:
            order = order[:1]
        if one["top_k"] is not None and one["top_k"] > 0:
            order = order[:int(one["top_k"])]
        y = row[order]
        if cap:
            y = cap * np.tanh(y / cap)
        w = np.exp((y - y[0]) / (one["temperature"] if one["temperature"] > 0 else 1.0))
        if one["top_p"] is not None and one["top_p"] < 1:
            through = np.cumsum(w)
            count = max(1, int(np.searchsorted(through, one["top_p"] * through[-1], side="left")) + 1)
            order, w = order[:count], w[:count]
        if one["min_p"] is not None:
            order, w = order[w >= one["min_p"]], w[w >= one["min_p"]]
        by_index = np.argsort(order)
        order, w = order[by_index], w[by_index]
        through = np.cumsum(w)
        at = min(int(np.searchsorted(through, one["uniforms"] * through[-1], side="right")), len(w) - 1)
        tokens.append(int(order[at]))
        shares.append(w[at] / through[-1])
    return torch.tensor(tokens, dtype=torch.int32), torch.tensor(shares, dtype=torch.float64)


def work(case):
    if case["kind"] == "plan":
        sequences, (low, high) = case["sequences"], _news(case)
        tokens = sum(low) if isinstance(low, list) else sequences * (low + high) // 2
        pages = -(-tokens // case["page"])
        # lengths, news and shifts in, offsets and lengths out; a slot and a position a token; new pages from the list to the table
        return {"bytes": 4 * (5 * sequences + 2 * _rows(case) + 2 * pages + 3), "flops": 0}
    if case["kind"] == "trim":
        sequences = case["sequences"]
        mean = case["most_past"] // 3
        pages = sequences * {"drafts": 5 / 2, "ended": mean / 3, "cut": mean / 2}[case["form"]] / case["page"]
        return {"bytes": int(4 * (3 * sequences + 2 * pages + 2)), "flops": 0}
    if case["kind"] == "place":
        tokens, heads, kv_heads, dim = case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        read = heads + 2 * kv_heads
        written = read + (2 * kv_heads if case["packed"] else 0)
        return {"bytes": 2 * dim * tokens * (read + written) + 4 * tokens * (1 + case["axes"]), "flops": 8 * dim * tokens * read}
    size = 4 if case["dtype"] == "float32" else 2
    return {"bytes": case["rows"] * (case["vocabulary"] * size + 28), "flops": 4 * case["rows"] * case["vocabulary"]}
