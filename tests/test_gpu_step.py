"""What a serving step has around its layers, through its Python mirror, against plain forms on the host.

Whole numbers have to be equal.  A token is compared where no rule's border lies within 2^-40 of the whole of what decides it: shares are off by at
most 2^-42.8 of themselves (tests/test_step_shares.py), and so are their sums, whatever the order.  (Capped ones by 2^-53 of the cap over
the temperature more: 2^-43 of themselves at a cap of 30 and a temperature of 0.03.)  Probabilities are rounded once to 32 bits
(2^-24), of numbers that are off by much less."""
import math

import numpy as np
import pytest
import torch

from gevva_b200 import attention as attn
from gevva_b200 import step
from tests import attention_ref, step_ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
NEAR = 2.0 ** -40


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


# ---- pages and places ----------------------------------------------------------------------------------

def requests(seed, sequences, page, past, width=None):
    rng = np.random.default_rng(seed)
    lengths = [int(x) for x in rng.integers(0, past + 1, sequences)]
    width = width or past // page + 8
    held = [-(-n // page) for n in lengths]
    pages = sum(held) + sequences * 8
    free = [int(x) for x in rng.permutation(pages)]
    given = list(rng.permutation(free[:sum(held)]))
    table = [[-7] * width for _ in lengths]
    for s, n in enumerate(held):
        for i in range(n):
            table[s][i] = int(given.pop())
    return rng, lengths, table, free, sum(held)


@pytest.mark.parametrize("sequences,page,past,most", [(1, 16, 0, 1), (1, 16, 100, 1), (1, 64, 500, 300), (2, 16, 0, 0), (3, 256, 700, 900), (33, 16, 40, 5),
                                                      (64, 32, 3000, 1), (257, 16, 90, 40), (1025, 16, 50, 2), (3000, 16, 20, 3)])
@pytest.mark.parametrize("padded", [0, 1, 77])
def test_plan(sequences, page, past, most, padded):
    rng, lengths, table, free, taken = requests(sequences + page, sequences, page, past, width=past // page + most // page + 8)
    free = free + list(range(len(free), len(free) + sequences * (most // page + 1)))
    news = [int(x) for x in rng.integers(0, most + 1, sequences)]
    shift = [int(x) for x in rng.integers(-50, 50, sequences)] if sequences % 2 else None
    tokens = sum(news) + padded
    want = step_ref.plan(lengths, news, table, free, taken, page, tokens, shift)
    # a table whose rows lie further apart
    wide = torch.full((sequences, len(table[0]) + 5), -9, dtype=torch.int32, device=DEV)
    rows = wide[:, :len(table[0])]
    rows.copy_(ints(table))
    pool = step.PagePool(ints(free), ints([taken]))
    plan = step.plan_step(ints(lengths), ints(news), rows, pool, page, tokens, shift=None if shift is None else ints(shift))
    pool.check()
    got = (plan.token_offsets, plan.lengths, plan.slots, plan.positions, plan.taken, rows)
    for a, b, name in zip(got, want, ("offsets", "lengths", "slots", "positions", "taken", "table")):
        assert a.flatten().tolist() == np.array(b).flatten().tolist(), name
    assert (wide[:, len(table[0]):] == -9).all() and pool.taken.item() == taken


def test_plan_of_as_many_requests_as_there_may_be():
    n = step.MAX_REQUESTS
    lengths, news = [i % 33 for i in range(n)], [(i * 7) % 5 for i in range(n)]
    table = torch.full((n, 4), -1, dtype=torch.int32)
    held = [-(-x // 16) for x in lengths]
    taken = 0
    for s, h in enumerate(held):
        for i in range(h):
            table[s, i] = taken
            taken += 1
    free = list(range(3 * n))
    want = step_ref.plan(lengths, news, table.tolist(), free, taken, 16, sum(news))
    pool, rows = step.PagePool(ints(free), ints([taken])), table.to(DEV)
    plan = step.plan_step(ints(lengths), ints(news), rows, pool, 16, sum(news))
    pool.check()
    assert plan.slots.tolist() == want[2] and plan.positions.tolist() == want[3] and rows.tolist() == want[5] and plan.taken.item() == want[4]
    back = step.trim_step(plan.lengths, ints(lengths), rows, step.PagePool(pool.free, plan.taken), 16)
    assert back.lengths.tolist() == lengths and back.taken.item() == taken and pool.free.tolist() == free
    with pytest.raises(ValueError, match="at most"):
        step.plan_step(ints([0] * (n + 1)), ints([0] * (n + 1)), torch.zeros(n + 1, 1, dtype=torch.int32, device=DEV), pool, 16, 0)


@pytest.mark.parametrize("what", ["pages", "rows", "news", "lengths", "table", "taken", "taken too many"])
def test_plan_that_cannot_be_changes_nothing(what):
    lengths, news, taken = [5, 40, 16], [1, 30, 17], 5
    table, free = [[0, -1, -1, -1, -1, -1], [1, 2, 3, -1, -1, -1], [4, -1, -1, -1, -1, -1]], list(range(9))
    tokens, status = 48, -7
    if what == "pages":
        free, status = list(range(8)), -8
    elif what == "rows":
        tokens, status = 47, -6
    elif what == "news":
        news[1] = -1
    elif what == "lengths":
        lengths[0] = -1
    elif what == "table":
        lengths[2], news[2] = 90, 7
    elif what == "taken":
        taken, status = -1, -8
    else:
        taken, status = 10, -8
    pool, rows, before = step.PagePool(ints(free), ints([taken])), ints(table), ints(lengths)
    plan = step.plan_step(before, ints(news), rows, pool, 16, tokens)
    assert plan.token_offsets.tolist() == [0] * 4 and plan.lengths.tolist() == lengths and plan.taken.item() == taken
    assert set(plan.slots.tolist()) == {-1} and set(plan.positions.tolist()) == {0} and rows.tolist() == table
    assert pool.last_status() == status and pool.last_status() == 0
    if what == "pages":  # with one page more it can be
        pool = step.PagePool(ints(list(range(9))), ints([taken]))
        plan = step.plan_step(before, ints(news), rows, pool, 16, tokens)
        pool.check()
        assert plan.taken.item() == 9


def test_a_page_that_is_none_gives_no_slot():
    pool, table = step.PagePool(ints([5, -3, 1 << 28]), ints([0])), ints([[-1, 0, 0], [7, 0, 0], [0, 0, 0], [0, 0, 0]])
    plan = step.plan_step(ints([3, 3, 0, 0]), ints([1, 1, 1, 1]), table, pool, 16, 4)
    assert plan.slots.tolist() == [-1, 7 * 16 + 3, 5 * 16, -1] and pool.last_status() == -7  # (-1 * 16 + 3 and -3 * 16 are below zero)


def test_steps_in_place_and_back():
    rng, lengths, table, free, taken = requests(3, 40, 16, 60, width=20)
    pool, rows, state = step.PagePool(ints(free), ints([taken])), ints(table), ints(lengths)
    plan = step.StepPlan.in_place(state, rows, pool, 400)
    history = [(lengths, list(free), taken)]
    for _ in range(5):
        news = [int(x) for x in rng.integers(0, 10, 40)]
        want = step_ref.plan(lengths, news, table, free, taken, 16, 400)
        got = step.plan_step(state, ints(news), rows, pool, 16, 400, out=plan)
        assert got is plan and state.tolist() == want[1] and pool.taken.item() == want[4] and rows.tolist() == want[5]
        assert plan.slots.tolist() == want[2] and plan.batch.lengths is state
        lengths, taken, table = want[1], want[4], want[5]
        history.append((lengths, list(free), taken))
    for lengths, free, taken in reversed(history[:-1]):
        step.trim_step(state, ints(lengths), rows, pool, 16, out=step.Trimmed(state, pool.taken))
        assert state.tolist() == lengths and pool.free.tolist() == free and pool.taken.item() == taken
    pool.check()


@pytest.mark.parametrize("sequences,page,past", [(1, 16, 0), (1, 16, 2000), (5, 64, 300), (64, 16, 900), (1030, 16, 60)])
@pytest.mark.parametrize("form", ["all", "none", "some", "cut"])
def test_trim(sequences, page, past, form):
    rng, lengths, table, free, taken = requests(sequences * 3 + page, sequences, page, past)
    keep = {"all": [0] * sequences, "none": [n + int(rng.integers(0, 3)) for n in lengths], "some": [0 if rng.random() < 0.4 else n for n in lengths],
            "cut": [int(rng.integers(-2, n + 1)) for n in lengths]}[form]
    want = step_ref.trim(lengths, keep, table, free, taken, page)
    pool = step.PagePool(ints(free), ints([taken]))
    got = step.trim_step(ints(lengths), ints(keep), ints(table), pool, page)
    pool.check()
    assert got.lengths.tolist() == want[0] and pool.free.tolist() == want[1] and got.taken.item() == want[2]


def test_trim_that_cannot_be_changes_nothing():
    free, table = list(range(20)), [[3, 4, 5], [6, 7, 8]]
    for lengths, taken, status in (([40, 40], 5, -8), ([-1, 3], 9, -7), ([49, 3], 9, -7), ([3, 3], 21, -8)):
        pool = step.PagePool(ints(free), ints([taken]))
        got = step.trim_step(ints(lengths), ints([0, 0]), ints(table), pool, 16)
        assert got.lengths.tolist() == lengths and got.taken.item() == taken and pool.free.tolist() == free and pool.last_status() == status


# ---- the append at given places --------------------------------------------------------------------------

def randn(gen, *shape, std=1.0):
    return (torch.randn(*shape, generator=gen, device=DEV) * std).to(torch.bfloat16)


def generator(seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    return gen


def cases_of_append():
    for dim, heads, kv_heads, tokens, page, axes, pairs in ((64, 4, 2, 5, 16, 3, 32), (128, 3, 1, 1, 16, 1, 64), (256, 16, 8, 64, 64, 2, 64), (512, 2, 2, 40, 32, 4, 256),
                                                            (128, 8, 1, 700, 16, 3, 48), (64, 1, 1, 1300, 128, 16, 8), (256, 1, 1, 3, 16, 1, 0)):
        for packed in (False, True):
            yield dim, heads, kv_heads, tokens, page, axes, pairs, packed


@pytest.mark.parametrize("dim,heads,kv_heads,tokens,page,axes,pairs,packed", list(cases_of_append()))
def test_append_at(dim, heads, kv_heads, tokens, page, axes, pairs, packed):
    gen = generator(dim + tokens)
    qkv = randn(gen, tokens, heads + 2 * kv_heads, dim, std=2.0)
    q, k, v = qkv.split((heads, kv_heads, kv_heads), 1)
    pages = -(-tokens // page) + 2
    cache = attn.KvCache(randn(gen, pages, page, kv_heads, dim), randn(gen, pages, page, kv_heads, dim))
    kc, vc = cache.k.clone(), cache.v.clone()
    slots = torch.randperm(pages * page, generator=gen, device=DEV)[:tokens].to(torch.int32)
    slots[torch.rand(tokens, generator=gen, device=DEV) < 0.2] = -1
    positions = torch.randint(-100, 1 << 20, (axes, tokens), generator=gen, device=DEV, dtype=torch.int32)
    frequencies = torch.rand(axes, pairs, generator=gen, device=DEV, dtype=torch.float64) if pairs else None
    if pairs and axes > 1:  # most pairs follow one axis, some several
        mine = torch.arange(pairs, device=DEV)[None] % axes == torch.arange(axes, device=DEV)[:, None]
        frequencies = torch.where(mine | (torch.arange(pairs, device=DEV) % 5 == 0), frequencies, 0.0)
    qw, kw = randn(gen, dim), (randn(gen, dim) if tokens % 2 else None)
    mark = torch.full((tokens, heads, dim), 77.0, dtype=torch.bfloat16, device=DEV)
    got = step.kv_append_at(q, k, v, cache, slots, positions if axes > 1 else positions[0], frequencies, qw, kw, True, 1e-6, packed, out=mark.clone())
    cache.check()
    angle = None if not pairs else positions.double().T @ frequencies
    real = slots >= 0

    def turned(x, weight):
        y = attention_ref.norm(x, weight, 1e-6) if weight is not None else x.double()
        if not pairs:
            return y, y.abs()
        a, b, rest = y[..., :pairs], y[..., pairs:2 * pairs], y[..., 2 * pairs:]
        c, s = angle.cos()[:, None], angle.sin()[:, None]
        both = a.abs() + b.abs()
        return torch.cat([a * c - b * s, b * c + a * s, rest], -1), torch.cat([both, both, rest.abs()], -1)

    # a value is rounded to bf16; the norm's sum of dim squares, its root and products, the sine (of an angle in half turns rounded to
    # 32 bits: 2^-24 of at most one, times pi) and the rotation are in 32 bits
    def bound(want, sizes):
        return attention_ref.BF16 * want.abs() + sizes * (dim + 40) * attention_ref.FP32

    wq, sq = turned(q, qw)
    wk, sk = turned(k, kw)
    wv = attention_ref.norm(v, None, 1e-6)
    queries = got.q if packed else got
    attention_ref.within(queries[real], wq[real], bound(wq, sq)[real], "queries")
    assert (queries[~real] == 77.0).all()
    at = slots[real].long()
    for cached, before, want, sizes, name in ((cache.k, kc, wk, sk, "keys"), (cache.v, vc, wv, wv.abs(), "values")):
        flat, whole = cached.flatten(0, 1), before.flatten(0, 1)
        attention_ref.within(flat[at], want[real], bound(want, sizes)[real], name)
        rest = torch.ones(pages * page, dtype=torch.bool, device=DEV)
        rest[at] = False
        assert torch.equal(flat[rest], whole[rest])
    if packed:
        attention_ref.within(got.k[real], wk[real], bound(wk, sk)[real], "packed keys")
        attention_ref.within(got.v[real], wv[real], bound(wv, wv.abs())[real], "packed values")


def test_one_axis_gives_the_bits_of_the_other_append():
    """Over plan_step's places and positions kv_append_at is kv_append, bit for bit."""
    gen = generator(5)
    news, lengths = [1, 70, 0, 33], [40, 0, 7, 100]
    tokens = sum(news)
    qkv = randn(gen, tokens, 8, 128)
    q, k, v = qkv.split((4, 2, 2), 1)
    pool, table = step.PagePool.whole(40, DEV), torch.full((4, 12), -1, dtype=torch.int32, device=DEV)
    empty = step.plan_step(ints([0] * 4), ints(lengths), table, pool, 16, sum(lengths))
    pool.taken = empty.taken
    plan = step.plan_step(empty.lengths, ints(news), table, pool, 16, tokens)
    frequencies = 1e4 ** (-torch.arange(64, dtype=torch.float64, device=DEV) / 64)
    caches = [attn.KvCache.empty(40, 16, 2, 128) for _ in range(3)]
    w = randn(gen, 128)
    one = attn.kv_append(q, k, v, caches[0], plan.batch, frequencies, w, w, True, packed=True)
    two = step.kv_append_at(q, k, v, caches[1], plan.slots, plan.positions, frequencies, w, w, True, packed=True)
    # three axes that say the same, an expanded tensor, each pair along one of them
    three = torch.where(torch.arange(64, device=DEV)[None] % 3 == torch.arange(3, device=DEV)[:, None], frequencies, 0.0)
    many = step.kv_append_at(q, k, v, caches[2], plan.slots, plan.positions.expand(3, tokens), three, w, w, True, packed=True)
    for other, cache in ((two, caches[1]), (many, caches[2])):
        for a, b in zip(one, other):
            assert torch.equal(a, b)
        assert torch.equal(cache.k, caches[0].k) and torch.equal(cache.v, caches[0].v)
        cache.check()


@pytest.mark.parametrize("tokens", [3, 800])
def test_append_at_slots_outside_the_cache(tokens):
    gen = generator(9)
    q, k, v = (randn(gen, tokens, h, 64) for h in (2, 1, 1))
    cache = attn.KvCache.empty(tokens // 16 + 1, 16, 1, 64)
    slots = torch.arange(tokens, dtype=torch.int32, device=DEV)
    slots[1] = cache.k.shape[0] * 16
    slots[2] = 0x7fffffff
    got = step.kv_append_at(q, k, v, cache, slots, slots, None)
    assert cache.last_status() == -7 and torch.equal(got, q)
    flat = cache.k.flatten(0, 1)
    assert torch.equal(flat[0], k[0]) and (flat[1:3] == 0).all() and torch.equal(flat[3:tokens], k[3:])


# ---- tokens from logits ------------------------------------------------------------------------------------

SETTINGS = {
    "open": {}, "greedy": dict(temperature=[0.0]), "cold and hot": dict(temperature=[0.05, 5.0, -1.0, 0.7]),
    "count": dict(top_k=[1, 2, 50, 64, 300, 0, 1000, 3000, -4, 1 << 30]), "sum": dict(top_p=[0.5, 0.9, 0.99, 1.0, 0.0, 0.1, 2.0]),
    "floor": dict(min_p=[0.1, 0.01, 1e-6, 1.0, 3.0, 0.0, -1.0], temperature=[1.0, 0.5, 1.5]),
    "all": dict(temperature=[0.8, 1.0, 1.3], top_k=[50, 0, 5, 700], top_p=[0.9, 1.0, 0.6, 0.999, 0.95], min_p=[0.0, 0.05]),
}


def settings(name, rows):
    kinds = dict(temperature=torch.float32, top_k=torch.int32, top_p=torch.float32, min_p=torch.float32)
    return {n: torch.tensor([x[i % len(x)] for i in range(rows)], dtype=kinds[n], device=DEV) for n, x in SETTINGS[name].items()}


def compare(logits, uniforms, given, softcap=0.0, most_near=0.2, off=0.0, **more):
    """`off`: by how much exponents may be off beyond the last bits of 64."""
    tokens, shares = step.sample_tokens(logits, uniforms, softcap=softcap, probability=True, **given, **more)
    rows = logits.float().cpu().numpy().astype(np.float64)
    host = {n: t.cpu().double().tolist() for n, t in given.items()}
    got, got_shares, u = tokens.tolist(), shares.double().tolist(), uniforms.double().tolist()
    near = 0
    for r in range(len(rows)):
        one = {n: x[r] for n, x in host.items()}
        if "top_k" in one:
            one["top_k"] = int(one["top_k"])
        token, share, border = step_ref.sample(rows[r], u[r], softcap=softcap, **one)
        if border < NEAR + 2 * off:
            near += 1
            continue
        assert got[r] == token, (r, one, got[r], token, border)
        assert abs(got_shares[r] - share) <= (2.0 ** -23 + 2 * off) * share, (r, one, got_shares[r], share)
    assert near <= most_near * len(rows)
    return tokens


def logits_of(kind, gen, rows, vocabulary, dtype):
    x = torch.randn(rows, vocabulary, generator=gen, device=DEV) * 2.5
    if kind == "ahead":
        x.scatter_reduce_(1, torch.randint(0, vocabulary, (rows, 30), generator=gen, device=DEV), 5 + 10 * torch.rand(rows, 30, generator=gen, device=DEV), "amax")
    elif kind == "near":  # nearly flat
        x *= 0.01
    elif kind == "ties":  # a few values only
        x = (x * 0.8).round()
    elif kind == "masked":
        out = torch.rand(rows, vocabulary, generator=gen, device=DEV) < 0.8
        row = torch.arange(rows, device=DEV)[:, None] % 3
        x = torch.where(out & (row == 0), -math.inf, torch.where(out & (row == 1), torch.finfo(dtype).min, torch.where(out, math.nan, x)))
    elif kind == "far":
        x *= 1e30
    elif kind == "rising":
        x = torch.linspace(-8, 8, vocabulary, device=DEV).expand(rows, -1) + 0.0
    return x.to(dtype)


@pytest.mark.parametrize("vocabulary", [1, 2, 3, 7, 33, 255, 1024, 1025, 2049, 5000, 16387, 50257, 131073])
@pytest.mark.parametrize("name", list(SETTINGS))
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sample(vocabulary, name, dtype):
    gen = generator(vocabulary)
    rows = 11 if vocabulary < 20000 else 4
    for kind in ("bulk", "ahead", "near", "masked", "rising"):
        logits = logits_of(kind, gen, rows, vocabulary, dtype)
        uniforms = torch.rand(rows, generator=gen, device=DEV)
        compare(logits, uniforms, settings(name, rows))


@pytest.mark.parametrize("name", ["open", "count", "sum", "floor", "all"])
@pytest.mark.parametrize("softcap", [30.0, 2.0])
@pytest.mark.parametrize("vocabulary", [100, 9000, 70001])
def test_capped(name, softcap, vocabulary):
    gen = generator(vocabulary + 1)
    for dtype in (torch.float32, torch.bfloat16):
        for kind in ("ahead", "masked"):
            compare(logits_of(kind, gen, 5, vocabulary, dtype), torch.rand(5, generator=gen, device=DEV), settings(name, 5), softcap)


@pytest.mark.parametrize("softcap", [1e-40, 1e-6, 0.02, 100.0, 1e3, 1e5, 1e8, 1e20, 1e38])
@pytest.mark.parametrize("vocabulary", [100, 9000, 70001])
def test_capped_by_any_size(softcap, vocabulary):
    """Caps far above the logits change next to nothing, those far below them leave ranks alone; temperatures on both sides of the cap's size.
    Two of five floors are one, to which
    the shares 1 - 2 exp(-2 |x| / cap) cap / T of values beyond 13 caps come nearer than can be told.  (Where |x| is over cap / 185, softened values are off by cap * 2^-51, of |x| <= 15 at most 2775 * 2^-51 = 1.3e-12 over T = 0.3, twice.)"""
    gen = generator(vocabulary + 3)
    for temperature in (0.3, 1.0, max(softcap, 1e-30)):
        for name in ("open", "count", "sum", "floor"):
            given = settings(name, 5)
            given["temperature"] = torch.full((5,), min(temperature, 1e37), device=DEV)
            for kind in ("ahead", "masked"):
                compare(logits_of(kind, gen, 5, vocabulary, torch.float32), torch.rand(5, generator=gen, device=DEV), given, softcap, off=1e-11, most_near=0.4)
            assert given["temperature"].isfinite().all()


@pytest.mark.parametrize("vocabulary", [100, 9000, 70001])
def test_hot(vocabulary):
    """Shares that are one, or next to it, at temperatures far above the logits.  (Two of seven floors are one, to which 1 - 10 / T comes nearer
    than can be told at 10^12.)"""
    gen = generator(vocabulary + 4)
    for temperature in (1e3, 1e12, 1e20, 1e36):
        for name in ("open", "count", "sum", "floor"):
            given = dict(settings(name, 7), temperature=torch.full((7,), temperature, device=DEV))
            compare(logits_of("masked", gen, 7, vocabulary, torch.bfloat16), torch.rand(7, generator=gen, device=DEV), given, most_near=0.3)


@pytest.mark.parametrize("vocabulary", [9000, 70001, 262144])
@pytest.mark.parametrize("softcap", [0.0, 1.0, 12.0, 40.0])
def test_borders_far_below_the_largest(vocabulary, softcap):
    """A border among many values whose shares are next to none, or whose cap leaves them as much as the largest.  (Shares of
    exp(-25) = 1.4e-11 of the whole lie between borders: 2 * 2^-40 = 1.8e-12 of it is near one, in one of eight rows, by top_p and by the number.)"""
    gen = generator(vocabulary + 7)
    rows = 6
    logits = torch.randn(rows, vocabulary, generator=gen, device=DEV) * torch.tensor([0.1, 1.0, 4.0, 0.5, 2.0, 8.0], device=DEV)[:, None] - 25.0
    logits.scatter_(1, torch.randint(0, vocabulary, (rows, 1), generator=gen, device=DEV), 0.0)
    for p in (1 - 2.0 ** -24, 1 - 2.0 ** -20, 0.9999, 0.99, 0.5):
        for temperature in (1.0, 1.5, 6.0):
            given = dict(temperature=torch.full((rows,), temperature, device=DEV), top_p=torch.full((rows,), p, device=DEV))
            u = torch.rand(rows, generator=gen, device=DEV)
            compare(logits, u, given, softcap, most_near=0.7)
            compare(logits, 1 - u * 2.0 ** -18, given, softcap, most_near=0.7)


@pytest.mark.parametrize("vocabulary", [100, 9000, 70001])
@pytest.mark.parametrize("softcap", [0.0, 30.0])
def test_settings_at_the_ends_of_their_types(vocabulary, softcap):
    gen = generator(vocabulary + 6)
    for temperature in (1e-45, 1e-38, 1e-31, 3e38, math.inf):
        for name in ("open", "count", "sum"):
            given = dict(settings(name, 7), temperature=torch.full((7,), temperature, device=DEV))
            compare(logits_of("masked", gen, 7, vocabulary, torch.bfloat16), torch.rand(7, generator=gen, device=DEV), given, softcap, off=1e-15)
    # no number: none of that rule, and of a random number zero; others are taken to be in [0, 1)
    logits = logits_of("bulk", gen, 5, vocabulary, torch.float32)
    u = torch.rand(5, generator=gen, device=DEV)
    nan = torch.full((5,), math.nan, device=DEV)
    zeros, ones = torch.zeros(5, device=DEV), torch.full((5,), 1 - 2.0 ** -24, device=DEV)
    assert torch.equal(step.sample_tokens(logits, u, top_p=nan, min_p=nan, softcap=softcap), step.sample_tokens(logits, u, softcap=softcap))
    assert torch.equal(step.sample_tokens(logits, u, temperature=nan, softcap=softcap), logits.argmax(1).int())
    for bad, same in ((nan, zeros), (zeros - 3, zeros), (zeros - math.inf, zeros), (zeros + 1, ones), (zeros + math.inf, ones)):
        for more in ({}, dict(top_p=zeros + 0.9), dict(top_k=torch.full((5,), 70, dtype=torch.int32, device=DEV))):
            assert torch.equal(step.sample_tokens(logits, bad, softcap=softcap, **more), step.sample_tokens(logits, same, softcap=softcap, **more))


@pytest.mark.parametrize("temperature", [1e-7, 1e-5, 1e-3, 0.05, 0.2, 0.24])
def test_capped_and_cold(temperature):
    """Values a few steps of 32 bits apart, whose shares are apart by ordinary factors at low temperatures.  (Softened values of up
    to 30 are off by 30 * 2^-51.3 here and 12 * 3 * 2^-53 there, a distance by twice that: 3e-14, over T.)"""
    gen = generator(5)
    for vocabulary in (64, 5000, 70001):
        logits = 12.0 + torch.rand(6, vocabulary, generator=gen, device=DEV) * temperature * 30
        given = dict(temperature=torch.full((6,), temperature, device=DEV))
        compare(logits, torch.rand(6, generator=gen, device=DEV), given, 30.0, off=3e-14 / temperature)
        compare(logits, torch.rand(6, generator=gen, device=DEV), dict(given, top_p=torch.full((6,), 0.8, device=DEV)), 30.0, off=3e-14 / temperature)


@pytest.mark.parametrize("name", list(SETTINGS))
@pytest.mark.parametrize("vocabulary", [300, 3001, 40000, 262144])
def test_ties(name, vocabulary):
    """Many equal logits: ties stay by index, and more of them than a list holds are counted.  (Sums of equal shares meet borders such as a half
    exactly; random numbers keep off them.)"""
    gen = generator(vocabulary + 2)
    for kind in ("ties", "flat", "two"):
        logits = logits_of("ties", gen, 6, vocabulary, torch.float32)
        if kind == "flat":
            logits = torch.full_like(logits, -3.25)
        elif kind == "two":
            logits = torch.where(torch.arange(vocabulary, device=DEV) % 3 == 0, 0.0, -0.0).expand(6, -1) - (torch.arange(6, device=DEV)[:, None] % 2) * 2.0
        given = settings(name, 6)
        if "top_p" in given:
            given["top_p"] = given["top_p"] * 0.99
        compare(logits.contiguous().to(torch.bfloat16), torch.rand(6, generator=gen, device=DEV), given, most_near=0.7)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_values_at_the_ends(dtype):
    inf, low, high = math.inf, torch.finfo(dtype).min, torch.finfo(dtype).max
    rows = [[-inf] * 6, [math.nan] * 6, [inf, 1, inf, -inf, 0, inf], [low] * 6, [high, low, 0, high, -inf, math.nan], [low, -inf, -inf, -inf, -inf, low],
            [-inf, -inf, 3, -inf, -inf, -inf], [0.0, -0.0, -0.0, 0.0, -inf, -0.0], [1e-38, 0, -1e-38, 2e-38, -2e-38, 0]]
    for width in (6, 2500, 30000):
        x = torch.full((len(rows), width), -inf)
        at = torch.linspace(0, width - 1, 6).long()
        x[:, at] = torch.tensor(rows, dtype=torch.float64).float()
        logits = x.to(dtype).to(DEV)
        for name in SETTINGS:
            for u in (0.0, 0.3, 0.9999999):
                compare(logits, torch.full((len(rows),), u, device=DEV), settings(name, len(rows)), most_near=1.0)


def test_random_numbers_at_the_ends():
    gen = generator(3)
    logits = logits_of("near", gen, 5, 3000, torch.float32)
    logits[:, 0] = logits[:, -1] = -math.inf
    u = torch.tensor([0.0, 1.0, -3.0, math.nan, 7.0], device=DEV)
    assert step.sample_tokens(logits, u).tolist() == [1, 2998, 1, 1, 2998]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocabulary", [9, 1001, 30011])
def test_rows_anywhere(dtype, vocabulary):
    """Views at every offset, rows that lie apart, one row for many; what lies around the rows is no logit."""
    gen = generator(vocabulary + 3)
    around = torch.full((3, vocabulary + 40), 1e30, device=DEV).to(dtype)
    for offset in range(9):
        view = around[:, offset:offset + vocabulary]
        view.copy_(logits_of("ahead", gen, 3, vocabulary, dtype))
        compare(view, torch.rand(3, generator=gen, device=DEV), settings("all", 3))
        around.fill_(1e30)
    one = logits_of("ahead", gen, 1, vocabulary, dtype)
    compare(one.expand(9, vocabulary), torch.rand(9, generator=gen, device=DEV), settings("all", 9))


def test_the_largest_vocabulary():
    gen = generator(8)
    for dtype in (torch.float32, torch.bfloat16):
        for kind, name in (("ahead", "all"), ("near", "sum"), ("bulk", "open"), ("near", "count")):
            compare(logits_of(kind, gen, 3, step.MAX_VOCABULARY, dtype), torch.rand(3, generator=gen, device=DEV), settings(name, 3), most_near=0.4)
    with pytest.raises(ValueError, match="contiguous values a row"):
        step.sample_tokens(torch.zeros(1, step.MAX_VOCABULARY + 1, device=DEV), torch.zeros(1, device=DEV))


def test_many_rows():
    gen = generator(21)
    for rows, vocabulary in ((2000, 255), (700, 5000)):
        compare(logits_of("ahead", gen, rows, vocabulary, torch.bfloat16), torch.rand(rows, generator=gen, device=DEV), settings("all", rows))
    assert step.sample_tokens(torch.zeros(0, 7, device=DEV), torch.zeros(0, device=DEV)).shape == (0,)


def test_frequencies_of_tokens():
    """One row expanded, random numbers spread evenly: every token comes as often as its share says, to within one."""
    gen = generator(31)
    row, n = torch.randn(1, 40, generator=gen, device=DEV), 20000
    tokens = step.sample_tokens(row.expand(n, 40), (torch.arange(n, device=DEV) / n).float())
    share = torch.softmax(row[0].double(), 0) * n
    assert ((torch.bincount(tokens.long(), minlength=40) - share).abs() <= 1.01).all()


# ---- streams, graphs, several calls at once ------------------------------------------------------------------

def test_streams_and_graphs():
    gen = generator(41)
    rows, vocabulary = 7, 60000
    logits, uniforms = logits_of("ahead", gen, rows, vocabulary, torch.float32), torch.rand(rows, generator=gen, device=DEV)
    given = settings("all", rows)
    want = step.sample_tokens(logits, uniforms, **given)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    many = [step.sample_tokens(logits, uniforms, **given, stream=other if i % 2 else None) for i in range(6)]
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in many)
    out = torch.zeros(rows, dtype=torch.int32, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step.sample_tokens(logits, uniforms, **given, out=out)
    for _ in range(3):
        logits.copy_(logits_of("ahead", gen, rows, vocabulary, torch.float32))
        uniforms.uniform_(generator=gen)
        given["top_k"].random_(0, 90, generator=gen)
        graph.replay()
        assert torch.equal(out, step.sample_tokens(logits, uniforms, **given))
        compare(logits, uniforms, given)


def test_a_captured_step_goes_on_by_itself():
    """plan, append at its places, attention over the pages, tokens: captured once and replayed, against the same steps by the calls that take
    lengths and tables from the host."""
    gen = generator(51)
    sequences, heads, kv_heads, dim, page, vocabulary, steps = 6, 4, 2, 64, 16, 999, 40
    table = torch.full((sequences, 8), -1, dtype=torch.int32, device=DEV)
    pool, lengths, news = step.PagePool.whole(48, DEV), ints([0] * sequences), ints([1, 1, 1, 1, 0, 1])
    cache, plain_cache = attn.KvCache.empty(48, page, kv_heads, dim), attn.KvCache.empty(48, page, kv_heads, dim)
    embed = randn(gen, vocabulary, (heads + 2 * kv_heads) * dim, std=0.5)
    head = randn(gen, vocabulary, heads * dim, std=0.3)
    frequencies = 1e4 ** (-torch.arange(32, dtype=torch.float64, device=DEV) / 32)
    uniforms = torch.rand(sequences, generator=gen, device=DEV)
    plan = step.StepPlan.in_place(lengths, table, pool, sequences)
    tokens = ints(list(range(sequences)))
    k = torch.full((sequences,), 20, dtype=torch.int32, device=DEV)

    def one():
        step.plan_step(lengths, news, table, pool, page, sequences, out=plan)
        q, key, value = embed[tokens.long()].view(sequences, heads + 2 * kv_heads, dim).split((heads, kv_heads, kv_heads), 1)
        q = step.kv_append_at(q, key, value, cache, plan.slots, plan.positions, frequencies, out=queries)
        y = attn.chunk_attention(q, cache, plan.batch, dim ** -0.5, out=seen)
        step.sample_tokens(torch.mm(y.view(sequences, -1), head.t()), uniforms, top_k=k, softcap=30.0, out=tokens)

    queries, seen = torch.zeros(sequences, heads, dim, dtype=torch.bfloat16, device=DEV), torch.zeros(sequences, heads, dim, dtype=torch.bfloat16, device=DEV)
    state = [t.clone() for t in (lengths, table, pool.taken, tokens)]
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        one()
    torch.cuda.current_stream().wait_stream(warm)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one()
    for t, was in zip((lengths, table, pool.taken, tokens), state):
        t.copy_(was)
    got = []
    for _ in range(steps):
        uniforms.uniform_(generator=gen)
        graph.replay()
        got.append((uniforms.clone(), tokens.clone()))
    pool.check()
    cache.check()
    # the same with the host's numbers: request 4 has no token, five rows are tokens
    past, last = [0] * sequences, ints(list(range(sequences)))
    host_table = torch.arange(sequences * 8, dtype=torch.int32, device=DEV).view(sequences, 8)
    for u, want in got:
        offsets = ints([0, 1, 2, 3, 4, 4, 5])
        past = [n + (s != 4) for s, n in enumerate(past)]
        batch = attn.PagedBatch(offsets, ints(past), host_table)
        q, key, value = embed[last.long()].view(sequences, heads + 2 * kv_heads, dim).split((heads, kv_heads, kv_heads), 1)
        q2 = attn.kv_append(q, key, value, plain_cache, batch, frequencies, out=torch.zeros_like(queries))
        y = attn.chunk_attention(q2, plain_cache, batch, dim ** -0.5, out=torch.zeros_like(seen))
        last = step.sample_tokens(torch.mm(y.view(sequences, -1), head.t()), u, top_k=k, softcap=30.0)
        assert torch.equal(last[:5], want[:5])
        last = want
    assert lengths.tolist() == past and plan.token_offsets.tolist() == [0, 1, 2, 3, 4, 4, 5]


def test_calls_at_once_on_states_of_their_own():
    states = []
    for i in range(4):
        stream = torch.cuda.Stream()
        _, lengths, table, free, taken = requests(i, 50 + i, 16, 40, width=20)
        with torch.cuda.stream(stream):
            state = (stream, ints(lengths), ints(table), step.PagePool(ints(free), ints([taken])), ints([1 + i] * (50 + i)))
        states.append((state, lengths, table, free, taken))
    torch.cuda.synchronize()
    plans = []
    for (stream, lengths, table, pool, news), *_ in states:
        with torch.cuda.stream(stream):
            plans.append([step.plan_step(lengths, news, table, pool, 16, news.numel() * int(news[0])) for _ in range(3)])
    torch.cuda.synchronize()
    for i, ((_, lengths, table, free, taken), plan) in enumerate(zip(states, plans)):
        want = step_ref.plan(lengths, [1 + i] * (50 + i), table, free, taken, 16, (1 + i) * (50 + i))
        for one in plan:
            assert one.slots.tolist() == want[2] and one.lengths.tolist() == want[1]


# ---- in a layer, and from tokens to tokens --------------------------------------------------------------------

def attention_layer(gen, axes=1, hidden=256, heads=4, kv_heads=2, dim=64, window=0):
    frequencies = 1e4 ** (-torch.arange(dim // 2, dtype=torch.float64, device=DEV) / (dim // 2))
    if axes > 1:
        mine = torch.arange(dim // 2, device=DEV)[None] % axes == torch.arange(axes, device=DEV)[:, None]
        frequencies = torch.where(mine, frequencies, 0.0)
    return attn.AttentionLayer(
        pre=randn(gen, hidden), post=randn(gen, hidden), qkv_w=randn(gen, (heads + 2 * kv_heads) * dim, hidden, std=0.1),
        out_w=randn(gen, hidden, heads * dim, std=0.1), q_norm=randn(gen, dim), k_norm=randn(gen, dim), frequencies=frequencies,
        cache=attn.KvCache.empty(64, 16, kv_heads, dim), heads=heads, scale=dim ** -0.5, window=window)


def test_a_layer_over_a_plan_is_the_layer_over_the_batch():
    """Prompts, then steps of several tokens, with rows behind the last request's: bit for bit what the batch gives."""
    gen = generator(61)
    layer = attention_layer(gen)
    pool, table, lengths = step.PagePool.whole(64, DEV), torch.full((5, 12), -1, dtype=torch.int32, device=DEV), ints([0] * 5)
    caches = [layer.cache, attn.KvCache.empty(64, 16, 2, 64)]
    for turn, news in enumerate(([20, 1, 0, 37, 5], [1, 2, 0, 1, 5], [1, 1, 30, 1, 0])):
        tokens = sum(news)
        hidden = randn(gen, tokens + 3, 256)
        plan = step.plan_step(lengths, ints(news), table, pool, 16, tokens + 3)
        layer.cache = caches[0]
        prompt = turn == 0
        got = layer.forward(hidden, plan, prompt)
        layer.cache = caches[1]
        want = layer.forward(hidden[:tokens].contiguous(), plan.batch, prompt)
        assert torch.equal(got[:tokens], want) and torch.isfinite(got[tokens:].float()).all()
        assert torch.equal(caches[0].k, caches[1].k) and torch.equal(caches[0].v, caches[1].v)
        lengths, pool.taken = plan.lengths, plan.taken
    pool.check()
    with pytest.raises(ValueError, match="plan"):
        layer.forward(hidden, plan.batch, positions=plan.positions)


def test_a_layer_with_positions_of_three_axes():
    """Positions that differ along the axes turn differently; the same along all axes they are the plan's own."""
    gen = generator(62)
    layer = attention_layer(gen, axes=3)
    pool, table = step.PagePool.whole(64, DEV), torch.full((2, 12), -1, dtype=torch.int32, device=DEV)
    plan = step.plan_step(ints([0, 0]), ints([30, 12]), table, pool, 16, 42)
    hidden = randn(gen, 42, 256)
    one = layer.forward(hidden, plan, True)
    keys = layer.cache.k.clone()
    two = layer.forward(hidden, plan, True, plan.positions.repeat(3, 1))
    assert torch.equal(one, two) and torch.equal(keys, layer.cache.k)
    layer.forward(hidden, plan, True, torch.stack([plan.positions, plan.positions // 5, plan.positions % 5]))
    assert not torch.equal(keys, layer.cache.k)


def test_a_stack_decodes_from_tokens_to_tokens():
    """The layers, the head and the plans together, against the same calls over a batch and a token chosen by the plain form."""
    from gevva_b200.synthetic import SyntheticAttention, SyntheticStack
    gen = generator(63)
    stack = SyntheticStack(2, 256, DEV, distinct_experts=False, attention=SyntheticAttention(window=24, whole_every=2, pages=32, page_size=16), vocabulary=1201)
    pool, table, state = step.PagePool.whole(32, DEV), torch.full((3, 8), -1, dtype=torch.int32, device=DEV), ints([0, 0, 0])
    news = [9, 1, 30]
    plan = step.plan_step(state, ints(news), table, pool, 16, 40)
    state, pool.taken = plan.lengths, plan.taken
    tokens = torch.randint(0, 1201, (40,), generator=gen, device=DEV, dtype=torch.int32)
    hidden = stack.forward(stack.head.rows[tokens.long()], batch=plan, prompt=True)
    rows = hidden[(plan.token_offsets[1:] - 1).long()].contiguous()
    given = dict(temperature=torch.tensor([1.0, 0.0, 0.8], device=DEV), top_k=ints([0, 0, 40]), top_p=torch.tensor([0.9, 1.0, 1.0], device=DEV))
    u = torch.rand(3, generator=gen, device=DEV)
    last = stack.head.forward(rows, u, **given)
    compare(stack.head.logits(rows), u, given, 30.0)
    places = step.StepPlan.in_place(state, table, pool, 3)
    for _ in range(20):
        u = torch.rand(3, generator=gen, device=DEV)
        step.plan_step(state, ints([1, 1, 1]), table, pool, 16, 3, out=places)
        chosen = stack.decode(last, places, u, **given)
        # again over the batch: the same slots get the same keys and values
        again = stack.forward(stack.head.rows[last.long()], batch=places.batch)
        assert torch.equal(compare(stack.head.logits(again), u, given, 30.0), chosen)
        last = chosen
    pool.check()
    with pytest.raises(ValueError, match="vocabulary"):
        SyntheticStack(1, 16, DEV, distinct_experts=False).decode(last, places, u)


def test_other_devices_and_types_are_refused():
    logits, u = torch.zeros(2, 7, device=DEV), torch.zeros(2, device=DEV)
    for name, value in (("uniforms", u.cpu()), ("uniforms", u.double()), ("uniforms", u[:1])):
        with pytest.raises(ValueError, match=name):
            step.sample_tokens(logits, value)
    for name, value in (("temperature", u.int()), ("top_k", u), ("top_p", u[:1]), ("min_p", u.half()), ("out", u)):
        with pytest.raises(ValueError, match=name):
            step.sample_tokens(logits, u, **{name: value})
    with pytest.raises(ValueError, match="contiguous values"):
        step.sample_tokens(torch.zeros(7, 2, device=DEV).t(), u)
    pool, table, two = step.PagePool.whole(4, DEV), torch.zeros(2, 3, dtype=torch.int32, device=DEV), ints([0, 0])
    with pytest.raises(ValueError, match="news"):
        step.plan_step(two, ints([1]), table, pool, 16, 2)
    with pytest.raises(ValueError, match="table"):
        step.plan_step(two, two, table[:1], pool, 16, 2)
    with pytest.raises(ValueError, match="another table"):
        step.plan_step(two, two, table, pool, 16, 2, out=step.StepPlan.empty(2, table[:, :2], 2))
    with pytest.raises(ValueError, match="out.slots"):
        step.plan_step(two, two, table, pool, 16, 3, out=step.StepPlan.empty(2, table, 2))
    with pytest.raises(step.GevvaMoeError if hasattr(step, "GevvaMoeError") else RuntimeError):
        step.plan_step(two, two, table, pool, 24, 2)
    x = torch.zeros(2, 1, 64, dtype=torch.bfloat16, device=DEV)
    cache = attn.KvCache.empty(2, 16, 1, 64)
    frequencies = torch.zeros(2, 8, dtype=torch.float64, device=DEV)
    for bad in (dict(slots=two.long()), dict(positions=two.float()), dict(positions=ints([[0, 0]] * 17)), dict(positions=ints([0, 0, 0])),
                dict(frequencies=frequencies), dict(frequencies=frequencies[0].float())):
        with pytest.raises(ValueError, match=next(iter(bad))):
            step.kv_append_at(x, x, x, cache, **dict(dict(slots=two, positions=two, frequencies=frequencies[0]), **bad))
