"""The attention operators on a GPU against plain forms in 64 bits."""
import os
import subprocess
import sys

import pytest
import torch

from tests import attention_ref as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def attn():
    from gevva_b200 import attention
    return attention


def randn(shape, device, seed, std=1.0, mean=0.0):
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    return (torch.randn(shape, generator=gen, device=device) * std + mean).to(torch.bfloat16)


def offsets_of(news, device):
    return torch.tensor([0] + torch.tensor(news).cumsum(0).tolist(), dtype=torch.int32, device=device)


def make_batch(attn, news, lengths, page, device, seed, spare=2, width=None):
    """Sequences over pages in random order; table entries that no position needs name no page at all."""
    gen = torch.Generator().manual_seed(seed)
    needed = [-(-n // page) for n in lengths]
    pages = sum(needed) + spare
    order = torch.randperm(pages, generator=gen).to(torch.int32)
    table = torch.full((len(news), max([width or 1] + needed)), -7, dtype=torch.int32)
    at = 0
    for s, n in enumerate(needed):
        table[s, :n] = order[at:at + n]
        at += n
    return attn.PagedBatch(offsets_of(news, device), torch.tensor(lengths, dtype=torch.int32, device=device), table.to(device)), pages


def gathered(cache, batch, s, length):
    rows = batch.table[s, :-(-length // cache.page_size)].long()
    return [c[rows].flatten(0, 1)[:length] for c in (cache.k, cache.v)]


# ---- prompts ----------------------------------------------------------------------------------
@pytest.mark.parametrize("dim", [64, 128, 256, 512])
@pytest.mark.parametrize("news,heads,kv_heads,window", [
    ([1], 1, 1, 0), ([128], 2, 2, 0), ([17, 1, 130], 4, 2, 0), ([129, 0, 300], 8, 1, 0), ([700], 6, 2, 100),
    ([64, 1000, 5], 5, 1, 128), ([1, 1, 1, 1], 7, 1, 3), ([257, 255], 3, 1, 1)])
def test_prompt(attn, cuda_device, dim, news, heads, kv_heads, window):
    tokens = sum(news)
    q, k, v = (randn((tokens, h, dim), cuda_device, i) for i, h in enumerate((heads, kv_heads, kv_heads)))
    scale = dim ** -0.5
    got = attn.prompt_attention(q, k, v, offsets_of(news, cuda_device), scale, window=window)
    at = 0
    for n in news:
        want, bound = ref.attention(q[at:at + n], k[at:at + n], v[at:at + n], 0, scale, window)
        ref.within(got[at:at + n], want, bound, f"rows {at}..{at + n}")
        at += n


def test_prompt_reads_views_and_leaves_padding(attn, cuda_device):
    """Operands as views of one projection's rows; rows outside the offsets stay; other sequences' and padding rows are never seen, whatever they hold."""
    news, heads, kv_heads, dim = [100, 190], 4, 2, 128
    first, tokens = 3, 3 + 290 + 9
    qkv = randn((tokens, heads + 2 * kv_heads, dim), cuda_device, 1)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
    at = torch.tensor([3, 103, 293], dtype=torch.int32, device=cuda_device)
    for bad in (float("nan"), float("inf")):
        qkv[:first] = bad
        qkv[first + 290:] = bad
        out = torch.full((tokens, heads, dim), 5.0, dtype=torch.bfloat16, device=cuda_device)
        assert attn.prompt_attention(q, k, v, at, 0.1, out=out) is out
        assert (out[:first] == 5).all() and (out[first + 290:] == 5).all()
        for a, b in ((3, 103), (103, 293)):
            want, bound = ref.attention(q[a:b], k[a:b], v[a:b], 0, 0.1, 0)
            ref.within(out[a:b], want, bound)
    # a sequence of nothing but infinities leaves its neighbours alone
    qkv[:first] = 0
    qkv[103:293] = float("inf")
    got = attn.prompt_attention(q, k, v, at, 0.1)
    want, bound = ref.attention(q[3:103], k[3:103], v[3:103], 0, 0.1, 0)
    ref.within(got[3:103], want, bound)


@pytest.mark.parametrize("dim", [64, 128, 256, 512])
def test_prompt_of_large_scores_and_growing_maxima(attn, cuda_device, dim):
    """Rows whose maximum grows with every key tile, so that what has been summed is scaled down again and again."""
    n, heads = 600, 2
    q, k, v = (randn((n, heads, dim), cuda_device, 10 + i) for i in range(3))
    k = (k.float() * torch.linspace(0.1, 12.0, n, device=cuda_device)[:, None, None]).to(torch.bfloat16)
    got = attn.prompt_attention(q, k, v, offsets_of([n], cuda_device), dim ** -0.5)
    want, bound = ref.attention(q, k, v, 0, dim ** -0.5, 0)
    ref.within(got, want, bound)


# ---- chunks over the cache ----------------------------------------------------------------------
@pytest.mark.parametrize("dim", [64, 128, 256, 512])
@pytest.mark.parametrize("news,lengths,heads,kv_heads,page,window", [
    ([1], [1], 1, 1, 16, 0), ([1], [700], 4, 2, 16, 0), ([1, 1, 1], [129, 5, 2000], 8, 1, 32, 0), ([5, 0, 5], [300, 40, 5], 6, 2, 64, 0),
    ([200, 1], [1500, 900], 4, 1, 128, 0), ([3, 1], [5000, 64], 5, 1, 256, 1000), ([130], [130], 3, 1, 16, 17),
    ([9, 4], [4, 0], 2, 1, 16, 0), ([1] * 40, [37 * i + 1 for i in range(40)], 2, 2, 32, 50), ([1], [20000], 7, 1, 16, 0)])
def test_chunk(attn, cuda_device, dim, news, lengths, heads, kv_heads, page, window):
    batch, pages = make_batch(attn, news, lengths, page, cuda_device, 3)
    cache = attn.KvCache(randn((pages, page, kv_heads, dim), cuda_device, 1), randn((pages, page, kv_heads, dim), cuda_device, 2))
    # slots that nobody sees hold anything
    for s, n in enumerate(lengths):
        if n % page:
            last = int(batch.table[s, n // page])
            cache.k[last, n % page:] = float("nan")
            cache.v[last, n % page:] = float("inf")
    q = randn((sum(news), heads, dim), cuda_device, 4)
    scale = dim ** -0.5
    got = attn.chunk_attention(q, cache, batch, scale, window=window)
    cache.check()
    at = 0
    for s, (n, length) in enumerate(zip(news, lengths)):
        k, v = gathered(cache, batch, s, length)
        want, bound = ref.attention(q[at:at + n], k, v, length - n, scale, window)
        ref.within(got[at:at + n], want, bound, f"sequence {s}")
        at += n


def test_chunk_of_strided_cache_and_padded_batch(attn, cuda_device):
    """Heads in front of slots, keys and values side by side in one tensor; a batch padded with rows behind the last sequence."""
    page, kv_heads, dim, heads = 32, 2, 128, 4
    batch, pages = make_batch(attn, [1, 2], [100, 333], page, cuda_device, 8, width=40)
    both = randn((pages, kv_heads, page, 2, dim), cuda_device, 1)
    cache = attn.KvCache(both[:, :, :, 0].transpose(1, 2), both[:, :, :, 1].transpose(1, 2))
    q = randn((6, heads, 2 * dim), cuda_device, 2)[:, :, dim:]
    out = torch.full((6, heads, dim), -3.0, dtype=torch.bfloat16, device=cuda_device)
    attn.chunk_attention(q, cache, batch, 0.09, out=out)
    assert (out[3:] == -3).all()
    for s, (a, b, length) in enumerate(((0, 1, 100), (1, 3, 333))):
        k, v = gathered(cache, batch, s, length)
        want, bound = ref.attention(q[a:b], k, v, length - (b - a), 0.09, 0)
        ref.within(out[a:b], want, bound)


def test_chunk_ignores_pages_in_front_of_the_window(attn, cuda_device):
    """A window's old pages may have been given to others already: what stands there is not seen."""
    page, dim, length, window = 16, 256, 1000, 200
    batch, pages = make_batch(attn, [3], [length], page, cuda_device, 2)
    cache = attn.KvCache(randn((pages, page, 1, dim), cuda_device, 1), randn((pages, page, 1, dim), cuda_device, 2))
    q = randn((3, 2, dim), cuda_device, 3)
    k, v = gathered(cache, batch, 0, length)
    want, bound = ref.attention(q, k, v, length - 3, 0.05, window)
    first = length - 3 - window + 1
    rows = batch.table[0, :first // page].long()
    cache.k[rows] = float("nan")
    cache.v[rows] = float("nan")
    part = int(batch.table[0, first // page])
    cache.v[part, :first % page] = float("inf")
    batch.table[0, :first // page] = 1 << 30  # no page at all
    ref.within(attn.chunk_attention(q, cache, batch, 0.05, window=window), want, bound)


def test_chunk_reports_lengths_beyond_the_table(attn, cuda_device):
    from gevva_b200 import GevvaMoeError
    cache = attn.KvCache(randn((4, 16, 1, 64), cuda_device, 1), randn((4, 16, 1, 64), cuda_device, 2))
    batch = attn.PagedBatch(offsets_of([1, 1], cuda_device), torch.tensor([20, 33], dtype=torch.int32, device=cuda_device),
                            torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=cuda_device))
    q = randn((2, 1, 64), cuda_device, 3)
    got = attn.chunk_attention(q, cache, batch, 0.125)
    with pytest.raises(GevvaMoeError, match="page"):
        cache.check()
    k, v = gathered(cache, batch, 0, 20)
    want, bound = ref.attention(q[:1], k, v, 19, 0.125, 0)
    ref.within(got[:1], want, bound)
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads", [1, 3, 8, 16])
def test_query_tiles_with_few_rows_behind_many_keys(attn, cuda_device, dim, heads):
    """The last query tile has rows for some of the warps only, and keys enough that the others could be far ahead of them."""
    step = 128 // heads * 2
    for n in [7 * 128 // step * step + rest for rest in (1, 31 // heads + 1, 64 // heads + 1, step // 2, step // 2 + 1, step - 1)]:
        q, k, v = (randn((n, h, dim), cuda_device, n + i) for i, h in enumerate((heads, 1, 1)))
        want, bound = ref.attention(q, k, v, 0, dim ** -0.5, 0)
        for _ in range(3):
            ref.within(attn.prompt_attention(q, k, v, offsets_of([n], cuda_device), dim ** -0.5), want, bound, f"{n} tokens")
        batch, pages = make_batch(attn, [n], [n], 64, cuda_device, 2)
        cache = attn.KvCache.empty(pages, 64, 1, dim, cuda_device)
        at = batch.table[0, :-(-n // 64)].long()
        for x, to in ((k, cache.k), (v, cache.v)):
            whole = torch.zeros((len(at) * 64, 1, dim), dtype=torch.bfloat16, device=cuda_device)
            whole[:n] = x
            to[at] = whole.view(len(at), 64, 1, dim)
        ref.within(attn.chunk_attention(q, cache, batch, dim ** -0.5), want, bound, f"{n} tokens over pages")


@pytest.mark.parametrize("dim,news,past,window", [(64, 4096, 0, 100), (256, 4096, 37, 300), (256, 1000, 9000, 0), (512, 700, 5000, 0)])
def test_chunk_of_many_query_tiles(attn, cuda_device, dim, news, past, window):
    """Runs of key tiles inside one sequence, longer and shorter than a query tile's, that begin and end inside them."""
    page, heads = 64, 16
    batch, pages = make_batch(attn, [news], [news + past], page, cuda_device, 2)
    cache = attn.KvCache(randn((pages, page, 1, dim), cuda_device, 1), randn((pages, page, 1, dim), cuda_device, 2))
    q = randn((news, heads, dim), cuda_device, 3)
    k, v = gathered(cache, batch, 0, news + past)
    got = attn.chunk_attention(q, cache, batch, dim ** -0.5, window)
    cache.check()
    ref.within(got, *ref.attention(q, k, v, past, dim ** -0.5, window))


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 64), (256, 256), (512, 32)])
def test_chunk_reports_pages_outside_the_cache(attn, cuda_device, dim, page):
    """One that a row sees reads as zeros and is reported; those in front of a window and behind the last key are nobody's."""
    from gevva_b200 import GevvaMoeError
    batch, pages = make_batch(attn, [2, 3], [500, 1000], page, cuda_device, 2)
    cache = attn.KvCache(randn((pages, page, 1, dim), cuda_device, 1), randn((pages, page, 1, dim), cuda_device, 2))
    q = randn((5, 2, dim), cuda_device, 3)
    batch.table[1, :(1000 - 3 - 200 + 1) // page] = pages
    batch.table[:, -(-1000 // page):] = -1
    attn.chunk_attention(q, cache, batch, 0.05, window=200)
    cache.check()
    for wrong in (-1, pages, -2 ** 31, 2 ** 31 - 1):
        batch.table[1, 900 // page] = wrong
        got = attn.chunk_attention(q, cache, batch, 0.05, window=200)
        with pytest.raises(GevvaMoeError, match="page"):
            cache.check()
        cache.check()  # (reported once)
        (k, v), seen = gathered(cache, batch, 0, 500), slice(0, 2)
        ref.within(got[seen], *ref.attention(q[seen], k, v, 498, 0.05, 200))
        assert torch.isfinite(got).all()


@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 4, 4), (256, 16, 8), (512, 16, 2)])
def test_chunk_repeats_its_bits_and_equals_the_prompt_form(attn, cuda_device, dim, heads, kv_heads):
    n, page = 900, 64
    batch, pages = make_batch(attn, [n], [n], page, cuda_device, 5)
    k, v = (randn((n, kv_heads, dim), cuda_device, i) for i in (1, 2))
    cache = attn.KvCache.empty(pages, page, kv_heads, dim, cuda_device)
    rows = batch.table[0].long()
    for store, x in ((cache.k, k), (cache.v, v)):
        padded = torch.zeros(len(rows) * page, kv_heads, dim, dtype=torch.bfloat16, device=cuda_device)
        padded[:n] = x
        store[rows] = padded.view(len(rows), page, kv_heads, dim)
    q = randn((n, heads, dim), cuda_device, 3)
    first = attn.chunk_attention(q, cache, batch, 0.06)
    for _ in range(5):
        assert torch.equal(first, attn.chunk_attention(q, cache, batch, 0.06))
    prompt = attn.prompt_attention(q, k, v, batch.token_offsets, 0.06)
    assert torch.equal(prompt, attn.prompt_attention(q, k, v, batch.token_offsets, 0.06))
    want, bound = ref.attention(q, k, v, 0, 0.06, 0)
    ref.within(first, want, bound)
    ref.within(prompt, want, bound)


def test_chunk_with_offsets_past_32_bits(attn, cuda_device):
    """A cache of more than 2^32 bytes a tensor: the last page lies behind 32-bit offsets."""
    page, kv_heads, dim = 128, 8, 256
    pages = (1 << 32) // (page * kv_heads * dim * 2) + 9
    cache = attn.KvCache(*(torch.empty((pages, page, kv_heads, dim), dtype=torch.bfloat16, device=cuda_device) for _ in range(2)))
    batch = attn.PagedBatch(offsets_of([2], cuda_device), torch.tensor([250], dtype=torch.int32, device=cuda_device),
                            torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device=cuda_device))
    for i, store in enumerate((cache.k, cache.v)):
        store[pages - 2:] = randn((2, page, kv_heads, dim), cuda_device, i)
    q = randn((2, 16, dim), cuda_device, 7)
    k, v = gathered(cache, batch, 0, 250)
    want, bound = ref.attention(q, k, v, 248, 0.0625, 0)
    ref.within(attn.chunk_attention(q, cache, batch, 0.0625), want, bound)
    # and the append stores there
    new = randn((2, 2 * kv_heads + 16, dim), cuda_device, 9)
    attn.kv_append(new[:, :16], new[:, 16:24], new[:, 24:], cache, batch, None)
    cache.check()
    for c, x in ((cache.k, new[:, 16:24]), (cache.v, new[:, 24:])):
        assert torch.equal(c[pages - 2, 248 - page:250 - page], x)


# ---- append -------------------------------------------------------------------------------------
@pytest.mark.parametrize("dim", [64, 128, 256, 512])
@pytest.mark.parametrize("news,lengths,heads,kv_heads,page,rotated,normed,packed", [
    ([1], [1], 1, 1, 16, 1.0, True, False), ([1, 1, 1], [5, 100000, 17], 16, 8, 16, 1.0, True, False),
    ([7, 0, 20], [7, 30, 4000], 6, 3, 64, 0.5, True, True), ([33], [33], 5, 1, 32, 0.25, False, True), ([3, 4], [900, 4], 2, 2, 128, 0, True, False)])
def test_append(attn, cuda_device, dim, news, lengths, heads, kv_heads, page, rotated, normed, packed):
    batch, pages = make_batch(attn, news, lengths, page, cuda_device, 3)
    cache = attn.KvCache(randn((pages, page, kv_heads, dim), cuda_device, 1), randn((pages, page, kv_heads, dim), cuda_device, 2))
    before = cache.k.clone(), cache.v.clone()
    tokens = sum(news)
    qkv = randn((tokens, heads + 2 * kv_heads, dim), cuda_device, 4, std=3.0)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
    qw, kw = (randn((dim,), cuda_device, 5 + i, 0.2, 1.0) if normed else None for i in range(2))
    half = int(dim * rotated) // 2
    freq = (1e4 ** (-torch.arange(half, dtype=torch.float64, device=cuda_device) / max(half, 1))) if half else None
    eps = 1e-6
    got = attn.kv_append(q, k, v, cache, batch, freq, q_weight=qw, k_weight=kw, normalize_v=normed, eps=eps, packed=packed)
    cache.check()
    position = torch.cat([torch.arange(length - n, length, device=cuda_device) for n, length in zip(news, lengths)])
    sequence = torch.repeat_interleave(torch.arange(len(news), device=cuda_device), torch.tensor(news, device=cuda_device))
    at = (batch.table[sequence, position // page].long(), position % page)

    def check(x, weight, turn, result, what):
        y = ref.norm(x, weight, eps) if (weight is not None or (not turn and normed)) else x.double()
        want, size = ref.rotate(y, position, freq) if turn else (y, y.abs())
        # norm: a sum of dim squares, a square root and three products; angle: 2^-20 of a radian at most
        ref.within(result, want, ref.BF16 * want.abs() + size * ((dim / 2 + 16) * ref.FP32 + 2.0 ** -20) + 1e-30, what)

    check(q, qw, True, got.q if packed else got, "q")
    check(k, kw, True, cache.k[at], "k")
    check(v, None, False, cache.v[at], "v")
    if packed:
        assert torch.equal(got.k, cache.k[at]) and torch.equal(got.v, cache.v[at])
    for now, old in zip((cache.k, cache.v), before):
        old[at] = now[at]
        assert torch.equal(now, old)  # nothing else has been written


@pytest.mark.parametrize("dim", [64, 128, 256, 512])
@pytest.mark.parametrize("heads,kv_heads", [(3, 1), (16, 8)])
def test_append_of_many_tokens(attn, cuda_device, dim, heads, kv_heads):
    """More tokens than are in work at a time, with rows in front of the first and behind the last sequence and a sequence without pages:
    the same bits as a few tokens at a time."""
    news, page, tokens = [700, 0, 1, 900, 600], 32, 2300
    batch, pages = make_batch(attn, news, [n + 40 for n in news], page, cuda_device, 2)
    batch.token_offsets += 30
    batch.table[2] = -1
    q, k, v = (randn((tokens, h, dim), cuda_device, 3 + i) for i, h in enumerate((heads, kv_heads, kv_heads)))
    weight = randn((dim,), cuda_device, 6)
    freq = torch.rand(dim // 4, dtype=torch.float64, device=cuda_device)

    norms = (weight, weight, True, 1e-6)
    cache, want_cache = (attn.KvCache.empty(pages, page, kv_heads, dim, cuda_device) for _ in range(2))
    got = attn.kv_append(q, k, v, cache, batch, freq, *norms, packed=True)
    offsets = batch.token_offsets.tolist()
    for s, (begin, end) in enumerate(zip(offsets, offsets[1:])):
        for at in range(begin, end, 300):
            to = min(at + 300, end)
            part = attn.PagedBatch(offsets_of([to - at], cuda_device), batch.lengths[s:s + 1] - (end - to), batch.table[s:s + 1])
            for x, y in zip(got, attn.kv_append(q[at:to], k[at:to], v[at:to], want_cache, part, freq, *norms, packed=True)):
                assert torch.equal(x[at:to], y), (s, at)
    assert cache.last_status() == want_cache.last_status() == -7
    assert torch.equal(cache.k, want_cache.k) and torch.equal(cache.v, want_cache.v) and cache.k.any()


def test_append_without_pages_and_behind_the_last_sequence(attn, cuda_device):
    page, dim = 16, 64
    cache = attn.KvCache.empty(3, page, 1, dim, cuda_device)
    x = randn((8, 3, dim), cuda_device, 1)
    # sequence 0: position 16 is in a page that does not exist; sequence 1: position 40 is outside the table; rows 5.. are padding
    batch = attn.PagedBatch(torch.tensor([0, 3, 5], dtype=torch.int32, device=cuda_device), torch.tensor([17, 41], dtype=torch.int32, device=cuda_device),
                            torch.tensor([[1, 3], [2, -1]], dtype=torch.int32, device=cuda_device))
    out = torch.full((8, 1, dim), 9.0, dtype=torch.bfloat16, device=cuda_device)
    attn.kv_append(x[:, :1], x[:, 1:2], x[:, 2:], cache, batch, None, out=out)
    from gevva_b200 import GevvaMoeError
    with pytest.raises(GevvaMoeError, match="page"):
        cache.check()
    cache.check()  # cleared
    assert torch.equal(out[:5], x[:5, :1]) and (out[5:] == 9).all()
    want = torch.zeros_like(cache.k)
    want[1, 14:16] = x[:2, 1:2]
    assert torch.equal(cache.k, want)


def test_append_turns_far_positions_as_exactly_as_near_ones(attn, cuda_device):
    page, dim, far = 256, 128, 262143
    width = (far + page) // page
    cache = attn.KvCache.empty(1, page, 1, dim, cuda_device)
    table = torch.zeros((1, width), dtype=torch.int32, device=cuda_device)
    batch = attn.PagedBatch(offsets_of([1], cuda_device), torch.tensor([far + 1], dtype=torch.int32, device=cuda_device), table)
    x = randn((1, 3, dim), cuda_device, 1)
    freq = 1e6 ** (-torch.arange(dim // 2, dtype=torch.float64, device=cuda_device) / (dim // 2))
    got = attn.kv_append(x[:, :1], x[:, 1:2], x[:, 2:], cache, batch, freq)
    want, size = ref.rotate(x[:, :1].double(), torch.tensor([far], device=cuda_device), freq)
    ref.within(got, want, ref.BF16 * want.abs() + size * 2.0 ** -20)


# ---- norms --------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows", [1, 3, 64, 777])
@pytest.mark.parametrize("width", [8, 64, 264, 512, 520, 2816, 4104, 8200, 32768])
def test_norms(attn, cuda_device, rows, width):
    x, residual = randn((rows, width), cuda_device, 1, 3.0), randn((rows, width), cuda_device, 2, 2.0)
    weight, gate, following = (randn((width,), cuda_device, 3 + i, 0.3, 1.0) for i in range(3))
    scale = randn((1,), cuda_device, 6, 0.1, 0.8)
    if rows > 2:
        x[1] = 0
        residual[2] = 0
    eps = 1e-5
    small = (width / 2 + 16) * ref.FP32  # a sum of `width` squares under a square root, and a few products
    y = ref.norm(x, weight, eps)
    ref.within(attn.block_norm(x, weight, eps=eps), y, y.abs() * (ref.BF16 + small) + 1e-30, "norm")
    for g, s, f in ((None, None, None), (gate, None, None), (gate, scale, following), (None, scale, following)):
        part = y if g is None else y * g.double()
        want = residual.double() + part
        size = residual.double().abs() + part.abs()
        if s is not None:
            want, size = want * s.double(), size * s.double().abs()
        got = attn.block_norm_add(x, weight, residual, gate=g, scale=s, next_weight=f, eps=eps)
        if f is not None:
            got, after = got
            # each value is off by small * size before the second norm, its statistic by no more than the largest of them relative to the row's size
            second = ref.norm(want, f, eps)
            rms = torch.sqrt((want * want).mean(-1, keepdim=True) + eps)
            off = 2 * small * size
            bound = ref.BF16 * second.abs() + (off / rms + (want.abs() / rms) * (off.amax(-1, keepdim=True) / rms + small)) * f.double().abs()
            ref.within(after, second, bound + 1e-30, "next")
        ref.within(got, want, want.abs() * ref.BF16 + 2 * small * size + 1e-30, "add")


def test_norm_add_in_place(attn, cuda_device):
    x, residual, weight = randn((50, 2816), cuda_device, 1), randn((50, 2816), cuda_device, 2), randn((2816,), cuda_device, 3)
    want = attn.block_norm_add(x, weight, residual)
    hidden = residual.clone()
    assert attn.block_norm_add(x, weight, hidden, out=hidden) is hidden and torch.equal(hidden, want)


# ---- together, streams and graphs ---------------------------------------------------------------
def test_append_then_attention_as_one_graph_of_growing_lengths(attn, cuda_device):
    """A decode step captured once and replayed while lengths, positions and pages move on; checked against the prompt form of the same tokens."""
    heads, kv_heads, dim, page, steps, sequences = 4, 2, 256, 16, 40, 3
    starts = [0, 5, 130]
    width = 16
    gen = torch.Generator().manual_seed(2)
    table = torch.randperm(sequences * width, generator=gen).to(torch.int32).view(sequences, width).to(cuda_device)
    cache = attn.KvCache.empty(sequences * width, page, kv_heads, dim, cuda_device)
    freq = 1e4 ** (-torch.arange(dim // 2, dtype=torch.float64, device=cuda_device) / (dim // 2))
    total = [s + steps for s in starts]
    qkv = [randn((n, heads + 2 * kv_heads, dim), cuda_device, 20 + i) for i, n in enumerate(total)]

    def split(x):
        return x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:]

    # the prompts' share, all at once
    if sum(starts):
        batch = attn.PagedBatch(offsets_of(starts, cuda_device), torch.tensor(starts, dtype=torch.int32, device=cuda_device), table)
        attn.kv_append(*split(torch.cat([x[:n] for x, n in zip(qkv, starts)])), cache, batch, freq)
    static = torch.empty((sequences, heads + 2 * kv_heads, dim), dtype=torch.bfloat16, device=cuda_device)
    lengths = torch.tensor(starts, dtype=torch.int32, device=cuda_device)
    batch = attn.PagedBatch(offsets_of([1] * sequences, cuda_device), lengths, table)
    lengths += 1
    static.copy_(torch.stack([x[n] for x, n in zip(qkv, starts)]))

    def step():
        return attn.chunk_attention(attn.kv_append(*split(static), cache, batch, freq), cache, batch, 0.0625)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    got = [[] for _ in range(sequences)]
    for i in range(steps):
        static.copy_(torch.stack([x[n + i] for x, n in zip(qkv, starts)]))
        lengths.copy_(torch.tensor([n + i + 1 for n in starts], dtype=torch.int32))
        graph.replay()
        for s in range(sequences):
            got[s].append(out[s].clone())
    cache.check()
    for s, n in enumerate(total):
        own = attn.KvCache.empty(width, page, kv_heads, dim, cuda_device)
        whole = attn.PagedBatch(offsets_of([n], cuda_device), torch.tensor([n], dtype=torch.int32, device=cuda_device),
                                torch.arange(width, dtype=torch.int32, device=cuda_device)[None])
        q, k, v = attn.kv_append(*split(qkv[s]), own, whole, freq, packed=True)
        want, bound = ref.attention(q, k, v, 0, 0.0625, 0)
        ref.within(torch.stack(got[s]), want[starts[s]:], bound[starts[s]:], f"sequence {s}")


def test_two_streams_at_once(attn, cuda_device):
    """Chunk calls on streams of their own overlap, each with a workspace of its own."""
    cases = []
    for i in range(2):
        batch, pages = make_batch(attn, [1] * 20, [400 + 111 * j for j in range(20)], 32, cuda_device, i)
        cache = attn.KvCache(randn((pages, 32, 2, 128), cuda_device, i), randn((pages, 32, 2, 128), cuda_device, 10 + i))
        cases.append((randn((20, 8, 128), cuda_device, 20 + i), cache, batch, 0.09))
    want = [attn.chunk_attention(*c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (c, s) in enumerate(zip(cases, streams)):
            out = torch.empty_like(want[i])
            got[i].append(attn.chunk_attention(*c, out=out, stream=s))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert torch.equal(g, want[i])


def test_what_a_call_makes_belongs_to_its_stream(attn, cuda_device):
    """On a stream other than the current one: what the call gives back to the allocator may still be in use there, and here it is not handed out."""
    x = randn((200, 2, 64), cuda_device, 1)
    offsets = offsets_of([200], cuda_device)
    batch, pages = make_batch(attn, [200], [200], 16, cuda_device, 2)
    cache = attn.KvCache(randn((pages, 16, 2, 64), cuda_device, 1), randn((pages, 16, 2, 64), cuda_device, 2))
    rows = x.view(200, 128)
    weight = torch.ones(128, dtype=torch.bfloat16, device=cuda_device)
    calls = [lambda s: attn.block_norm(rows, weight, stream=s), lambda s: attn.block_norm_add(rows, weight, rows, stream=s),
             lambda s: attn.kv_append(x, x, x, cache, batch, None, stream=s), lambda s: attn.prompt_attention(x, x, x, offsets, 0.125, stream=s),
             lambda s: attn.chunk_attention(x, cache, batch, 0.125, stream=s)]
    for i, call in enumerate(calls):
        side = torch.cuda.Stream(cuda_device)
        torch.cuda.synchronize()
        want = call(None)
        for stream in (side, side.cuda_stream, 0):
            torch.cuda.synchronize()
            got = call(stream)
            torch.cuda.synchronize()
            assert torch.equal(got, want), i
            if stream:
                at = got.data_ptr()
                del got
                held = [torch.empty_like(x) for _ in range(8)]
                assert all(h.data_ptr() != at for h in held), i
    cache.check()


def test_a_process_may_begin_with_a_captured_call(attn, cuda_device):
    """Nothing has to be called once before it is captured."""
    code = """
import torch
import gevva_b200 as g
d = torch.device("cuda:0")
bf16, i32 = torch.bfloat16, torch.int32
qkv = torch.randn(40, 6, 256, device=d).to(bf16)
weight, freq = torch.ones(256, dtype=bf16, device=d), torch.ones(128, dtype=torch.float64, device=d)
cache = g.KvCache.empty(4, 32, 1, 256, d)
batch = g.PagedBatch(torch.tensor([0, 40], dtype=i32, device=d), torch.tensor([40], dtype=i32, device=d), torch.arange(4, dtype=i32, device=d)[None])
rows = qkv.view(40, 1536)
row_weight = torch.ones(1536, dtype=bf16, device=d)

def calls():
    q, k, v = g.kv_append(*qkv.split((4, 1, 1), 1), cache, batch, freq, weight, weight, packed=True)
    a, b = g.prompt_attention(q, k, v, batch.token_offsets, 0.06), g.chunk_attention(q, cache, batch, 0.06)
    return a, b, g.block_norm(rows, row_weight), g.block_norm_add(rows, row_weight, rows)

graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    captured = calls()
graph.replay()
torch.cuda.synchronize()
for x, y in zip(captured, calls()):
    assert torch.equal(x, y) and x.any()
cache.check()
"""
    subprocess.run([sys.executable, "-c", code], check=True, timeout=300, cwd=ROOT)


def test_nothing_to_do(attn, cuda_device):
    x = torch.empty((0, 2, 64), dtype=torch.bfloat16, device=cuda_device)
    zero = torch.zeros(2, dtype=torch.int32, device=cuda_device)
    assert attn.prompt_attention(x, x, x, zero, 1.0).shape == (0, 2, 64)
    cache = attn.KvCache.empty(1, 16, 2, 64, cuda_device)
    batch = attn.PagedBatch(zero, zero[:1], torch.zeros((1, 1), dtype=torch.int32, device=cuda_device))
    assert attn.chunk_attention(x, cache, batch, 1.0).shape == (0, 2, 64)
    assert attn.kv_append(x, x, x, cache, batch, None).shape == (0, 2, 64)
    assert attn.block_norm(torch.empty((0, 64), dtype=torch.bfloat16, device=cuda_device), torch.ones(64, dtype=torch.bfloat16, device=cuda_device)).shape == (0, 64)


def test_layers_of_a_stack(attn, cuda_device):
    """A stack with attention: prompts, then a chunk and single tokens over the same cache.  Each layer's call is the sequence of its parts, and
    both forms of attention see the same context."""
    from gevva_b200.synthetic import SyntheticAttention, SyntheticStack
    shape = SyntheticAttention(heads=4, kv_heads=2, head_dim=256, window=100, whole_every=2, pages=40, page_size=16)
    stack = SyntheticStack(2, 512, cuda_device, distinct_experts=False, attention=shape)
    assert [a.window for a in stack.attention] == [100, 0]
    news = [130, 7]
    table = torch.randperm(40, generator=torch.Generator().manual_seed(1)).to(torch.int32).view(2, 20).to(cuda_device)

    def batch_of(news, lengths):
        return attn.PagedBatch(offsets_of(news, cuda_device), torch.tensor(lengths, dtype=torch.int32, device=cuda_device), table)

    hidden = randn((sum(news), 2816), cuda_device, 5)
    with pytest.raises(ValueError, match="batch"):
        stack.forward(hidden)
    out = stack.forward(hidden, batch=batch_of(news, news), prompt=True)
    assert torch.isfinite(out).all()
    # the parts of the first layer, one by one; its cache holds these tokens
    layer, batch = stack.attention[0], batch_of(news, news)
    x = attn.block_norm(hidden, layer.pre)
    qkv = torch.mm(x, layer.qkv_w.t()).view(-1, 8, 256)
    q, k, v = attn.kv_append(qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], layer.cache, batch, layer.frequencies, layer.q_norm, layer.k_norm, True, packed=True)
    seen = attn.prompt_attention(q, k, v, batch.token_offsets, layer.scale, 100)
    paged = attn.chunk_attention(q, layer.cache, batch, layer.scale, 100)
    at = 0
    for n in news:
        want, bound = ref.attention(q[at:at + n], k[at:at + n], v[at:at + n], 0, layer.scale, 100)
        ref.within(seen[at:at + n], want, bound)
        ref.within(paged[at:at + n], want, bound)
        at += n
    y = attn.block_norm_add(torch.mm(seen.view(-1, 1024), layer.out_w.t()), layer.post, hidden)
    assert torch.equal(y, layer.forward(hidden, batch, prompt=True))
    # a chunk, then tokens one by one
    for news, lengths in (([5, 3], [135, 10]), ([1, 1], [136, 11]), ([1, 1], [137, 12])):
        out = stack.forward(randn((sum(news), 2816), cuda_device, lengths[0]), batch=batch_of(news, lengths))
        assert torch.isfinite(out).all()
    for a, f in zip(stack.attention, stack.layers):
        a.cache.check()
        f.experts.check()
