"""The attention operators at the edges of what they take."""
import pytest
import torch

from tests import attention_ref as ref
from tests.test_gpu_attention import attn, gathered, make_batch, offsets_of, randn  # noqa: F401  (attn: a fixture)

pytestmark = pytest.mark.gpu


# ---- scores that are no numbers -------------------------------------------------------------------
@pytest.mark.parametrize("dim", [64, 128, 256, 512])
def test_scores_that_are_no_numbers_give_none(attn, cuda_device, dim):
    """A query that is NaN, and products that leave the range of 32 bits, give NaN and nothing else, whichever key they meet; the other rows are
    as they were.  (A window of one: a row sees the key in its own place only.)"""
    n, heads = 300, 2
    q, k, v = (randn((n, heads, dim), cuda_device, i) for i in range(3))
    broken = torch.zeros(n, dtype=torch.bool, device=cuda_device)
    for first, value in ((0, float("nan")), (1, 1e30)):
        rows = torch.arange(first, n, 3, device=cuda_device)
        broken[rows] = True
        q[rows] = value
        if value == value:
            k[rows] = value
    batch, pages = make_batch(attn, [n], [n], 64, cuda_device, 2)
    cache = attn.KvCache.empty(pages, 64, heads, dim, cuda_device)
    attn.kv_append(q, k, v, cache, batch, None)
    for got in (attn.prompt_attention(q, k, v, batch.token_offsets, 0.125, window=1), attn.chunk_attention(q, cache, batch, 0.125, window=1)):
        assert torch.isnan(got[broken]).all()
        assert torch.equal(got[~broken], v[~broken])


# ---- every key counts -----------------------------------------------------------------------------
def counted(tokens, length, heads, kv_heads, dim, device, seed):
    """Operands for which p is zero or one: every key has a class of its key head and a score of 128 for the queries of that class, zero for
    the others, so that a row's result is the mean of v over the keys of its class (exp(-128) is nothing), or over all that it sees where
    none is of its class.  v is whole numbers, so sums are exact; a key lost, seen twice or taken from elsewhere changes the mean by more than its
    rounding."""
    gen = torch.Generator(device=device)
    gen.manual_seed(seed)
    group = heads // kv_heads
    kind = torch.randint(0, group, (length, kv_heads), generator=gen, device=device)
    k = 128.0 * torch.nn.functional.one_hot(kind, dim)
    q = torch.nn.functional.one_hot(torch.arange(heads, device=device) % group, dim).float().expand(tokens, heads, dim)
    v = torch.randint(-2, 3, (length, kv_heads, dim), generator=gen, device=device)
    return [x.to(torch.bfloat16).contiguous() for x in (q, k, v)]


def whole_mean(got, q, k, v, past, window, what=""):
    """The mean is rounded once; the sum that divides it and its inverse are off by a few 2^-24, an exponential of zero by 2^-18 at most."""
    want, _ = ref.attention(q, k, v, past, 1.0, window)
    ref.within(got, want, want.abs() * (ref.BF16 + 2.0 ** -17) + 1e-30, what)
    # the test itself: one key less would have been noticed
    h, group, row = q.shape[1] - 1, q.shape[1] // k.shape[1], q.shape[0] - 1
    if past + row > 0 and window != 1:
        low = max(0, past + row - window + 1) if window else 0
        score = q[row, h].double() @ k[low:past + row + 1, h // group].double().T
        mine = (score == score.amax()).nonzero()[:, 0] + low
        lost = mine[len(mine) // 2]
        less = (v[mine, h // group].double().sum(0) - v[lost, h // group].double()) / max(len(mine) - 1, 1)
        assert ((less - want[row, h]).abs() > want[row, h].abs() * (ref.BF16 + 2.0 ** -17)).any(), (what, "a lost key would not be noticed")


@pytest.mark.parametrize("dim", [64, 128, 256, 512])
@pytest.mark.parametrize("news,lengths,heads,kv_heads,page,window", [
    ([1], [20000], 7, 1, 16, 0), ([1], [20000], 8, 8, 16, 0), ([1, 1, 1], [5000, 3, 12345], 12, 3, 32, 0), ([1, 1], [30000, 9000], 4, 2, 64, 7000),
    ([5, 3], [6001, 129], 6, 1, 16, 1024), ([300], [2300], 8, 2, 128, 0), ([200, 7], [900, 4000], 3, 1, 1024, 333)])
def test_chunk_counts_every_key(attn, cuda_device, dim, news, lengths, heads, kv_heads, page, window):
    batch, pages = make_batch(attn, news, lengths, page, cuda_device, 3)
    cache = attn.KvCache(*(torch.full((pages, page, kv_heads, dim), 96.0, dtype=torch.bfloat16, device=cuda_device) for _ in range(2)))
    parts = [counted(n, length, heads, kv_heads, dim, cuda_device, s) for s, (n, length) in enumerate(zip(news, lengths))]
    for s, ((_, k, v), length) in enumerate(zip(parts, lengths)):
        at = torch.arange(length, device=cuda_device)
        rows = batch.table[s].long()[at // page]
        cache.k[rows, at % page] = k
        cache.v[rows, at % page] = v
    got = attn.chunk_attention(torch.cat([q for q, _, _ in parts]), cache, batch, 1.0, window)
    cache.check()
    at = 0
    for s, ((q, k, v), n, length) in enumerate(zip(parts, news, lengths)):
        whole_mean(got[at:at + n], q, k, v, length - n, window, f"sequence {s}")
        at += n


@pytest.mark.parametrize("dim", [64, 128, 256, 512])
@pytest.mark.parametrize("news,heads,kv_heads,window", [([1500], 4, 2, 0), ([700, 0, 33, 260], 7, 1, 129), ([400, 650], 2, 2, 0)])
def test_prompt_counts_every_key(attn, cuda_device, dim, news, heads, kv_heads, window):
    parts = [counted(n, n, heads, kv_heads, dim, cuda_device, s) for s, n in enumerate(news)]
    q, k, v = (torch.cat(x) for x in zip(*parts))
    got = attn.prompt_attention(q, k, v, offsets_of(news, cuda_device), 1.0, window=window)
    at = 0
    for s, (n, part) in enumerate(zip(news, parts)):
        if n:
            whole_mean(got[at:at + n], *part, 0, window, f"sequence {s}")
        at += n


# ---- many heads to a key head, many sequences, long contexts ----------------------------------------
@pytest.mark.parametrize("dim", [64, 128, 256, 512])
@pytest.mark.parametrize("heads,kv_heads", [(17, 1), (34, 2), (32, 1), (65, 1), (100, 1), (128, 1), (256, 2)])
def test_many_query_heads_to_a_key_head(attn, cuda_device, dim, heads, kv_heads):
    news, lengths, page, window = [40, 1, 3], [40, 300, 200], 16, 37
    q = randn((sum(news), heads, dim), cuda_device, 1)
    k, v = (randn((sum(news), kv_heads, dim), cuda_device, 2 + i) for i in range(2))
    got = attn.prompt_attention(q, k, v, offsets_of(news, cuda_device), dim ** -0.5, window=window)
    batch, pages = make_batch(attn, news, lengths, page, cuda_device, 3)
    cache = attn.KvCache(randn((pages, page, kv_heads, dim), cuda_device, 5), randn((pages, page, kv_heads, dim), cuda_device, 6))
    paged = attn.chunk_attention(q, cache, batch, dim ** -0.5)
    cache.check()
    at = 0
    for s, (n, length) in enumerate(zip(news, lengths)):
        rows = slice(at, at + n)
        ref.within(got[rows], *ref.attention(q[rows], k[rows], v[rows], 0, dim ** -0.5, window), f"prompt {s}")
        ref.within(paged[rows], *ref.attention(q[rows], *gathered(cache, batch, s, length), length - n, dim ** -0.5, 0), f"sequence {s}")
        at += n


@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 4, 2), (256, 2, 1)])
def test_many_sequences(attn, cuda_device, dim, heads, kv_heads):
    """More than a warp looks at together, some of them empty, as prompts, appended and over pages."""
    news = [(0, 1, 3, 8, 0, 17, 2, 131)[i * 5 % 8] if i % 67 else 0 for i in range(500)]
    q, k, v = (randn((sum(news), h, dim), cuda_device, i) for i, h in enumerate((heads, kv_heads, kv_heads)))
    batch, pages = make_batch(attn, news, news, 16, cuda_device, 1)
    cache = attn.KvCache.empty(pages, 16, kv_heads, dim, cuda_device)
    packed = attn.kv_append(q, k, v, cache, batch, None, packed=True)
    cache.check()
    assert all(torch.equal(x, y) for x, y in zip(packed, (q, k, v)))
    prompt = attn.prompt_attention(q, k, v, batch.token_offsets, 0.125)
    chunk = attn.chunk_attention(q, cache, batch, 0.125)
    at = 0
    for s, n in enumerate(news):
        if n:
            want, bound = ref.attention(q[at:at + n], k[at:at + n], v[at:at + n], 0, 0.125, 0)
            ref.within(prompt[at:at + n], want, bound, f"prompt {s}")
            ref.within(chunk[at:at + n], want, bound, f"sequence {s}")
        at += n


def test_work_past_the_divisions_in_32_bits(attn, cuda_device):
    """2^22 key tiles: 64 sequences of a million keys in 8 heads.  A sequence's table names one page again and again, and another at its end."""
    sequences, heads, dim, page, width = 64, 8, 64, 256, 4096
    pages = 24
    batch = attn.PagedBatch(offsets_of([1] * sequences, cuda_device), torch.full((sequences,), width * page, dtype=torch.int32, device=cuda_device),
                            (torch.arange(sequences, dtype=torch.int32, device=cuda_device) % 8)[:, None].repeat(1, width))
    batch.table[:, -1] = 8 + torch.arange(sequences, dtype=torch.int32, device=cuda_device) % 16
    cache = attn.KvCache(randn((pages, page, heads, dim), cuda_device, 1), randn((pages, page, heads, dim), cuda_device, 2))
    # the last page's keys weigh about as much as all others together
    cache.k[8:] *= 0
    cache.k[8:, :, :, 0] = 10.5
    q = randn((sequences, heads, dim), cuda_device, 3)
    q[:, :, 0] = 7.0
    got = attn.chunk_attention(q, cache, batch, 0.125)
    cache.check()
    q64, k64, v64 = q.double(), cache.k.double(), cache.v.double()
    for s in range(sequences):
        first, last = s % 8, 8 + s % 16
        score = torch.cat([torch.einsum("hd,phd->hp", q64[s], k64[x]) for x in (first, last)], 1) * 0.125
        times = torch.cat([torch.full((page,), width - 1.0), torch.ones(page)]).to(cuda_device).double()
        p = torch.exp(score - score.amax(1, keepdim=True)) * times
        total = p.sum(1, keepdim=True)
        v = torch.cat([v64[first], v64[last]])
        want, terms = torch.einsum("hp,phd->hd", p, v) / total, torch.einsum("hp,phd->hd", p, v.abs()) / total
        # as in the 64-bit form of the tests, and the sums: 2^16 products of 16 keys and 2^13 key tiles, each added with an error of 2^-23 of the sum at most
        size = torch.cat([torch.einsum("hd,phd->hp", q64[s].abs(), k64[x].abs()) for x in (first, last)], 1).amax(1, keepdim=True) * 0.125
        off = ref.BF16 + 2 * (dim + 4) * ref.FP32 * size + 64 * ref.FP32 + 2.0 ** -23 * (2 ** 16 + 2 ** 13)
        ref.within(got[s], want, ref.BF16 * want.abs() + terms * off, f"sequence {s}")


# ---- sharp rows -------------------------------------------------------------------------------------
@pytest.mark.parametrize("dim", [64, 128, 256, 512])
def test_a_row_of_few_keys_is_as_exact_as_its_output(attn, cuda_device, dim):
    """Where a few keys have all the weight, what is rounded of p cancels: the sum that divides is of the rounded values, so that a result is a mean
    of v whose weights are off, and errs by 2^-8 of what v differs from it."""
    n, heads = 512, 4
    q, k, v = (randn((n, heads, dim), cuda_device, 30 + i) for i in range(3))
    q = (q.float() * 6).to(torch.bfloat16)
    scale = dim ** -0.5
    batch, pages = make_batch(attn, [n], [n], 64, cuda_device, 2)
    cache = attn.KvCache.empty(pages, 64, heads, dim, cuda_device)
    attn.kv_append(q, k, v, cache, batch, None)
    q64, k64, v64 = q.double(), k.double(), v.double()
    hidden = torch.ones(n, n, dtype=torch.bool, device=cuda_device).triu(1)
    bound = torch.empty_like(q64)
    want = torch.empty_like(q64)
    for h in range(heads):
        score = (q64[:, h] @ k64[:, h].T * scale).masked_fill(hidden, -torch.inf)
        size = (q64[:, h].abs() @ k64[:, h].abs().T * scale).masked_fill(hidden, 0.0)
        share = torch.softmax(score, -1)
        want[:, h] = share @ v64[:, h]
        # each weight is off by 2^-8 from its rounding, by what its score is off ((dim + 4) 2^-24 of its products' sizes) and its exponential (2^-18
        # and the rounding of an exponent of 60 at most); the sum of the weights by as much, which is the 1.01
        off = 1.01 * share * (ref.BF16 + (dim + 4) * ref.FP32 * size + 128 * ref.FP32)
        bound[:, h] = torch.stack([(off * (v64[None, :, h, x] - want[:, h, x, None]).abs()).sum(1) for x in range(dim)], 1)
        bound[:, h] += want[:, h].abs() * (ref.BF16 + 16 * ref.FP32) + (share @ v64[:, h].abs()) * 2.0 ** -23 * (n // 16)
    for got, what in ((attn.prompt_attention(q, k, v, batch.token_offsets, scale), "prompt"), (attn.chunk_attention(q, cache, batch, scale), "chunk")):
        ref.within(got, want, bound + 1e-30, what)


# ---- outputs in place of inputs -----------------------------------------------------------------------
@pytest.mark.parametrize("tokens", [1, 5, 900])
def test_append_in_place_of_packed_queries(attn, cuda_device, tokens):
    heads, kv_heads, dim, page = 6, 2, 128, 16
    batch, pages = make_batch(attn, [tokens], [tokens + 9], page, cuda_device, 3)
    caches = [attn.KvCache.empty(pages, page, kv_heads, dim, cuda_device) for _ in range(2)]
    q, k, v = (randn((tokens, h, dim), cuda_device, i) for i, h in enumerate((heads, kv_heads, kv_heads)))
    weight, freq = randn((dim,), cuda_device, 6), torch.rand(dim // 2, dtype=torch.float64, device=cuda_device)
    want = attn.kv_append(q, k, v, caches[0], batch, freq, weight, weight)
    assert attn.kv_append(q, k, v, caches[1], batch, freq, weight, weight, out=q) is q
    assert torch.equal(q, want) and torch.equal(caches[0].k, caches[1].k) and torch.equal(caches[0].v, caches[1].v)


def test_outputs_over_what_a_call_reads_are_refused(attn, cuda_device):
    from gevva_b200 import GevvaMoeError
    tokens, heads, kv_heads, dim = 40, 4, 2, 64
    batch, pages = make_batch(attn, [tokens], [tokens], 16, cuda_device, 3)
    cache = attn.KvCache.empty(pages, 16, kv_heads, dim, cuda_device)
    rows = randn((tokens, heads + 2 * kv_heads, dim), cuda_device, 1)
    q, k, v = rows.split((heads, kv_heads, kv_heads), 1)
    before = rows.clone()
    over = rows.view(-1)[:tokens * heads * dim].view(tokens, heads, dim)
    packed = q.contiguous()
    for call in (lambda: attn.kv_append(q, k, v, cache, batch, None, out=over),
                 lambda: attn.kv_append(packed, packed[:, :2], v, cache, batch, None, out=packed),
                 lambda: attn.prompt_attention(q, k, v, batch.token_offsets, 0.125, out=over),
                 lambda: attn.prompt_attention(packed, k, v, batch.token_offsets, 0.125, out=packed),
                 lambda: attn.chunk_attention(q, cache, batch, 0.125, out=over),
                 lambda: attn.chunk_attention(packed, cache, batch, 0.125, out=packed)):
        with pytest.raises(GevvaMoeError, match="argument"):
            call()
    assert torch.equal(rows, before) and torch.equal(packed, q)


def test_a_batch_follows_its_tensors(attn, cuda_device):
    """Tensors of a batch and of a cache that are replaced are the ones that the next call reads."""
    page, dim, length = 16, 64, 100
    batch, pages = make_batch(attn, [1], [length], page, cuda_device, 3, width=20)
    cache = attn.KvCache(*(randn((pages, page, 1, dim), cuda_device, i) for i in range(2)))
    q = randn((1, 2, dim), cuda_device, 3)
    for step in range(10):
        batch.lengths = batch.lengths - 5
        batch.table = batch.table.clone()
        cache.v = cache.v.clone() + 1
        junk = [torch.full((64,), 1 << 20, dtype=torch.int32, device=cuda_device) for _ in range(4)]  # (over what has been given back)
        got = attn.chunk_attention(q, cache, batch, 0.125)
        cache.check()
        length -= 5
        ref.within(got, *ref.attention(q, *gathered(cache, batch, 0, length), length - 1, 0.125, 0), f"step {step}")
        del junk


# ---- reports ------------------------------------------------------------------------------------------
def test_calls_without_a_status_word_report_too(attn, cuda_device):
    import ctypes
    from gevva_b200 import GevvaMoeError
    attn.check(cuda_device)
    lib = attn._lib()
    cache = attn.KvCache(randn((2, 16, 1, 64), cuda_device, 1), randn((2, 16, 1, 64), cuda_device, 2))
    batch = attn.PagedBatch(torch.tensor([0, 1], dtype=torch.int32, device=cuda_device), torch.tensor([20], dtype=torch.int32, device=cuda_device),
                            torch.tensor([[1, 2]], dtype=torch.int32, device=cuda_device))  # (there is no page 2)
    q, out = randn((1, 1, 64), cuda_device, 3), torch.empty((1, 1, 64), dtype=torch.bfloat16, device=cuda_device)
    workspace = torch.empty(lib.gevva_attn_chunk_workspace_bytes(64), dtype=torch.uint8, device=cuda_device)
    stream = torch.cuda.current_stream().cuda_stream
    chunk = attn._CHUNK.pack(q.data_ptr(), 64, 64, cache._address, batch._address, out.data_ptr(), workspace.data_ptr(), 0, 1, 1, 1, 64, 0, 0.125)
    append = attn._APPEND.pack(q.data_ptr(), 64, 64, q.data_ptr(), 64, 64, q.data_ptr(), 64, 64, cache._address, batch._address, 0, 0, 0, out.data_ptr(), 0, 0,
                               0, 1, 1, 1, 64, 0, 0, 1e-6, 0)
    for call in (lambda: lib.gevva_attn_chunk(chunk, stream), lambda: lib.gevva_attn_append(append, stream)):
        assert call() == 0
        with pytest.raises(GevvaMoeError, match="page"):
            attn.check()
        assert attn.last_status(cuda_device) == 0
    attn.prompt_attention(q, q, q, batch.token_offsets, 0.125)
    attn.check()
    assert cache.last_status() == 0
