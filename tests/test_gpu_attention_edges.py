"""The attention operators at the edges of what they take."""
import pytest
import torch

from tests import attention_ref as ref
from tests.test_gpu_attention import attn, gathered, make_batch, randn  # noqa: F401  (attn: a fixture)

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
