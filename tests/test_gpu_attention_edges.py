"""The attention operators at the edges of what they take."""
import pytest
import torch

from tests.test_gpu_attention import attn, make_batch, randn  # noqa: F401  (attn: a fixture)

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
