"""KvCache and PagedBatch pass addresses on: they are those of the tensors that the handles hold now.  Stand-ins for tensors on a GPU."""
import copy
import ctypes

import pytest
import torch

from gevva_b200 import attention as attn

DEVICE = torch.device("cuda:0")


class Stand:
    """What the handles ask of a tensor."""
    is_cuda = True

    def __init__(self, address, shape, dtype=torch.int32, strides=None, device=DEVICE):
        self.address, self.shape, self.dtype, self.device = address, torch.Size(shape), dtype, device
        self.strides = strides or [int(torch.tensor(shape[i + 1:]).prod()) for i in range(len(shape))]

    def dim(self):
        return len(self.shape)

    def stride(self, i=None):
        return tuple(self.strides) if i is None else self.strides[i]

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return self.address


def batch(sequences=2, width=3):
    return attn.PagedBatch(Stand(4096, (sequences + 1,)), Stand(8192, (sequences,)), Stand(12288, (sequences, width)))


@pytest.fixture
def cache(monkeypatch):
    monkeypatch.setattr(torch, "zeros", lambda *shape, **_: Stand(64, shape))
    return attn.KvCache(*(Stand(at, (4, 16, 2, 64), torch.bfloat16) for at in (4096, 1 << 20)))


def test_a_batch_passes_the_tensors_that_it_holds():
    b = batch()
    b.lengths = Stand(1 << 16, (2,))
    b.token_offsets = Stand(1 << 17, (3,))
    b.table = Stand(1 << 18, (2, 5), strides=(7, 1))
    assert (b.lengths.address, b.token_offsets.address, b.table.address) == (1 << 16, 1 << 17, 1 << 18)
    p = b._packed
    assert (p.lengths, p.token_offsets, p.table, p.sequences, p.table_width, p.table_stride) == (1 << 16, 1 << 17, 1 << 18, 2, 5, 7)
    assert b._address == ctypes.addressof(p)


def test_a_batch_refuses_tensors_that_do_not_fit():
    b = batch()
    with pytest.raises(ValueError, match="expected contiguous"):
        b.lengths = Stand(0, (3,))  # (as many sequences as before)
    before = bytes(b._packed)
    for name, wrong in (("lengths", Stand(0, (2,), torch.int64)), ("token_offsets", Stand(0, (2,))),
                        ("table", Stand(0, (3, 3))), ("table", Stand(0, (2, 3), torch.int64)), ("table", Stand(0, (2, 3), strides=(1, 2))),
                        ("table", Stand(0, (2, 3), strides=(1 << 31, 1))),  # (a number that the call's argument cannot hold)
                        ("lengths", Stand(0, (2,), device=torch.device("cuda:1")))):
        with pytest.raises(ValueError, match=name):
            setattr(b, name, wrong)
    assert bytes(b._packed) == before and b.lengths.address == 8192 and b.table.address == 12288


def test_a_cache_passes_the_tensors_that_it_holds(cache):
    cache.k = Stand(1 << 21, (4, 16, 2, 64), torch.bfloat16, strides=(4096, 128, 64, 1))
    cache.v = Stand(1 << 22, (4, 16, 2, 64), torch.bfloat16)
    p = cache._packed
    assert (p.keys, p.values, p.key_page_stride, p.value_page_stride) == (1 << 21, 1 << 22, 4096, 2048)
    for wrong in (Stand(0, (5, 16, 2, 64), torch.bfloat16), Stand(0, (4, 16, 2, 64), torch.float16), Stand(0, (4, 16, 2, 64), torch.bfloat16, device="cuda:1")):
        with pytest.raises(ValueError, match="cache"):
            cache.v = wrong
    assert p.values == 1 << 22 and cache.v.address == 1 << 22


def test_a_copy_of_a_handle_keeps_its_own(cache):
    b = batch()
    other, other_cache = copy.copy(b), copy.copy(cache)
    other.lengths = Stand(1 << 16, (2,))
    other_cache.v = Stand(1 << 22, (4, 16, 2, 64), torch.bfloat16)
    for handle, copied, field in ((b, other, "lengths"), (cache, other_cache, "values")):
        at = [type(h._packed).from_address(h._address) for h in (handle, copied)]
        assert getattr(at[0], field) == (8192 if field == "lengths" else 1 << 20) and getattr(at[1], field) == (1 << 16 if field == "lengths" else 1 << 22)
