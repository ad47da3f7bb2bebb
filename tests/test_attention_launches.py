"""What the attention calls launch, and what they refuse as too large, on the CUDA runtime that records launches (see test_launch_sequence.py)."""
import ctypes

import pytest
import torch

from gevva_b200 import attention as attn
from tests.test_launch_sequence import ADDRESS, recorder  # noqa: F401  (a fixture)


@pytest.fixture(scope="module")
def lib(recorder):  # noqa: F811
    f32, vp, i32 = ctypes.c_float, ctypes.c_void_p, ctypes.c_int
    recorder.lib.gevva_attn_norm.argtypes = [vp, vp, vp, i32, i32, f32, vp]
    recorder.lib.gevva_attn_norm_add.argtypes = [vp] * 8 + [i32, i32, f32, vp]
    return recorder


@pytest.mark.parametrize("rows", [1, 4, 5, 2 ** 31 - 5, 2 ** 31 - 4, 2 ** 31 - 3, 2 ** 31 - 1])
def test_norms_of_any_number_of_rows(lib, rows):
    x = 1 << 20  # (the weights lie in front of the rows)
    assert lib.lib.gevva_attn_norm(x, ADDRESS, x, rows, 64, 1e-6, None) == 0
    assert lib.lib.gevva_attn_norm_add(x, ADDRESS, x, None, None, None, x, None, rows, 64, 1e-6, None) == 0
    assert [(x["kernel"], x["grid"]) for x in lib.launches()] == [("block_norm_kernel<0>", -(-rows // 4))] * 2
    assert lib.lib.gevva_attn_norm(x, ADDRESS, x, rows, 2816, 1e-6, None) == 0
    assert [x["grid"] for x in lib.launches()] == [rows]


@pytest.mark.parametrize("shape", [(1 << 31, 8), ((1 << 32) + 5, 8), (8, (1 << 32) + 8)])
def test_rows_that_an_argument_cannot_hold(shape):
    """ctypes would cut them to 32 bits, and the call would leave the rest of the rows out."""
    class Stand:
        dtype, device, is_cuda = torch.bfloat16, torch.device("cuda:0"), True
        shape = None

        def dim(self):
            return 2

        def is_contiguous(self):
            return True

    Stand.shape = torch.Size(shape)
    for call in (lambda: attn.block_norm(Stand(), None), lambda: attn.block_norm_add(Stand(), None, None)):
        with pytest.raises(ValueError, match="at most"):
            call()


def test_a_prompt_of_more_items_than_a_grid_has(lib):
    heads = 1024

    def call(tokens):
        rows = (ADDRESS, heads * 64, 64)
        return lib.lib.gevva_attn_prompt(attn._PROMPT.pack(*rows, *rows, *rows, ADDRESS, 1 << 60, 0, 1, tokens, heads, heads, 64, 0, 0.1, 0), None)

    assert call(1 << 28) == 0 and [x["grid"] for x in lib.launches()] == [heads * (((1 << 28) + 255) // 256)]
    assert call(1 << 30) == -6 and lib.launches() == []
