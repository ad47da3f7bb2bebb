"""What the layer and the stack do around the step's calls, on the host with stand-ins for the kernels."""
import types

import pytest
import torch

from gevva_b200 import attention as attn
from gevva_b200.synthetic import SyntheticStack


def test_a_layer_of_no_rows(monkeypatch):
    """No rows give no rows (a batch none of whose sequences has a token)."""
    monkeypatch.setattr(attn, "block_norm_add", lambda y, post, hidden, eps: hidden + y)
    layer = attn.AttentionLayer(pre=None, post=None, qkv_w=None, out_w=torch.ones(32, 128), q_norm=None, k_norm=None, frequencies=None, cache=None, heads=2, scale=1.0)
    for rows in (0, 1, 3):
        assert layer._behind(torch.ones(rows, 32), torch.ones(rows, 2, 64)).tolist() == [[129.0] * 32] * rows


@pytest.mark.parametrize("probability", [False, True])
def test_a_row_without_a_token_stays_without_one(probability):
    """Minus one is not the vocabulary's last row: zeros go through the layers, and no token comes out, also where the tokens are written in place."""
    seen = []

    class Head:
        rows = torch.arange(1.0, 6.0)[:, None].expand(5, 3).contiguous()

        def forward(self, hidden, uniforms, probability=False, out=None):
            tokens = hidden[:, 0].int() % 5
            if out is not None:
                tokens = out.copy_(tokens)
            return (tokens, torch.ones(len(tokens))) if probability else tokens

    stack = types.SimpleNamespace(head=Head(), attention=[None], forward=lambda hidden, concurrent, plan: seen.append(hidden.clone()) or hidden)
    tokens = torch.tensor([3, -1, 0, 4, -7], dtype=torch.int32)
    for out in (None, tokens.clone()):
        given = tokens if out is None else out
        got = SyntheticStack.decode(stack, given, None, None, probability=probability, out=out)
        chosen = got[0] if probability else got
        assert chosen.tolist() == [4, -1, 1, 0, -1] and (not probability or got[1].tolist() == [1, 0, 1, 1, 0])
        assert seen.pop()[:, 0].tolist() == [4, 0, 1, 5, 0] and (out is None or out is chosen)
    assert tokens.tolist() == [3, -1, 0, 4, -7] and Head.rows[0, 0] == 1
