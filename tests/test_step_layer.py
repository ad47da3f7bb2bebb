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
