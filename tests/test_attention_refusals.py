"""What the attention calls refuse, before any CUDA call: the C ABI on addresses that are never followed, the Python mirror on CPU tensors."""
import ctypes
import os
import re

import pytest
import torch

from gevva_b200 import attention as attn

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A, BAD = 4096, -3  # an aligned address that nothing follows; the status of a refusal


@pytest.fixture(scope="module")
def lib():
    return attn._lib()


def rows(data=A, token=512, head=64):
    return data or 0, token, head


def cache(**change):
    fields = dict(keys=A, values=A, key_page_stride=16 * 128, key_slot_stride=128, key_head_stride=64, value_page_stride=16 * 128,
                  value_slot_stride=128, value_head_stride=64, pages=4, page_size=16)
    return attn._Cache(*dict(fields, **change).values())


def batch(**change):
    fields = dict(token_offsets=A, lengths=A, table=A, sequences=2, table_width=3, table_stride=3)
    return attn._Batch(*dict(fields, **change).values())


CACHE, BATCH = cache(), batch()


def chunk(lib, q=None, c=None, b=None, tokens=3, heads=4, kv_heads=2, dim=64, scale=0.1, window=0, out=A, workspace=A):
    return lib.gevva_attn_chunk(attn._CHUNK.pack(*(q or rows()), ctypes.addressof(c or CACHE), ctypes.addressof(b or BATCH), out or 0, workspace or 0, 0,
                                                 tokens, heads, kv_heads, dim, window, scale), None)


def prompt(lib, q=None, k=None, v=None, offsets=A, sequences=2, tokens=3, heads=4, kv_heads=2, dim=64, scale=0.1, window=0, out=A, reserved=0):
    return lib.gevva_attn_prompt(attn._PROMPT.pack(*(q or rows()), *(k or rows()), *(v or rows()), offsets or 0, out or 0, 0, sequences, tokens, heads,
                                                   kv_heads, dim, window, scale, reserved), None)


def append(lib, q=None, c=None, b=None, tokens=3, heads=4, kv_heads=2, dim=64, freq=A, rotated=64, eps=1e-6, q_out=A, k_out=None, v_out=None, qw=None,
           reserved=0):
    return lib.gevva_attn_append(attn._APPEND.pack(*(q or rows()), *rows(), *rows(), ctypes.addressof(c or CACHE), ctypes.addressof(b or BATCH), freq or 0,
                                                   qw or 0, 0, q_out or 0, k_out or 0, v_out or 0, 0, tokens, heads, kv_heads, dim, rotated, 0, eps,
                                                   reserved), None)


SHAPES = [dict(tokens=-1), dict(heads=0), dict(kv_heads=0), dict(heads=5), dict(heads=258, kv_heads=2), dict(dim=96), dict(dim=0), dict(dim=1024),
          dict(q=rows(A + 8)), dict(q=rows(None)), dict(q=rows(token=516)), dict(q=rows(token=0)), dict(q=rows(token=-512)), dict(q=rows(head=60)),
          dict(q=rows(head=0))]
PAGES = [dict(c=cache(keys=None)), dict(c=cache(values=A + 4)), dict(c=cache(pages=0)), dict(c=cache(page_size=8)), dict(c=cache(page_size=48)),
         dict(c=cache(key_slot_stride=100)), dict(c=cache(value_page_stride=0)), dict(c=cache(key_head_stride=-64)), dict(b=batch(token_offsets=None)),
         dict(b=batch(lengths=None)), dict(b=batch(table=None)), dict(b=batch(sequences=0)), dict(b=batch(table_width=0)), dict(b=batch(table_stride=2)),
         dict(b=batch(table_width=1 << 27, table_stride=1 << 27))]
SOFTMAX = [dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=1e31), dict(window=-1), dict(out=None), dict(out=A + 16)]


@pytest.mark.parametrize("change", SHAPES + PAGES + SOFTMAX + [dict(workspace=None), dict(workspace=A + 16)])
def test_chunk(lib, change):
    assert chunk(lib, **change) == BAD


@pytest.mark.parametrize("change", SHAPES + SOFTMAX + [dict(k=rows(A + 2)), dict(v=rows(head=4)), dict(offsets=None), dict(sequences=0), dict(reserved=1)])
def test_prompt(lib, change):
    assert prompt(lib, **change) == BAD


@pytest.mark.parametrize("change", SHAPES + PAGES + [dict(rotated=-16), dict(rotated=80), dict(rotated=8), dict(freq=None), dict(freq=A + 4),
                                                     dict(eps=-1.0), dict(eps=float("nan")), dict(q_out=None), dict(k_out=A), dict(v_out=A),
                                                     dict(qw=A + 2), dict(reserved=1)])
def test_append(lib, change):
    assert append(lib, **change) == BAD


def test_norms(lib):
    def norm(x=A, w=A, out=A, n=3, width=64, eps=1e-6):
        return lib.gevva_attn_norm(x, w, out, n, width, eps, None)

    def add(x=A, w=A, r=A, gate=None, scale=None, nw=None, out=A, nxt=None, n=3, width=64, eps=1e-6):
        return lib.gevva_attn_norm_add(x, w, r, gate, scale, nw, out, nxt, n, width, eps, None)

    for change in (dict(x=None), dict(x=A + 2), dict(w=None), dict(out=A + 8), dict(n=-1), dict(width=0), dict(width=12), dict(width=32776),
                   dict(eps=-1.0), dict(eps=float("nan"))):
        assert norm(**change) == BAD and add(**change) == BAD, change
    for change in (dict(r=None), dict(gate=A + 2), dict(scale=A + 1), dict(nw=A), dict(nxt=A), dict(nw=A + 2, nxt=A)):
        assert add(**change) == BAD, change


def test_packed_arguments_have_the_layout_of_the_header(lib, tmp_path):
    import shutil
    import subprocess
    if shutil.which("gcc") is None:
        pytest.skip("needs gcc")
    source = tmp_path / "sizes.c"
    names = ("append", "prompt", "chunk")
    source.write_text('#include <stdio.h>\n#include "gevva_moe.h"\nint main(void) {' + "".join(
        f'printf("%zu\\n", sizeof(gevva_attn_{n}_args));' for n in names) + "return 0; }")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), "-o", str(tmp_path / "sizes"), str(source)], check=True)
    sizes = [int(x) for x in subprocess.run([str(tmp_path / "sizes")], capture_output=True, text=True, check=True).stdout.split()]
    assert sizes == [attn._APPEND.size, attn._PROMPT.size, attn._CHUNK.size]
    for function in (lib.gevva_attn_append, lib.gevva_attn_prompt, lib.gevva_attn_chunk):
        assert function(None, None) == BAD


def test_calls_without_rows_do_nothing(lib):
    assert chunk(lib, q=rows(None), tokens=0, out=None) == 0 and prompt(lib, q=rows(None), k=rows(None), v=rows(None), tokens=0, out=None) == 0
    assert append(lib, q=rows(None), tokens=0, q_out=None) in (0, BAD)  # (its keys and values are given here)
    assert lib.gevva_attn_norm(None, A, None, 0, 64, 1e-6, None) == 0
    assert lib.gevva_attn_chunk_workspace_bytes(96) == 0


def test_every_declared_call_is_exported(lib):
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "gevva_moe.h")).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(gevva_attn_[a-z0-9_]+)\s*\(", text)))
    assert len(names) == 6
    for name in names:
        assert hasattr(lib, name), name
    assert lib.gevva_moe_strerror(-7).decode() == "position without a page of the cache"


def test_python_mirror_refuses():
    x = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    at = torch.zeros(2, dtype=torch.int32)
    w = torch.ones(64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        attn.prompt_attention(x, x, x, at, 1.0)
    with pytest.raises(ValueError, match="CUDA"):
        attn.KvCache(torch.zeros(1, 16, 1, 64, dtype=torch.bfloat16), torch.zeros(1, 16, 1, 64, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="token_offsets"):
        attn.PagedBatch(at, at[:1], torch.zeros(1, 1, dtype=torch.int32))
    with pytest.raises(ValueError, match="input"):
        attn.block_norm(x[:, 0], w)
    with pytest.raises(ValueError, match="input"):
        attn.block_norm_add(x[:, 0], w, x[:, 0])
    fields = [n for n, _ in attn._Cache._fields_]
    assert fields[-2:] == ["pages", "page_size"] and ctypes.sizeof(attn._Cache) == 72 and ctypes.sizeof(attn._Batch) == 40


def test_numbers_that_an_argument_cannot_hold():
    for window, scale in ((1 << 31, 0.1), (-(1 << 31) - 1, 0.1), (0, None)):
        with pytest.raises(ValueError, match="out of range"):
            attn._pack(attn._CHUNK, A, 8, 8, A, A, A, A, 0, 1, 1, 1, 64, window, scale)
