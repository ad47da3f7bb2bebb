"""Outputs of the attention calls over memory that they read, at addresses that nothing follows; and what is refused anyway, where outputs and inputs
stand apart."""
import ctypes

import pytest
import torch

from gevva_b200 import attention as attn
from tests import test_attention_refusals as refusals

Q, K, V, OUT, K_OUT, V_OUT = (n << 30 for n in range(1, 7))  # apart
BAD = -3
HEADS, KV, DIM = 4, 2, 64


@pytest.fixture(scope="module")
def lib():
    if torch.cuda.is_available():
        pytest.skip("calls that are not refused would be launched")
    return attn._lib()


def append(lib, tokens=5, q=(Q, HEADS * DIM, DIM), k=(K, KV * DIM, DIM), v=(V, KV * DIM, DIM), q_out=OUT, k_out=K_OUT, v_out=V_OUT):
    return lib.gevva_attn_append(attn._APPEND.pack(*q, *k, *v, ctypes.addressof(refusals.CACHE), ctypes.addressof(refusals.BATCH), 4096, 0, 0, q_out, k_out,
                                                   v_out, 0, tokens, HEADS, KV, DIM, 64, 0, 1e-6, 0), None)


def prompt(lib, tokens=5, q=(Q, HEADS * DIM, DIM), k=(K, KV * DIM, DIM), v=(V, KV * DIM, DIM), out=OUT):
    return lib.gevva_attn_prompt(attn._PROMPT.pack(*q, *k, *v, 4096, out, 0, 2, tokens, HEADS, KV, DIM, 0, 0.1, 0), None)


def chunk(lib, tokens=5, q=(Q, HEADS * DIM, DIM), out=OUT):
    return lib.gevva_attn_chunk(attn._CHUNK.pack(*q, ctypes.addressof(refusals.CACHE), ctypes.addressof(refusals.BATCH), out, 4096, 0, tokens, HEADS, KV, DIM,
                                                 0, 0.1), None)


FUSED = (HEADS + 2 * KV) * DIM  # values of a row of one projection
SIZE = 2 * 5 * HEADS * DIM     # bytes of five tokens' queries


def test_calls_that_share_nothing_are_not_refused(lib):
    assert append(lib) != BAD and prompt(lib) != BAD and chunk(lib) != BAD
    fused = dict(q=(Q, FUSED, DIM), k=(Q + 2 * HEADS * DIM, FUSED, DIM), v=(Q + 2 * (HEADS + KV) * DIM, FUSED, DIM))
    assert append(lib, **fused) != BAD and prompt(lib, **fused) != BAD
    # in place of its own input, packed; a single token of a projection is
    assert append(lib, q_out=Q) != BAD and append(lib, k_out=K, v_out=V) != BAD
    assert append(lib, tokens=1, q_out=Q, **fused) != BAD
    # right in front and right behind
    for out in (Q - SIZE, Q + SIZE):
        assert append(lib, q_out=out) != BAD and prompt(lib, out=out) != BAD and chunk(lib, out=out) != BAD


def test_outputs_over_inputs_are_refused(lib):
    fused = dict(q=(Q, FUSED, DIM), k=(Q + 2 * HEADS * DIM, FUSED, DIM), v=(Q + 2 * (HEADS + KV) * DIM, FUSED, DIM))
    assert append(lib, q_out=Q, **fused) == BAD  # later rows' queries, keys and values stand where packed queries go
    for out in (Q, Q + 32, Q - SIZE + 32, Q + SIZE - 32):
        assert prompt(lib, out=out) == BAD and chunk(lib, out=out) == BAD
        assert append(lib, q_out=out) == (append(lib) if out == Q else BAD)
    for out in (K, K + 32, V, V - 32):
        assert prompt(lib, out=out) == BAD and append(lib, q_out=out) == BAD
    assert append(lib, k_out=Q) == BAD and append(lib, v_out=K) == BAD and append(lib, k_out=V) == BAD and append(lib, k_out=K + 16) == BAD
    assert append(lib, tokens=1, q_out=Q + 2 * HEADS * DIM, **fused) == BAD  # the token's keys


def test_memory_between_rows_and_heads_is_free(lib):
    """Against every value written out, for strides in both orders and outputs all around."""
    tokens, heads, dim = 3, 2, 64
    bad = ok = 0
    for token_stride, head_stride in ((128, 64), (512, 64), (1024, 256), (64, 192), (64, 1024), (256, 128), (8192, 4096)):
        used = {t * token_stride + h * head_stride + i for t in range(tokens) for h in range(heads) for i in range(dim)}
        for at in range(-tokens * heads * dim - 64, 3 * 8192, 32):
            out = Q + 2 * at
            want = any(x in used for x in range(at, at + tokens * heads * dim, 16))
            got = lib.gevva_attn_chunk(attn._CHUNK.pack(Q, token_stride, head_stride, ctypes.addressof(refusals.CACHE), ctypes.addressof(refusals.BATCH), out,
                                                        4096, 0, tokens, heads, KV, dim, 0, 0.1), None)
            assert (got == BAD) == want, (token_stride, head_stride, at)
            bad, ok = bad + want, ok + (not want)
    assert bad > 100 and ok > 100


@pytest.mark.parametrize("change", refusals.SHAPES + refusals.PAGES + [s for s in refusals.SOFTMAX if "out" not in s])
def test_chunk_refuses_with_its_output_apart(lib, change):
    assert refusals.chunk(lib, out=OUT) != BAD
    assert refusals.chunk(lib, **dict(dict(out=OUT), **change)) == BAD


@pytest.mark.parametrize("change", refusals.SHAPES + [s for s in refusals.SOFTMAX if "out" not in s] + [
    dict(k=refusals.rows(4098)), dict(v=refusals.rows(head=4)), dict(offsets=None), dict(sequences=0), dict(reserved=1)])
def test_prompt_refuses_with_its_output_apart(lib, change):
    assert refusals.prompt(lib, out=OUT) != BAD
    assert refusals.prompt(lib, **dict(dict(out=OUT), **change)) == BAD


@pytest.mark.parametrize("change", refusals.SHAPES + refusals.PAGES + [
    dict(rotated=-16), dict(rotated=80), dict(rotated=8), dict(freq=None), dict(freq=4100), dict(eps=-1.0), dict(eps=float("nan")), dict(k_out=K_OUT),
    dict(v_out=V_OUT), dict(qw=4098), dict(reserved=1)])
def test_append_refuses_with_its_outputs_apart(lib, change):
    assert refusals.append(lib, q_out=OUT) != BAD
    assert refusals.append(lib, **dict(dict(q_out=OUT), **change)) == BAD


def test_an_append_without_rows_does_nothing(lib):
    assert refusals.append(lib, q=refusals.rows(None), tokens=0, q_out=None) == 0


def test_norms_over_what_they_read(lib):
    """Rows are read before they are written, other rows and the vectors are not: an output is an input, row for row, or shares nothing with any."""
    rows, width = 7, 64
    size, x, w, r, g, s, nw, out, nxt = 2 * rows * width, *(n << 30 for n in range(1, 9))

    def norm(to=out, x=x, w=w):
        return lib.gevva_attn_norm(x, w, to, rows, width, 1e-6, None)

    def add(to=out, nxt=nxt, x=x, r=r):
        return lib.gevva_attn_norm_add(x, w, r, g, s, nw, to, nxt, rows, width, 1e-6, None)

    for to in (out, x, x - size, x + size, w - size, w + 2 * width):
        assert norm(to) != BAD, to
    for to in (out, x, r, x - size, r + size, g - size, s - size, s + 16, nw + 2 * width, nxt - size, nxt + size):
        assert add(to) != BAD, to
    for to in (nxt, x, r, out - size):
        assert add(nxt=to) != BAD, to
    for to in (x + 16, x - size + 16, x + size - 16, w, w - 16, w + 2 * width - 16):
        assert norm(to) == BAD, to
    for to in (x + 16, r - 16, w, g, g + 2 * width - 16, s - 16, s, nw, nxt, nxt + 16, nxt - size + 16):
        assert add(to) == BAD, to
    for to in (out, out + 16, x + 16, r - 16, w, g, s - size + 16, nw - 16):
        assert add(nxt=to) == BAD, to
    assert add(r=x) != BAD and add(r=x, to=x) != BAD
