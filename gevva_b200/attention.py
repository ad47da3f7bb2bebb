"""The attention side of a decoder layer (ctypes mirror of the gevva_attn_* entry points): norms around the attention block, per-head
norms and rotation with the append to a paged cache, and causal attention over packed prompts or over the cache.  They stand where the
reference's layer loop has them (src/cuda/runtime/prefill.cuh:924-1199, src/cuda/kernels/qkv_transform.cuh).

Calls run on the current stream of their tensors' device, or on `stream`, whose work the caller orders behind what made the inputs; the
tensors that a call makes belong to the stream that it runs on."""
import ctypes
import struct
from dataclasses import dataclass

import torch

from .runtime import GevvaMoeError, _address, _enqueue, library

HEAD_DIMS = (64, 128, 256, 512)
_empty, _empty_like, _contiguous = torch.empty, torch.empty_like, torch.contiguous_format  # (empty_like: half the host's time of empty)


class _Cache(ctypes.Structure):
    _fields_ = ([("keys", ctypes.c_void_p), ("values", ctypes.c_void_p)] +
                [(n, ctypes.c_longlong) for n in ("key_page_stride", "key_slot_stride", "key_head_stride", "value_page_stride",
                                                  "value_slot_stride", "value_head_stride")] +
                [("pages", ctypes.c_int), ("page_size", ctypes.c_int)])


class _Batch(ctypes.Structure):
    _fields_ = [("token_offsets", ctypes.c_void_p), ("lengths", ctypes.c_void_p), ("table", ctypes.c_void_p),
                ("sequences", ctypes.c_int), ("table_width", ctypes.c_int), ("table_stride", ctypes.c_int)]


# gevva_attn_append_args, gevva_attn_prompt_args, gevva_attn_chunk_args: packed in one go, since the conversion of two dozen
# single arguments took the host longer than the launch.
_APPEND = struct.Struct("@" + "Pqq" * 3 + "P" * 9 + "6ifi")
_PROMPT = struct.Struct("@" + "Pqq" * 3 + "P" * 3 + "6ifi")
_CHUNK = struct.Struct("@Pqq" + "P" * 5 + "5if")


def _lib():
    lib = library()
    if getattr(lib, "_gv_attn_ready", False):
        return lib
    vp, i32, f32 = ctypes.c_void_p, ctypes.c_int, ctypes.c_float
    lib.gevva_attn_norm.argtypes = [vp, vp, vp, i32, i32, f32, vp]
    lib.gevva_attn_norm_add.argtypes = [vp] * 8 + [i32, i32, f32, vp]
    for function in (lib.gevva_attn_append, lib.gevva_attn_prompt, lib.gevva_attn_chunk):
        function.argtypes = [ctypes.c_char_p, vp]  # the packed arguments, the stream
    lib.gevva_attention_last_status.argtypes = []
    lib.gevva_attn_chunk_workspace_bytes.argtypes = [i32]
    lib.gevva_attn_chunk_workspace_bytes.restype = ctypes.c_size_t
    lib._gv_attn_ready = True
    return lib


def _status(status, where):
    if status != 0:
        raise GevvaMoeError(status, where)


def last_status(device=None):
    """Waits for the device (None: the current one), then returns and clears the status of the prompt_attention calls on it that were given no
    status word (0 = ok)."""
    with torch.cuda.device(device):
        return _lib().gevva_attention_last_status()


def check(device=None):
    _status(last_status(device), "device status")


def _at(tensor, dtype, shape, device, name):
    """Address of a contiguous tensor on `device`; 0 for None."""
    if tensor is None:
        return 0
    if tensor.dtype is dtype and tensor.shape == shape and tensor.device == device and tensor.is_contiguous():
        return tensor.data_ptr()
    raise ValueError(f"{name}: expected contiguous {dtype} {tuple(shape)} on {device}, got {tensor.dtype} {tuple(tensor.shape)} on {tensor.device}")


def _on(stream, device):
    """Makes `stream` (a torch.cuda.Stream or a raw handle) the current one: what a call makes then belongs to it, as on the current stream."""
    if isinstance(stream, int):
        stream = torch.cuda.ExternalStream(stream, device=device)
    if stream.device != device:
        raise ValueError(f"stream: expected one of {device}, got one of {stream.device}")
    return torch.cuda.stream(stream)


def _pack(layout, *values):
    try:
        return layout.pack(*values)
    except struct.error as error:
        raise ValueError(f"argument out of range: {error}") from None


def _heads(tensor, name, device, shape):
    """(address, strides of a token and of a head) of a bf16 [tokens, heads, dim] on the GPU, its last dimension contiguous."""
    if tensor.dtype is torch.bfloat16 and tensor.shape == shape and tensor.device == device:
        token_stride, head_stride, one = tensor.stride()
        if one == 1:
            return tensor.data_ptr(), token_stride, head_stride
    raise ValueError(f"{name}: expected bfloat16 {tuple(shape)} on {device} with contiguous heads, got {tensor.dtype} {tuple(tensor.shape)} "
                     f"strides {tensor.stride()} on {tensor.device}")


def _queries(q):
    device = q.device
    if q.dim() != 3 or q.shape[2] not in HEAD_DIMS or device.type != "cuda":
        raise ValueError(f"q: expected CUDA bfloat16 (tokens, heads, 64|128|256|512), got {q.dtype} {tuple(q.shape)} on {device}")
    return device, q.shape, _heads(q, "q", device, q.shape)


def _out(out, like, device, name="out"):
    """`out`, or a contiguous tensor of the shape and type of `like`."""
    if out is None:
        return _empty_like(like, memory_format=_contiguous)
    _at(out, torch.bfloat16, like.shape, device, name)
    return out


def _rows(x, name="input"):
    if x.dtype is not torch.bfloat16 or x.dim() != 2 or not x.is_contiguous() or not x.is_cuda:
        raise ValueError(f"{name}: expected contiguous CUDA bfloat16 (rows, width), got {x.dtype} {tuple(x.shape)} on {x.device}")
    if max(x.shape) >= 1 << 31:
        raise ValueError(f"{name}: at most 2^31 - 1 rows and values in one, got {tuple(x.shape)}")
    return x.device, x.shape


def block_norm(x, weight, eps=1e-6, out=None, stream=None):
    """x / sqrt(mean(x^2) + eps) * weight over rows [rows, width] of bf16; width is a multiple of 8 up to 32768.  `out` may be x,
    and otherwise shares no memory with the inputs."""
    device, shape = _rows(x)
    if stream is not None:
        with _on(stream, device):
            return block_norm(x, weight, eps, out)
    rows, width = shape
    out = _out(out, x, device)
    _status(_enqueue(_lib().gevva_attn_norm, device, None, x.data_ptr(), _at(weight, torch.bfloat16, (width,), device, "weight"),
                     out.data_ptr(), rows, width, eps), "block_norm")
    return out


def block_norm_add(x, weight, residual, gate=None, scale=None, next_weight=None, eps=1e-6, out=None, stream=None):
    """(residual + gate * norm(x) * weight) * scale, the norm behind a block; with `next_weight` also the next block's norm of
    the result, returned as (out, next).  gate bf16 [width] and scale bf16 [1] are optional; `out` may be residual or x, and otherwise shares no memory with
    the inputs."""
    device, shape = _rows(x)
    if stream is not None:
        with _on(stream, device):
            return block_norm_add(x, weight, residual, gate, scale, next_weight, eps, out)
    rows, width = shape
    bf16 = torch.bfloat16
    following = None
    out = _out(out, x, device)
    if next_weight is not None:
        following = _empty_like(x)
    _status(_enqueue(_lib().gevva_attn_norm_add, device, None, x.data_ptr(), _at(weight, bf16, (width,), device, "weight"),
                     _at(residual, bf16, shape, device, "residual"), _at(gate, bf16, (width,), device, "gate"),
                     _at(scale, bf16, (1,), device, "scale"), _at(next_weight, bf16, (width,), device, "next_weight"), out.data_ptr(),
                     _address(following), rows, width, eps), "block_norm_add")
    return out if following is None else (out, following)


class KvCache:
    """Keys and values in pages: two bf16 tensors [pages, page_size, kv_heads, dim] (any strides, the last dimension contiguous).
    page_size is a power of two, at least 16.  `status` is the int32 word that calls on this cache report into.  `k` and `v` may be
    replaced by tensors of the same shape; a captured call keeps those that it was captured with."""

    def __init__(self, k, v):
        self._take(k, v)
        self.status = torch.zeros(1, dtype=torch.int32, device=k.device)

    def _take(self, k, v):
        if (k.dtype is not torch.bfloat16 or v.dtype is not torch.bfloat16 or k.dim() != 4 or v.shape != k.shape or not k.is_cuda or
                v.device != k.device or k.stride(3) != 1 or v.stride(3) != 1 or k.shape[3] not in HEAD_DIMS):
            raise ValueError(f"cache: expected two CUDA bfloat16 tensors (pages, page_size, kv_heads, 64|128|256|512), got {k.dtype} "
                             f"{tuple(k.shape)} and {v.dtype} {tuple(v.shape)} on {k.device} and {v.device}")
        pages, page_size = k.shape[:2]
        if pages < 1 or page_size < 16 or page_size & (page_size - 1):
            raise ValueError(f"cache: page_size has to be a power of two, at least 16, and there has to be a page; got {tuple(k.shape)}")
        self._k, self._v = k, v
        self.page_size, self.kv_heads, self.head_dim = page_size, k.shape[2], k.shape[3]
        self.device = k.device
        # (a new one, so that a copy of this handle keeps its own)
        self._packed = _Cache(k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), k.stride(2), v.stride(0), v.stride(1), v.stride(2),
                              pages, page_size)
        self._address = ctypes.addressof(self._packed)

    k = property(lambda self: self._k, lambda self, k: self._take(k, self._v))
    v = property(lambda self: self._v, lambda self, v: self._take(self._k, v))

    @classmethod
    def empty(cls, pages, page_size, kv_heads, head_dim, device="cuda:0"):
        shape = (pages, page_size, kv_heads, head_dim)
        return cls(*(torch.zeros(shape, dtype=torch.bfloat16, device=device) for _ in range(2)))

    def last_status(self):
        """Waits for the device, then returns and clears the status of the calls on this cache (0 = ok)."""
        torch.cuda.synchronize(self.device)
        status = -int(self.status.item())
        if status:
            self.status.zero_()
        return status

    def check(self):
        _status(self.last_status(), "device status")


class PagedBatch:
    """The sequences of a call, int32 on the GPU: new tokens token_offsets[s] .. token_offsets[s + 1] - 1 (rows of the call's
    tensors), lengths[s] keys with the new ones counted, and table [sequences, pages a sequence], whose entry x / page_size is the page of
    position x.  The tensors are read when the calls run, so a captured call can be replayed with other contents (written in place:
    copy_, +=); rows outside the offsets are left as they were.  Each may be replaced by another for as many sequences, which later calls
    read; a captured call keeps those that it was captured with."""

    def __init__(self, token_offsets, lengths, table):
        self._take(token_offsets, lengths, table)

    def _take(self, token_offsets, lengths, table):
        sequences = lengths.shape[0] if lengths.dim() == 1 else -1
        for tensor, shape, name in ((token_offsets, (sequences + 1,), "token_offsets"), (lengths, (sequences,), "lengths")):
            if not tensor.is_cuda:
                raise ValueError(f"{name}: expected a CUDA tensor, got {tensor.device}")
            _at(tensor, torch.int32, shape, table.device, name)
        if table.dtype is not torch.int32 or table.dim() != 2 or table.shape[0] != sequences or table.shape[1] < 1 or sequences < 1 or (
                table.stride(1) != 1 and table.shape[1] > 1) or (sequences > 1 and table.stride(0) >= 1 << 31):
            raise ValueError(f"table: expected int32 ({sequences}, pages a sequence), got {table.dtype} {tuple(table.shape)} strides "
                             f"{table.stride()}")
        self._token_offsets, self._lengths, self._table = token_offsets, lengths, table
        self.device = table.device
        stride = table.stride(0) if sequences > 1 else table.shape[1]
        self._packed = _Batch(token_offsets.data_ptr(), lengths.data_ptr(), table.data_ptr(), sequences, table.shape[1], stride)
        self._address = ctypes.addressof(self._packed)

    token_offsets = property(lambda self: self._token_offsets, lambda self, x: self._take(x, self._lengths, self._table))
    lengths = property(lambda self: self._lengths, lambda self, x: self._take(self._token_offsets, x, self._table))
    table = property(lambda self: self._table, lambda self, x: self._take(self._token_offsets, self._lengths, x))


@dataclass
class Appended:
    """What kv_append leaves beside the cache: rotated queries and, packed, rotated keys and values."""
    q: torch.Tensor
    k: torch.Tensor
    v: torch.Tensor

    def __iter__(self):
        return iter((self.q, self.k, self.v))


def kv_append(q, k, v, cache, batch, frequencies, q_weight=None, k_weight=None, normalize_v=False, eps=1e-6, packed=False, out=None,
              stream=None):
    """Norms q and k over their heads (weights bf16 [dim], None: no norm) and, with normalize_v, v without a weight; turns the pairs
    (j, len(frequencies) + j) of q and k by position * frequencies[j] (a multiple of 8 float64 on the GPU, None: no rotation); stores k
    and v at their positions in the cache.  q, k, v are [tokens, heads, dim], views of one projection's rows for instance.  Returns the queries, with
    `packed` also keys and values as [tokens, kv_heads, dim] for prompt_attention.  `out` takes the queries; it
    may be q itself where that is contiguous, and otherwise shares no memory with q, k or v.  A token without a page is not stored;
    cache.check() reports it."""
    device, shape, q_rows = _queries(q)
    if stream is not None:
        with _on(stream, device):
            return kv_append(q, k, v, cache, batch, frequencies, q_weight, k_weight, normalize_v, eps, packed, out)
    tokens, heads, dim = shape
    kv_heads = cache.kv_heads
    if cache.head_dim != dim or cache.device != device or batch.device != device:
        raise ValueError(f"kv_append: queries of {dim} on {device}, cache of {cache.head_dim} on {cache.device}, batch on {batch.device}")
    k_rows, v_rows = _heads(k, "k", device, (tokens, kv_heads, dim)), _heads(v, "v", device, (tokens, kv_heads, dim))
    rotated = 0 if frequencies is None else 2 * frequencies.numel()
    out = _out(out, q, device)
    k_out, v_out = (_out(None, k, device), _out(None, v, device)) if packed else (None, None)
    bf16 = torch.bfloat16
    args = _pack(_APPEND, *q_rows, *k_rows, *v_rows, cache._address, batch._address,
                        0 if frequencies is None else _at(frequencies, torch.float64, frequencies.shape, device, "frequencies"),
                        _at(q_weight, bf16, (dim,), device, "q_weight"), _at(k_weight, bf16, (dim,), device, "k_weight"), out.data_ptr(),
                        k_out.data_ptr() if packed else 0, v_out.data_ptr() if packed else 0, cache.status.data_ptr(), tokens, heads, kv_heads, dim,
                        rotated, normalize_v, eps, 0)
    _status(_enqueue(_lib().gevva_attn_append, device, None, args), "kv_append")
    return Appended(out, k_out, v_out) if packed else out


def prompt_attention(q, k, v, token_offsets, scale, window=0, out=None, status=None, stream=None):
    """Causal attention of packed prompts: rows token_offsets[s] .. token_offsets[s + 1] - 1 (int32 on the GPU) are sequence s, and
    each sees its sequence's rows up to itself, the last `window` of them where that is not zero.  q [tokens, heads, dim], k and v
    [tokens, kv_heads, dim], kv_heads dividing heads.  Rows outside the offsets are left as they were in `out`, and may hold anything in k
    and v; a sequence's own keys and values have to be finite.  `out` shares no memory with q, k or v.  `status` is an int32 [1] device
    word that a wait which runs out is reported into (the output is then not whole); without one, check() of this module reports it."""
    device, shape, q_rows = _queries(q)
    if stream is not None:
        with _on(stream, device):
            return prompt_attention(q, k, v, token_offsets, scale, window, out, status)
    tokens, heads, dim = shape
    if k.dim() != 3:
        raise ValueError(f"k: expected (tokens, kv_heads, dim), got {tuple(k.shape)}")
    kv_heads = k.shape[1]
    k_rows, v_rows = (_heads(x, name, device, (tokens, kv_heads, dim)) for x, name in ((k, "k"), (v, "v")))
    sequences = token_offsets.numel() - 1
    out = _out(out, q, device)
    args = _pack(_PROMPT, *q_rows, *k_rows, *v_rows, _at(token_offsets, torch.int32, (sequences + 1,), device, "token_offsets"), out.data_ptr(),
                        _at(status, torch.int32, (1,), device, "status"), sequences, tokens, heads, kv_heads, dim, window, scale, 0)
    _status(_enqueue(_lib().gevva_attn_prompt, device, None, args), "prompt_attention")
    return out


def chunk_attention(q, cache, batch, scale, window=0, out=None, stream=None):
    """Causal attention of new tokens over the pages of their sequences, which hold their keys and values already (kv_append):
    one token a sequence when decoding, several for verification and chunked prefill.  A row that sees no key is zero; rows outside the
    offsets are left as they were in `out`, which shares no memory with q or the cache.  Slots that no row of a sequence sees may hold
    anything, others have to be finite.  cache.check() reports lengths beyond the table and pages outside the cache."""
    device, shape, q_rows = _queries(q)
    if stream is not None:
        with _on(stream, device):
            return chunk_attention(q, cache, batch, scale, window, out)
    tokens, heads, dim = shape
    if cache.head_dim != dim or cache.device != device or batch.device != device:
        raise ValueError(f"chunk_attention: queries of {dim} on {device}, cache of {cache.head_dim} on {cache.device}, batch on {batch.device}")
    lib = _lib()
    out = _out(out, q, device)

    def launch(handle):
        # (the workspace's size goes by the device, which is the current one in here)
        workspace = _empty(lib.gevva_attn_chunk_workspace_bytes(dim), dtype=torch.uint8, device=device)
        return lib.gevva_attn_chunk(_pack(_CHUNK, *q_rows, cache._address, batch._address, out.data_ptr(), workspace.data_ptr(),
                                                cache.status.data_ptr(), tokens, heads, cache.kv_heads, dim, window, scale), handle)

    _status(_enqueue(launch, device, None), "chunk_attention")
    return out


@dataclass
class AttentionLayer:
    """The attention half of one decoder layer, in front of a FeedForwardLayer (the wiring of
    src/cuda/runtime/prefill.cuh:924-1199): norm, projection, per-head norms with rotation and append, attention, output projection,
    and the norm behind it with the residual.  The two projections are plain products of a library (torch.mm)."""
    pre: torch.Tensor            # bf16 [hidden] norm in front
    post: torch.Tensor           # bf16 [hidden] norm behind
    qkv_w: torch.Tensor          # bf16 [(heads + 2 * kv_heads) * dim, hidden]: queries, keys, values
    out_w: torch.Tensor          # bf16 [hidden, heads * dim]
    q_norm: torch.Tensor         # bf16 [dim], or None
    k_norm: torch.Tensor
    frequencies: torch.Tensor    # f64 [pairs that turn], or with a step.StepPlan [axes, pairs]
    cache: KvCache
    heads: int
    scale: float
    window: int = 0              # 0: the whole context
    normalize_v: bool = True
    eps: float = 1e-6

    def forward(self, hidden, batch, prompt=False, positions=None):
        """The layer's output, a new tensor [tokens, hidden]; appends the tokens' keys and values to the cache.  With `prompt` every
        sequence is new, a whole prompt of its own, and attention reads the packed keys; otherwise it reads the pages.  Every row of `hidden`
        is a token of a sequence.  `batch` may be a step.StepPlan: tokens then go to the plan's slots, turned by `positions` (int32 [tokens] or
        [axes, tokens]; None: the plan's, the same along all axes), and rows behind the last sequence's pass through with attention of zero."""
        tokens, kv_heads, dim = hidden.shape[0], self.cache.kv_heads, self.cache.head_dim
        x = block_norm(hidden, self.pre, self.eps)
        qkv = torch.mm(x, self.qkv_w.t()).view(tokens, self.heads + 2 * kv_heads, dim)
        q, k, v = qkv.split((self.heads, kv_heads, kv_heads), 1)
        if hasattr(batch, "slots"):
            return self._planned(hidden, q, k, v, batch, prompt, positions)
        if positions is not None:
            raise ValueError("positions: they go with a plan")
        got = kv_append(q, k, v, self.cache, batch, self.frequencies, self.q_norm, self.k_norm, self.normalize_v, self.eps, packed=prompt)
        if prompt:
            seen = prompt_attention(got.q, got.k, got.v, batch.token_offsets, self.scale, self.window, status=self.cache.status)
        else:
            seen = chunk_attention(got, self.cache, batch, self.scale, self.window)
        return self._behind(hidden, seen)

    def _planned(self, hidden, q, k, v, plan, prompt, positions):
        from .step import kv_append_at
        if positions is None:
            positions = plan.positions
            if self.frequencies is not None and self.frequencies.dim() == 2:
                positions = positions.expand(self.frequencies.shape[0], -1)
        got = kv_append_at(q, k, v, self.cache, plan.slots, positions, self.frequencies, self.q_norm, self.k_norm, self.normalize_v, self.eps,
                           packed=prompt)
        seen = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
        if prompt:
            prompt_attention(got.q, got.k, got.v, plan.token_offsets, self.scale, self.window, out=seen, status=self.cache.status)
        else:
            chunk_attention(got, self.cache, plan.batch, self.scale, self.window, out=seen)
        return self._behind(hidden, seen)

    def _behind(self, hidden, seen):
        y = torch.mm(seen.view(hidden.shape[0], seen.shape[1] * seen.shape[2]), self.out_w.t())
        return block_norm_add(y, self.post, hidden, eps=self.eps)
