"""What a serving step has around its layers (ctypes mirror of the gevva_step_* entry points): rows, pages and places of its tokens from the
lengths of its requests, the append to the cache at those places with positions of one or several axes, and the tokens that its
logits give.

    plan = StepPlan.in_place(lengths, table, pool, tokens)          # once; a captured step goes on by itself
    plan_step(lengths, news, table, pool, page_size, tokens, out=plan)
    q = kv_append_at(q, k, v, cache, plan.slots, plan.positions, frequencies, ...)
    y = chunk_attention(q, cache, plan.batch, scale)
    tokens = sample_tokens(logits, uniforms, temperature=..., top_k=..., top_p=..., min_p=...)

Calls run on the current stream of their tensors' device, or on `stream`, whose work the caller orders behind what made the inputs; the
tensors that a call makes belong to the stream that it runs on."""
import ctypes
import struct
from dataclasses import dataclass

import torch

from .attention import Appended, PagedBatch, _at, _empty, _heads, _on, _out, _pack, _queries, _status, block_norm
from .runtime import _address, _enqueue, library

MAX_REQUESTS = 16384
MAX_VOCABULARY = 1 << 19

# gevva_step_plan_args, _trim_args, _append_args, _sample_args
_PLAN = struct.Struct("@12P6i")
_TRIM = struct.Struct("@8P6i")
_APPEND_AT = struct.Struct("@" + "Pqq" * 3 + "PPPq" + "P" * 7 + "7if")
_SAMPLE = struct.Struct("@Pq7P3if")


def _lib():
    lib = library()
    if getattr(lib, "_gv_step_ready", False):
        return lib
    for function in (lib.gevva_step_plan, lib.gevva_step_trim, lib.gevva_step_append, lib.gevva_step_sample):
        function.argtypes = [ctypes.c_char_p, ctypes.c_void_p]  # the packed arguments, the stream
    lib._gv_step_ready = True
    return lib


class PagePool:
    """Pages of a cache that requests get and give back: `free` int32 [pages] lists them, in any order, and the first `taken` (int32 [1], on
    the GPU as well) are handed out.  plan_step takes from it and trim_step gives back.  `status` is the int32 word that calls on this
    pool report into.  Each may be replaced, which later calls follow; a captured call keeps those that it was captured with."""

    def __init__(self, free, taken=None, status=None):
        taken = torch.zeros(1, dtype=torch.int32, device=free.device) if taken is None else taken
        self._take(free, taken, torch.zeros(1, dtype=torch.int32, device=free.device) if status is None else status)

    def _take(self, free, taken, status):
        if not free.is_cuda or free.dtype is not torch.int32 or free.dim() != 1 or free.numel() < 1 or not free.is_contiguous():
            raise ValueError(f"free: expected contiguous CUDA int32 (pages,), got {free.dtype} {tuple(free.shape)} on {free.device}")
        addresses = (free.data_ptr(), _at(taken, torch.int32, (1,), free.device, "taken"), _at(status, torch.int32, (1,), free.device, "status"))
        self.device, self.pages = free.device, free.numel()
        self._free, self._taken, self._status, self._addresses = free, taken, status, addresses

    free = property(lambda self: self._free, lambda self, x: self._take(x, self._taken, self._status))
    taken = property(lambda self: self._taken, lambda self, x: self._take(self._free, x, self._status))
    status = property(lambda self: self._status, lambda self, x: self._take(self._free, self._taken, x))

    @classmethod
    def whole(cls, pages, device="cuda:0"):
        """All of a cache's pages, none handed out."""
        return cls(torch.arange(pages, dtype=torch.int32, device=device))

    def last_status(self):
        """Waits for the device, then returns and clears the status of the calls on this pool (0 = ok)."""
        torch.cuda.synchronize(self.device)
        status = -int(self.status.item())
        if status:
            self.status.zero_()
        return status

    def check(self):
        _status(self.last_status(), "device status")


class StepPlan:
    """What plan_step says of a step: token_offsets [sequences + 1], lengths [sequences] with the new tokens counted, slots and positions
    [tokens], taken [1] and the table that it was made for; all int32 on the GPU.  `batch` is what chunk_attention takes: one handle, whose
    tensors are the plan's."""

    def __init__(self, token_offsets, lengths, slots, positions, taken, table):
        self.token_offsets, self.lengths, self.slots, self.positions, self.taken, self.table = token_offsets, lengths, slots, positions, taken, table
        self._batch, self._goes_on = None, False

    @classmethod
    def empty(cls, sequences, table, tokens, lengths=None, taken=None):
        own = _empty(2 * sequences + 2 + 2 * tokens, dtype=torch.int32, device=table.device)
        offsets, after, slots, positions, count = own.split_with_sizes((sequences + 1, sequences, tokens, tokens, 1))
        return cls(offsets, after if lengths is None else lengths, slots, positions, count if taken is None else taken, table)

    @classmethod
    def in_place(cls, lengths, table, pool, tokens):
        """One whose lengths and count of pages are the state itself: the step goes on from what it has written.  That is the lengths and the
        pool's count which plan_step is given with this plan, also where they are other tensors than before (what trim_step returned, for
        instance); the plan's own follow, and a captured call keeps those that it was captured with."""
        plan = cls.empty(lengths.shape[0], table, tokens, lengths, pool.taken)
        plan._goes_on = True
        return plan

    @property
    def batch(self):
        batch = self._batch
        if batch is None:
            batch = self._batch = PagedBatch(self.token_offsets, self.lengths, self.table)
        elif batch.token_offsets is not self.token_offsets or batch.lengths is not self.lengths or batch.table is not self.table:
            batch._take(self.token_offsets, self.lengths, self.table)
        return batch

    def _follow(self, lengths, taken):
        self.lengths, self.taken = lengths, taken
        if self._batch is not None:
            self.batch


@dataclass
class Trimmed:
    """What trim_step leaves: lengths [sequences], taken [1]."""
    lengths: torch.Tensor
    taken: torch.Tensor


def _requests(lengths, counts, name, table, pool):
    """(device, number of requests, stride of the table) of a call over a pool."""
    device, i32 = pool.device, torch.int32
    sequences = lengths.shape[0] if lengths.dim() == 1 else -1
    if sequences < 1 or not lengths.is_cuda:
        raise ValueError(f"lengths: expected CUDA int32 (sequences,), got {lengths.dtype} {tuple(lengths.shape)} on {lengths.device}")
    if sequences > MAX_REQUESTS:
        raise ValueError(f"lengths: at most {MAX_REQUESTS} requests, got {sequences}")
    _at(lengths, i32, (sequences,), device, "lengths")
    _at(counts, i32, (sequences,), device, name)
    rows, width = table.shape if table.dim() == 2 else (-1, 0)
    stride, one = table.stride() if rows > 0 else (0, 1)
    if table.dtype is not i32 or rows != sequences or width < 1 or table.device != device or (one != 1 and width > 1):
        raise ValueError(f"table: expected int32 ({sequences}, pages a sequence) on {device}, got {table.dtype} {tuple(table.shape)} strides "
                         f"{table.stride()} on {table.device}")
    return device, sequences, stride if sequences > 1 else width


def plan_step(lengths, news, table, pool, page_size, tokens, shift=None, out=None, stream=None):
    """Rows, pages and places of the step's new tokens, as a StepPlan: request s, which has lengths[s] tokens in the cache and the pages for
    them in its row of `table`, gets news[s] more.  The table is written with pages out of `pool`; `tokens` is how many rows the
    step's tensors have, and rows behind the last request's get slot -1.  `shift` [sequences] is added to the positions (not to the
    places).  `out` takes the plan; one in place (StepPlan.in_place) writes its lengths to `lengths` and its count to pool.taken, other outputs
    share no memory with what is read.  Without it the pool's count stays as it was, and the plan has the new one.  Requests whose
    numbers cannot be, too few pages or more tokens than rows leave everything as it was and no row a token; pool.check() reports them."""
    device, sequences, stride = _requests(lengths, news, "news", table, pool)
    if stream is not None:
        with _on(stream, device):
            return plan_step(lengths, news, table, pool, page_size, tokens, shift, out)
    i32 = torch.int32
    if out is None:
        out = StepPlan.empty(sequences, table, tokens)
        at = out.token_offsets.data_ptr()
        addresses = (at, at + 4 * (sequences + 1), at + 4 * (2 * sequences + 1), at + 4 * (2 * sequences + 1 + tokens), at + 4 * (2 * sequences + 1 + 2 * tokens))
    else:
        if out.table is not table and (out.table.data_ptr() != table.data_ptr() or out.table.shape != table.shape or out.table.stride() != table.stride()):
            raise ValueError("out: a plan for another table")
        after, count = (lengths, pool.taken) if out._goes_on else (out.lengths, out.taken)
        addresses = (_at(out.token_offsets, i32, (sequences + 1,), device, "out.token_offsets"), _at(after, i32, (sequences,), device, "out.lengths"),
                     _at(out.slots, i32, (tokens,), device, "out.slots"), _at(out.positions, i32, (tokens,), device, "out.positions"),
                     _at(count, i32, (1,), device, "out.taken"))
    free, taken, status = pool._addresses
    args = _pack(_PLAN, lengths.data_ptr(), news.data_ptr(), _at(shift, i32, (sequences,), device, "shift"), table.data_ptr(), free, taken, *addresses, status,
                 sequences, table.shape[1], stride, pool.pages, page_size, tokens)
    _status(_enqueue(_lib().gevva_step_plan, device, None, args), "plan_step")
    if out._goes_on and (out.lengths is not lengths or out.taken is not pool.taken):
        out._follow(lengths, pool.taken)
    return out


def trim_step(lengths, keep, table, pool, page_size, out=None, stream=None):
    """Requests that get shorter or end: of request s min(lengths[s], max(keep[s], 0)) tokens stay, and the pages that it then does not need
    go back to the pool's list, in the places where plan_step would hand them out again in the same order.  Returns the new lengths and
    count of pages (a Trimmed, or `out`, whose lengths may be `lengths` and whose taken pool.taken); the table is left as it is.
    pool.check() reports lengths that cannot be and more pages than were handed out; both leave everything as it was."""
    device, sequences, stride = _requests(lengths, keep, "keep", table, pool)
    if stream is not None:
        with _on(stream, device):
            return trim_step(lengths, keep, table, pool, page_size, out)
    i32 = torch.int32
    if out is None:
        out = Trimmed(*_empty(sequences + 1, dtype=i32, device=device).split_with_sizes((sequences, 1)))
    free, taken, status = pool._addresses
    args = _pack(_TRIM, lengths.data_ptr(), keep.data_ptr(), table.data_ptr(), free, taken, _at(out.lengths, i32, (sequences,), device, "out.lengths"),
                 _at(out.taken, i32, (1,), device, "out.taken"), status, sequences, table.shape[1], stride, pool.pages, page_size, 0)
    _status(_enqueue(_lib().gevva_step_trim, device, None, args), "trim_step")
    return out


def kv_append_at(q, k, v, cache, slots, positions, frequencies, q_weight=None, k_weight=None, normalize_v=False, eps=1e-6, packed=False, out=None,
                 stream=None):
    """kv_append at given places and with positions of several axes (time, height, width).  slots int32 [tokens] is page * page_size + slot in
    the page (StepPlan.slots); a row with one below zero is no token and is left as it was.  positions int32 is [tokens] or
    [axes, tokens] (the last dimension contiguous, axes as far apart as they like; up to 16), frequencies float64 [pairs] or [axes, pairs] to match: pair
    (j, pairs + j) turns by the sum of positions[a] * frequencies[a, j], so each pair has zeros for the axes that it does not follow.  The rest is as in
    kv_append, and `out` shares no memory with slots, positions, frequencies or weights either."""
    device, shape, q_rows = _queries(q)
    if stream is not None:
        with _on(stream, device):
            return kv_append_at(q, k, v, cache, slots, positions, frequencies, q_weight, k_weight, normalize_v, eps, packed, out)
    tokens, heads, dim = shape
    kv_heads = cache.kv_heads
    if cache.head_dim != dim or cache.device != device:
        raise ValueError(f"kv_append_at: queries of {dim} on {device}, cache of {cache.head_dim} on {cache.device}")
    k_rows, v_rows = _heads(k, "k", device, (tokens, kv_heads, dim)), _heads(v, "v", device, (tokens, kv_heads, dim))
    axes = positions.shape[0] if positions.dim() == 2 else 1
    if (positions.dtype is not torch.int32 or positions.device != device or positions.dim() not in (1, 2) or positions.shape[-1] != tokens or
            (tokens > 1 and positions.stride(-1) != 1) or not 1 <= axes <= 16):
        raise ValueError(f"positions: expected int32 ({tokens},) or (1 to 16 axes, {tokens}) on {device}, got {positions.dtype} "
                         f"{tuple(positions.shape)} strides {positions.stride()} on {positions.device}")
    pairs = 0
    if frequencies is not None:
        pairs = frequencies.shape[-1] if frequencies.dim() else 0
        if frequencies.dim() != positions.dim() and axes * pairs != frequencies.numel():
            raise ValueError(f"frequencies: expected ({axes} axes, pairs), got {tuple(frequencies.shape)}")
        _at(frequencies, torch.float64, (axes, pairs) if frequencies.dim() == 2 else (pairs,), device, "frequencies")
        if frequencies.numel() != axes * pairs:
            raise ValueError(f"frequencies: expected ({axes} axes, pairs), got {tuple(frequencies.shape)}")
    out = _out(out, q, device)
    k_out, v_out = (_out(None, k, device), _out(None, v, device)) if packed else (None, None)
    bf16 = torch.bfloat16
    args = _pack(_APPEND_AT, *q_rows, *k_rows, *v_rows, cache._address, _at(slots, torch.int32, (tokens,), device, "slots"), positions.data_ptr(),
                 positions.stride(0) if axes > 1 else 0, _address(frequencies) or 0, _at(q_weight, bf16, (dim,), device, "q_weight"),
                 _at(k_weight, bf16, (dim,), device, "k_weight"), out.data_ptr(), k_out.data_ptr() if packed else 0, v_out.data_ptr() if packed else 0,
                 cache.status.data_ptr(), tokens, heads, kv_heads, dim, 2 * pairs, axes, normalize_v, eps)
    _status(_enqueue(_lib().gevva_step_append, device, None, args), "kv_append_at")
    return Appended(out, k_out, v_out) if packed else out


def sample_tokens(logits, uniforms, temperature=None, top_k=None, top_p=None, min_p=None, softcap=0.0, probability=False, out=None, stream=None):
    """One token a row (int32 [rows]) from logits [rows, vocabulary], float32 or bfloat16, rows as far apart as they like (an expanded row too),
    by uniforms float32 [rows] in [0, 1).  A token's share is exp((y - y_max) / temperature), y the logit or, with a softcap,
    softcap * tanh(logit / softcap).  Tokens rank by logit, the lower index first among equals; kept are the first top_k, of those the ones in
    front of which less than top_p of the sum of shares has been, of those the ones with a share of at least min_p times the
    largest.  The row's token is the first of the vocabulary up to which the kept shares' sum exceeds its random number times the whole sum.
    temperature, top_p and min_p are float32 [rows], top_k int32 [rows], each None for none; a temperature that is not above zero
    takes the best token, a top_k of zero or less, a top_p of one or more and a min_p of zero or less keep all.  Minus infinity and NaN are never
    taken; a row of nothing else gives -1.  Shares are off by up to 2^-42.8 of themselves, with a softcap by 2^-50 of softcap / temperature more, and may
    be none below 2^-200 of the largest.  With `probability` also the token's share of the kept ones, float32 [rows].  `out` takes the
    tokens."""
    if logits.dim() != 2 or not logits.is_cuda or logits.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"logits: expected CUDA float32 or bfloat16 (rows, vocabulary), got {logits.dtype} {tuple(logits.shape)} on {logits.device}")
    device, (rows, vocabulary) = logits.device, logits.shape
    if stream is not None:
        with _on(stream, device):
            return sample_tokens(logits, uniforms, temperature, top_k, top_p, min_p, softcap, probability, out)
    if not 1 <= vocabulary <= MAX_VOCABULARY or (vocabulary > 1 and logits.stride(1) != 1):
        raise ValueError(f"logits: expected 1 to {MAX_VOCABULARY} contiguous values a row, got {tuple(logits.shape)} strides {logits.stride()}")
    f32, i32, each = torch.float32, torch.int32, (rows,)
    if out is None:
        out = _empty(rows, dtype=i32, device=device)
    shares = _empty(rows, dtype=f32, device=device) if probability else None
    args = _pack(_SAMPLE, logits.data_ptr(), logits.stride(0) if rows > 1 else 0, _at(uniforms, f32, each, device, "uniforms"),
                 _at(temperature, f32, each, device, "temperature"), _at(top_k, i32, each, device, "top_k"), _at(top_p, f32, each, device, "top_p"),
                 _at(min_p, f32, each, device, "min_p"), _at(out, i32, each, device, "out"), shares.data_ptr() if probability else 0, rows,
                 vocabulary, logits.dtype is f32, softcap)
    _status(_enqueue(_lib().gevva_step_sample, device, None, args), "sample_tokens")
    return (out, shares) if probability else out


@dataclass
class TokenHead:
    """What stands behind the last layer: norm, the product with the vocabulary's rows (a library's, torch.mm) and the token of each row.  The
    reference caps these logits at 30 (src/cuda/runtime/decision_logits.cuh)."""
    norm: torch.Tensor           # bf16 [hidden]
    rows: torch.Tensor           # bf16 [vocabulary, hidden]
    softcap: float = 30.0
    eps: float = 1e-6

    def logits(self, hidden):
        """bf16 [tokens, vocabulary], not capped yet."""
        return torch.mm(block_norm(hidden, self.norm, self.eps), self.rows.t())

    def forward(self, hidden, uniforms, temperature=None, top_k=None, top_p=None, min_p=None, probability=False, out=None):
        """A token for each row of `hidden` [tokens, hidden], by sample_tokens."""
        return sample_tokens(self.logits(hidden), uniforms, temperature, top_k, top_p, min_p, self.softcap, probability, out)
