// C ABI of the attention side of a decoder layer (declared in include/gevva_moe.h): what a call may be, and what it launches.
#include <cuda_runtime.h>
#include <math.h>

#include <atomic>
#include <initializer_list>

#include "../../include/gevva_moe.h"
#include "gv_attention.h"
#include "gv_launchers.h"
#include "gv_step.h"

namespace gv {

int launched(cudaError_t e) {
  if (e == cudaSuccess) return GEVVA_MOE_OK;
  cudaGetLastError();  // reported here; not again by the next call
  if (e == cudaErrorInvalidConfiguration) return GEVVA_MOE_TOO_LARGE;  // (more items than a grid has)
  return e == cudaErrorInvalidValue ? GEVVA_MOE_BAD_ARGUMENT : GEVVA_MOE_CUDA_ERROR;
}

bool touch(const void* a, long long a_bytes, const void* b, long long b_bytes) {
  const intptr_t x = reinterpret_cast<intptr_t>(a), y = reinterpret_cast<intptr_t>(b);
  return a && b && x < y + b_bytes && y < x + a_bytes;
}

// What calls without a status word of their own report into, one of each device.  (In host code the name is only a handle.)
static __device__ int g_attention_status;
constexpr int kMaxDevices = 64;
static std::atomic<int*> g_status_address[kMaxDevices];

// The call's word, or else the current device's.
cudaError_t status_word(int* own, int** out) {
  *out = own;
  if (own) return cudaSuccess;
  int device = -1;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  if (device < 0 || device >= kMaxDevices) return cudaErrorInvalidDevice;
  *out = g_status_address[device].load(std::memory_order_relaxed);
  if (*out) return cudaSuccess;
  e = cudaGetSymbolAddress(reinterpret_cast<void**>(out), g_attention_status);
  if (e == cudaSuccess) g_status_address[device].store(*out, std::memory_order_relaxed);
  return e;
}

}  // namespace gv

namespace {

constexpr int kMaxPositions = 1 << 30;
constexpr int kMaxGroup = 128;

using gv::launched;
using gv::status_word;
using gv::touch;

bool aligned(const void* p) { return p && (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool aligned_or_null(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// (attention stores 32 bytes at a time)
bool aligned_32(const void* p, int rows) { return (rows == 0 || p) && (reinterpret_cast<uintptr_t>(p) & 31) == 0; }
// Rows of a call without any may be nowhere.
bool aligned_for(const void* p, int rows) { return rows > 0 ? aligned(p) : aligned_or_null(p); }

// A stride of a dimension of `extent`: one that is never taken may be anything.
bool stride_ok(long long& stride, int extent, long long otherwise) {
  if (extent <= 1) {
    stride = otherwise;
    return true;
  }
  return stride > 0 && (stride & 7) == 0 && stride < (1ll << 38);
}

bool heads_ok(int tokens, int heads, int kv_heads, int dim) {
  return tokens >= 0 && heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && heads / kv_heads <= kMaxGroup && heads <= 65536 &&
         (dim == 64 || dim == 128 || dim == 256 || dim == 512);
}

bool rows_ok(gv::AttnRows* out, const void* data, long long token_stride, long long head_stride, int tokens, int heads, int dim) {
  if (!aligned_for(data, tokens)) return false;
  *out = gv::AttnRows{data, token_stride, head_stride};
  return stride_ok(out->head_stride, heads, dim) && stride_ok(out->token_stride, tokens, static_cast<long long>(heads) * dim);
}

// Whether `count` values at `out` share memory with these rows; what lies between the rows and between their heads is not theirs.
bool meets(const void* out, long long count, const gv::AttnRows& rows, int tokens, int heads, int dim) {
  long long at = static_cast<long long>(reinterpret_cast<intptr_t>(out) - reinterpret_cast<intptr_t>(rows.data)) / 2;  // (both are aligned)
  const bool token_outer = rows.token_stride >= rows.head_stride;
  const long long strides[2] = {token_outer ? rows.token_stride : rows.head_stride, token_outer ? rows.head_stride : rows.token_stride};
  const long long extents[2] = {token_outer ? tokens : heads, token_outer ? heads : tokens};
  for (int i = 0; i < 2; ++i) {
    const long long piece = i == 0 ? (extents[1] - 1) * strides[1] + dim : dim;  // from the first value to behind the last of what one step holds
    if (at + count <= 0) return false;
    if (at <= 0) return true;
    if (piece >= strides[i]) return at < (extents[i] - 1) * strides[i] + piece;
    const long long step = at / strides[i];
    if (step >= extents[i]) return false;
    if (step + 1 < extents[i] && at + count > (step + 1) * strides[i]) return true;
    at -= step * strides[i];
  }
  return at < dim;
}

// A row is written when it has been read, not when others have: an output is an input, row for row, or lies apart from it, and apart from the vectors.
bool norm_apart(const void* out, const gv::BlockNormCall& call) {
  const long long vector = 2ll * call.width, rows = call.rows * vector;
  for (const void* in : {call.x, call.residual})
    if (in != out && touch(out, rows, in, rows)) return false;
  for (const void* in : {call.weight, call.gate, call.next_weight})
    if (touch(out, rows, in, vector)) return false;
  return !touch(out, rows, call.scale, 2);
}

bool packed(const gv::AttnRows& rows, int heads, int dim) {
  return rows.head_stride == dim && rows.token_stride == static_cast<long long>(heads) * dim;
}

bool ints(const void* p) { return p && (reinterpret_cast<uintptr_t>(p) & 3) == 0; }

bool cache_ok(gv::AttnPages* out, const gevva_attn_cache* c, int kv_heads, int dim) {
  if (!c || !aligned(c->keys) || !aligned(c->values) || c->pages < 1 || c->page_size < 16 || (c->page_size & (c->page_size - 1))) return false;
  *out = gv::AttnPages{c->keys,           c->values,            c->key_page_stride,   c->key_slot_stride, c->key_head_stride,
                       c->value_page_stride, c->value_slot_stride, c->value_head_stride, c->pages,           c->page_size,
                       nullptr,           nullptr,              0,                    0};
  const long long whole = static_cast<long long>(c->page_size) * kv_heads * dim;
  return stride_ok(out->key_head_stride, kv_heads, dim) && stride_ok(out->value_head_stride, kv_heads, dim) &&
         stride_ok(out->key_slot_stride, c->page_size, dim) && stride_ok(out->value_slot_stride, c->page_size, dim) &&
         stride_ok(out->key_page_stride, c->pages, whole) && stride_ok(out->value_page_stride, c->pages, whole);
}

bool pages_ok(gv::AttnPages* out, const gevva_attn_cache* c, const gevva_attn_batch* b, int kv_heads, int dim) {
  if (!cache_ok(out, c, kv_heads, dim) || !b || !b->token_offsets || !b->lengths || !b->table || b->sequences < 1 || b->table_width < 1 ||
      b->table_stride < b->table_width || static_cast<long long>(b->table_width) * c->page_size > kMaxPositions)
    return false;
  out->lengths = b->lengths;
  out->table = b->table;
  out->table_width = b->table_width;
  out->table_stride = b->table_stride;
  return true;
}

// What both forms of the append have; the places of the tokens are the caller's to fill.
template <class Args>
bool fill_append(gv::AppendCall* call, const Args& a) {
  if (!heads_ok(a.tokens, a.heads, a.kv_heads, a.dim) ||
      !rows_ok(&call->q, a.q, a.q_token_stride, a.q_head_stride, a.tokens, a.heads, a.dim) ||
      !rows_ok(&call->k, a.k, a.k_token_stride, a.k_head_stride, a.tokens, a.kv_heads, a.dim) ||
      !rows_ok(&call->v, a.v, a.v_token_stride, a.v_head_stride, a.tokens, a.kv_heads, a.dim) || a.rotated < 0 || a.rotated > a.dim ||
      a.rotated % 16 || (a.rotated > 0 && (!a.frequencies || (reinterpret_cast<uintptr_t>(a.frequencies) & 7))) ||
      !aligned_or_null(a.q_weight) || !aligned_or_null(a.k_weight) || !(a.eps >= 0.0f) || !aligned_for(a.q_out, a.tokens) ||
      !aligned_or_null(a.k_out) || !aligned_or_null(a.v_out) || (a.tokens > 0 && !a.k_out != !a.v_out))
    return false;
  // A token's rows are written when that token's have been read, not when others' have: an output may stand where its own input does,
  // row for row, and nowhere else among the inputs.
  const gv::AttnRows* const inputs[3] = {&call->q, &call->k, &call->v};
  void* const outputs[3] = {a.q_out, a.k_out, a.v_out};
  for (int o = 0; o < 3 && a.tokens > 0; ++o) {
    const auto heads = [&](int i) { return i == 0 ? a.heads : a.kv_heads; };
    for (int i = 0; i < 3 && outputs[o]; ++i) {
      if (o == i && outputs[o] == inputs[i]->data && packed(*inputs[i], heads(i), a.dim)) continue;
      if (meets(outputs[o], static_cast<long long>(a.tokens) * heads(o) * a.dim, *inputs[i], a.tokens, heads(i), a.dim)) return false;
    }
  }
  call->tokens = a.tokens;
  call->heads = a.heads;
  call->kv_heads = a.kv_heads;
  call->dim = a.dim;
  call->frequencies = a.frequencies;
  call->rotated = a.rotated;
  call->q_weight = a.q_weight;
  call->k_weight = a.k_weight;
  call->normalize_v = a.normalize_v != 0;
  call->eps = a.eps;
  call->q_out = a.q_out;
  call->k_out = a.k_out;
  call->v_out = a.v_out;
  return true;
}

bool attention_ok(int tokens, float scale, int window) {
  return tokens <= kMaxPositions && scale > 0.0f && scale <= 1e30f && window >= 0;
}

// What both attention calls have.
template <class Args>
void fill_attention(gv::AttnCall* call, const Args& a) {
  call->tokens = a.tokens;
  call->heads = a.heads;
  call->kv_heads = a.kv_heads;
  call->dim = a.dim;
  call->window = a.window < kMaxPositions ? a.window : 0;  // (a window that no sequence is longer than)
  call->scale = a.scale;
  call->out = a.out;
  call->out_token_stride = static_cast<long long>(a.heads) * a.dim;
  call->out_head_stride = a.dim;
  call->sm_count = gv::current_sm_count();
}

}  // namespace

extern "C" {

int gevva_attn_norm(const void* x, const void* weight, void* out, int rows, int width, float eps, gevva_stream_t stream) {
  if (rows < 0 || !aligned_for(x, rows) || !aligned(weight) || !aligned_for(out, rows) || width < 8 || width > 32768 || width % 8 ||
      !(eps >= 0.0f))
    return GEVVA_MOE_BAD_ARGUMENT;
  if (rows == 0) return GEVVA_MOE_OK;
  gv::BlockNormCall call{};
  call.x = x;
  call.weight = weight;
  call.out = out;
  call.rows = rows;
  call.width = width;
  call.eps = eps;
  if (!norm_apart(out, call)) return GEVVA_MOE_BAD_ARGUMENT;
  return launched(gv::launch_block_norm(call, gv::current_sm_count(), stream));
}

int gevva_attn_norm_add(const void* x, const void* weight, const void* residual, const void* gate, const void* scale,
                        const void* next_weight, void* out, void* next, int rows, int width, float eps, gevva_stream_t stream) {
  if (rows < 0 || !aligned_for(x, rows) || !aligned(weight) || !aligned_for(residual, rows) || !aligned_or_null(gate) ||
      (reinterpret_cast<uintptr_t>(scale) & 1) || !aligned_or_null(next_weight) || !aligned_for(out, rows) || !aligned_or_null(next) ||
      (rows > 0 && !next_weight != !next) || width < 8 || width > 32768 || width % 8 || !(eps >= 0.0f))
    return GEVVA_MOE_BAD_ARGUMENT;
  if (rows == 0) return GEVVA_MOE_OK;
  gv::BlockNormCall call{};
  call.x = x;
  call.weight = weight;
  call.residual = residual;
  call.gate = gate;
  call.scale = scale;
  call.next_weight = next_weight;
  call.out = out;
  call.next = next;
  call.rows = rows;
  call.width = width;
  call.eps = eps;
  if (!norm_apart(out, call) || !norm_apart(next, call) || touch(out, 2ll * rows * width, next, 2ll * rows * width)) return GEVVA_MOE_BAD_ARGUMENT;
  return launched(gv::launch_block_norm(call, gv::current_sm_count(), stream));
}

int gevva_attn_append(const gevva_attn_append_args* a, gevva_stream_t stream) {
  gv::AppendCall call{};
  if (!a || !fill_append(&call, *a) || !pages_ok(&call.pages, a->cache, a->batch, a->kv_heads, a->dim) || a->reserved) return GEVVA_MOE_BAD_ARGUMENT;
  if (a->tokens == 0) return GEVVA_MOE_OK;
  call.token_offsets = a->batch->token_offsets;
  call.sequences = a->batch->sequences;
  const cudaError_t e = status_word(a->device_status, &call.status);
  if (e != cudaSuccess) return launched(e);
  return launched(gv::launch_kv_append(call, gv::current_sm_count(), stream));
}

int gevva_step_append(const gevva_step_append_args* a, gevva_stream_t stream) {
  gv::PlacedCall call{};
  if (!a || !fill_append(&call.rows, *a) || !cache_ok(&call.rows.pages, a->cache, a->kv_heads, a->dim) || a->axes < 1 || a->axes > 16 ||
      (a->tokens > 0 && (!ints(a->slots) || !ints(a->positions))) || (a->axes > 1 && (a->position_stride < 0 || a->position_stride >= 1ll << 38)))
    return GEVVA_MOE_BAD_ARGUMENT;
  // (a slot is a whole number of 32 bits)
  if (static_cast<long long>(a->cache->pages) * a->cache->page_size > 1ll << 31) return GEVVA_MOE_TOO_LARGE;
  if (a->tokens == 0) return GEVVA_MOE_OK;
  // A token's place is read when others' rows have been written.
  const long long tokens = a->tokens, stride = a->axes > 1 ? a->position_stride : 0;
  for (int o = 0; o < 3; ++o) {
    void* const out = o == 0 ? a->q_out : o == 1 ? a->k_out : a->v_out;
    const long long bytes = 2 * tokens * (o == 0 ? a->heads : a->kv_heads) * a->dim;
    if (touch(out, bytes, a->slots, 4 * tokens) || touch(out, bytes, a->positions, 4 * ((a->axes - 1) * stride + tokens)) ||
        (a->rotated > 0 && touch(out, bytes, a->frequencies, 4ll * a->axes * a->rotated)) || touch(out, bytes, a->q_weight, 2ll * a->dim) ||
        touch(out, bytes, a->k_weight, 2ll * a->dim))
      return GEVVA_MOE_BAD_ARGUMENT;
  }
  call.slots = a->slots;
  call.positions = a->positions;
  call.position_stride = stride;
  call.axes = a->axes;
  const cudaError_t e = status_word(a->device_status, &call.rows.status);
  if (e != cudaSuccess) return launched(e);
  return launched(gv::launch_kv_append_placed(call, gv::current_sm_count(), stream));
}

int gevva_attn_prompt(const gevva_attn_prompt_args* a, gevva_stream_t stream) {
  gv::AttnCall call{};
  if (!a || !heads_ok(a->tokens, a->heads, a->kv_heads, a->dim) ||
      !rows_ok(&call.q, a->q, a->q_token_stride, a->q_head_stride, a->tokens, a->heads, a->dim) ||
      !rows_ok(&call.k, a->k, a->k_token_stride, a->k_head_stride, a->tokens, a->kv_heads, a->dim) ||
      !rows_ok(&call.v, a->v, a->v_token_stride, a->v_head_stride, a->tokens, a->kv_heads, a->dim) || !a->token_offsets ||
      a->sequences < 1 ||
      !attention_ok(a->tokens, a->scale, a->window) || !aligned_32(a->out, a->tokens) || a->reserved)
    return GEVVA_MOE_BAD_ARGUMENT;
  if (a->tokens == 0) return GEVVA_MOE_OK;
  const long long values = static_cast<long long>(a->tokens) * a->heads * a->dim;
  if (meets(a->out, values, call.q, a->tokens, a->heads, a->dim) || meets(a->out, values, call.k, a->tokens, a->kv_heads, a->dim) ||
      meets(a->out, values, call.v, a->tokens, a->kv_heads, a->dim))
    return GEVVA_MOE_BAD_ARGUMENT;
  call.token_offsets = a->token_offsets;
  call.sequences = a->sequences;
  fill_attention(&call, *a);
  const cudaError_t e = status_word(a->device_status, &call.status);
  if (e != cudaSuccess) return launched(e);
  return launched(gv::launch_attention(call, stream));
}

size_t gevva_attn_chunk_workspace_bytes(int dim) {
  return dim == 64 || dim == 128 || dim == 256 || dim == 512 ? gv::attention_workspace_bytes(dim, gv::current_sm_count()) : 0;
}

int gevva_attn_chunk(const gevva_attn_chunk_args* a, gevva_stream_t stream) {
  gv::AttnCall call{};
  if (!a || !heads_ok(a->tokens, a->heads, a->kv_heads, a->dim) ||
      !rows_ok(&call.q, a->q, a->q_token_stride, a->q_head_stride, a->tokens, a->heads, a->dim) ||
      !pages_ok(&call.pages, a->cache, a->batch, a->kv_heads, a->dim) || !attention_ok(a->tokens, a->scale, a->window) ||
      !aligned_32(a->out, a->tokens) || !aligned_32(a->workspace, 1))
    return GEVVA_MOE_BAD_ARGUMENT;
  if (a->tokens == 0) return GEVVA_MOE_OK;
  if (meets(a->out, static_cast<long long>(a->tokens) * a->heads * a->dim, call.q, a->tokens, a->heads, a->dim)) return GEVVA_MOE_BAD_ARGUMENT;
  call.paged = true;
  call.token_offsets = a->batch->token_offsets;
  call.sequences = a->batch->sequences;
  call.workspace = a->workspace;
  fill_attention(&call, *a);
  if (call.sm_count < 1) return GEVVA_MOE_NO_DEVICE;
  const cudaError_t e = status_word(a->device_status, &call.status);
  if (e != cudaSuccess) return launched(e);
  return launched(gv::launch_attention(call, stream));
}

int gevva_attention_last_status(void) {
  int* word = nullptr;
  int status = 0;
  cudaError_t e = status_word(nullptr, &word);
  if (e == cudaSuccess) e = cudaDeviceSynchronize();
  if (e == cudaSuccess) e = cudaMemcpy(&status, word, sizeof(int), cudaMemcpyDeviceToHost);
  if (e == cudaSuccess && status != 0) e = cudaMemset(word, 0, sizeof(int));
  return e == cudaSuccess ? -status : launched(e);
}

}  // extern "C"
