// C ABI of the attention side of a decoder layer (declared in include/gevva_moe.h): what a call may be, and what it launches.
#include <cuda_runtime.h>
#include <math.h>

#include "../../include/gevva_moe.h"
#include "gv_attention.h"
#include "gv_launchers.h"

namespace {

constexpr int kMaxPositions = 1 << 30;
constexpr int kMaxGroup = 128;

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

bool pages_ok(gv::AttnPages* out, const gevva_attn_cache* c, const gevva_attn_batch* b, int kv_heads, int dim) {
  if (!c || !b || !aligned(c->keys) || !aligned(c->values) || c->pages < 1 || c->page_size < 16 || (c->page_size & (c->page_size - 1)) ||
      !b->token_offsets || !b->lengths || !b->table || b->sequences < 1 || b->table_width < 1 || b->table_stride < b->table_width ||
      static_cast<long long>(b->table_width) * c->page_size > kMaxPositions)
    return false;
  *out = gv::AttnPages{c->keys,           c->values,            c->key_page_stride,   c->key_slot_stride, c->key_head_stride,
                       c->value_page_stride, c->value_slot_stride, c->value_head_stride, c->pages,           c->page_size,
                       b->lengths,        b->table,             b->table_width,       b->table_stride};
  const long long whole = static_cast<long long>(c->page_size) * kv_heads * dim;
  return stride_ok(out->key_head_stride, kv_heads, dim) && stride_ok(out->value_head_stride, kv_heads, dim) &&
         stride_ok(out->key_slot_stride, c->page_size, dim) && stride_ok(out->value_slot_stride, c->page_size, dim) &&
         stride_ok(out->key_page_stride, c->pages, whole) && stride_ok(out->value_page_stride, c->pages, whole);
}

int launched(cudaError_t e) {
  if (e == cudaSuccess) return GEVVA_MOE_OK;
  cudaGetLastError();  // reported here; not again by the next call
  return e == cudaErrorInvalidValue ? GEVVA_MOE_BAD_ARGUMENT : GEVVA_MOE_CUDA_ERROR;
}

bool attention_ok(float scale, int window) { return scale > 0.0f && scale <= 1e30f && window >= 0; }

}  // namespace

extern "C" {

int gevva_attn_norm(const void* x, const void* weight, void* out, int rows, int width, float eps, gevva_stream_t stream) {
  if (rows < 0 || !aligned_for(x, rows) || !aligned(weight) || !aligned_for(out, rows) || width < 8 || width > 32768 || width % 8 || !(eps >= 0.0f))
    return GEVVA_MOE_BAD_ARGUMENT;
  if (rows == 0) return GEVVA_MOE_OK;
  gv::BlockNormCall call{};
  call.x = x;
  call.weight = weight;
  call.out = out;
  call.rows = rows;
  call.width = width;
  call.eps = eps;
  return launched(gv::launch_block_norm(call, gv::current_sm_count(), stream));
}

int gevva_attn_norm_add(const void* x, const void* weight, const void* residual, const void* gate, const void* scale,
                        const void* next_weight, void* out, void* next, int rows, int width, float eps, gevva_stream_t stream) {
  if (rows < 0 || !aligned_for(x, rows) || !aligned(weight) || !aligned_for(residual, rows) || !aligned_or_null(gate) || (reinterpret_cast<uintptr_t>(scale) & 1) ||
      !aligned_or_null(next_weight) || !aligned_for(out, rows) || !aligned_or_null(next) || (rows > 0 && !next_weight != !next) || width < 8 ||
      width > 32768 || width % 8 || !(eps >= 0.0f))
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
  return launched(gv::launch_block_norm(call, gv::current_sm_count(), stream));
}

int gevva_attn_append(const void* q, long long q_token_stride, long long q_head_stride,
                      const void* k, long long k_token_stride, long long k_head_stride,
                      const void* v, long long v_token_stride, long long v_head_stride,
                      const gevva_attn_cache* cache,
                      const gevva_attn_batch* batch, int tokens, int heads, int kv_heads, int dim, const double* frequencies,
                      int rotated, const void* q_weight, const void* k_weight, int normalize_v, float eps, void* q_out, void* k_out,
                      void* v_out, int* device_status, gevva_stream_t stream) {
  gv::AppendCall call{};
  if (!heads_ok(tokens, heads, kv_heads, dim) || !rows_ok(&call.q, q, q_token_stride, q_head_stride, tokens, heads, dim) || !rows_ok(&call.k, k, k_token_stride, k_head_stride, tokens, kv_heads, dim) ||
      !rows_ok(&call.v, v, v_token_stride, v_head_stride, tokens, kv_heads, dim) || !pages_ok(&call.pages, cache, batch, kv_heads, dim) || rotated < 0 || rotated > dim ||
      rotated % 16 || (rotated > 0 && (!frequencies || (reinterpret_cast<uintptr_t>(frequencies) & 7))) || !aligned_or_null(q_weight) ||
      !aligned_or_null(k_weight) || !(eps >= 0.0f) || !aligned_for(q_out, tokens) || !aligned_or_null(k_out) || !aligned_or_null(v_out) || (tokens > 0 && !k_out != !v_out))
    return GEVVA_MOE_BAD_ARGUMENT;
  if (tokens == 0) return GEVVA_MOE_OK;
  call.token_offsets = batch->token_offsets;
  call.sequences = batch->sequences;
  call.tokens = tokens;
  call.heads = heads;
  call.kv_heads = kv_heads;
  call.dim = dim;
  call.frequencies = frequencies;
  call.rotated = rotated;
  call.q_weight = q_weight;
  call.k_weight = k_weight;
  call.normalize_v = normalize_v != 0;
  call.eps = eps;
  call.q_out = q_out;
  call.k_out = k_out;
  call.v_out = v_out;
  call.status = device_status;
  return launched(gv::launch_kv_append(call, gv::current_sm_count(), stream));
}

int gevva_attn_prompt(const void* q, long long q_token_stride, long long q_head_stride,
                      const void* k, long long k_token_stride, long long k_head_stride,
                      const void* v, long long v_token_stride, long long v_head_stride,
                      const int* token_offsets,
                      int sequences, int tokens, int heads, int kv_heads, int dim, float scale, int window, void* out,
                      int* device_status, gevva_stream_t stream) {
  gv::AttnCall call{};
  if (!heads_ok(tokens, heads, kv_heads, dim) || !rows_ok(&call.q, q, q_token_stride, q_head_stride, tokens, heads, dim) || !rows_ok(&call.k, k, k_token_stride, k_head_stride, tokens, kv_heads, dim) ||
      !rows_ok(&call.v, v, v_token_stride, v_head_stride, tokens, kv_heads, dim) || !token_offsets || sequences < 1 || tokens > kMaxPositions || !attention_ok(scale, window) ||
      !aligned_32(out, tokens))
    return GEVVA_MOE_BAD_ARGUMENT;
  if (tokens == 0) return GEVVA_MOE_OK;
  call.token_offsets = token_offsets;
  call.sequences = sequences;
  call.tokens = tokens;
  call.heads = heads;
  call.kv_heads = kv_heads;
  call.dim = dim;
  call.window = window < kMaxPositions ? window : 0;  // (a window that no sequence is longer than)
  call.scale = scale;
  call.out = out;
  call.out_token_stride = static_cast<long long>(heads) * dim;
  call.out_head_stride = dim;
  call.status = device_status;
  call.sm_count = gv::current_sm_count();
  return launched(gv::launch_attention(call, stream));
}

size_t gevva_attn_chunk_workspace_bytes(int dim) {
  return dim == 64 || dim == 128 || dim == 256 || dim == 512 ? gv::attention_workspace_bytes(dim, gv::current_sm_count()) : 0;
}

int gevva_attn_chunk(const void* q, long long q_token_stride, long long q_head_stride,
                     const gevva_attn_cache* cache, const gevva_attn_batch* batch, int tokens, int heads,
                     int kv_heads, int dim, float scale, int window, void* out, void* workspace, int* device_status,
                     gevva_stream_t stream) {
  gv::AttnCall call{};
  if (!heads_ok(tokens, heads, kv_heads, dim) || !rows_ok(&call.q, q, q_token_stride, q_head_stride, tokens, heads, dim) || !pages_ok(&call.pages, cache, batch, kv_heads, dim) ||
      tokens > kMaxPositions || !attention_ok(scale, window) || !aligned_32(out, tokens) || !workspace || !aligned_32(workspace, 1))
    return GEVVA_MOE_BAD_ARGUMENT;
  if (tokens == 0) return GEVVA_MOE_OK;
  call.paged = true;
  call.token_offsets = batch->token_offsets;
  call.sequences = batch->sequences;
  call.tokens = tokens;
  call.heads = heads;
  call.kv_heads = kv_heads;
  call.dim = dim;
  call.window = window < kMaxPositions ? window : 0;
  call.scale = scale;
  call.out = out;
  call.out_token_stride = static_cast<long long>(heads) * dim;
  call.out_head_stride = dim;
  call.workspace = workspace;
  call.status = device_status;
  call.sm_count = gv::current_sm_count();
  if (call.sm_count < 1) return GEVVA_MOE_NO_DEVICE;
  return launched(gv::launch_attention(call, stream));
}

}  // extern "C"
