// Launchers of the attention kernels (attention.cu) and of the row kernels around them (attention_rows.cu).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace gv {

// Queries or packed keys: bf16 [tokens, heads, dim], strides in elements.
struct AttnRows {
  const void* data;
  long long token_stride, head_stride;
};

// Cache side of a paged call: bf16 [pages, page_size, kv_heads, dim] for keys and for values, strides in elements.
struct AttnPages {
  void* keys;
  void* values;
  long long key_page_stride, key_slot_stride, key_head_stride;
  long long value_page_stride, value_slot_stride, value_head_stride;
  int page_count, page_size;
  const int* lengths;  // [sequences]
  const int* table;    // [sequences, table_stride], the first table_width of each row in use
  int table_width, table_stride;
};

struct AttnCall {
  AttnRows q, k, v;            // k, v: prompt form only
  AttnPages pages;             // paged form only
  bool paged;
  const int* token_offsets;    // [sequences + 1]
  int sequences;
  int tokens;                  // rows of q
  int heads, kv_heads, dim;
  int window;                  // 0: none
  float scale;
  void* out;                   // bf16 [tokens, heads, dim]
  long long out_token_stride, out_head_stride;
  void* workspace;             // paged form: attention_workspace_bytes
  int* status;                 // optional
  int sm_count;
};

size_t attention_workspace_bytes(int dim, int sm_count);
cudaError_t launch_attention(const AttnCall& call, cudaStream_t stream);

struct AppendCall {
  AttnRows q, k, v;
  AttnPages pages;
  const int* token_offsets;
  int sequences, tokens, heads, kv_heads, dim;
  const double* frequencies;   // [rotated / 2]
  int rotated;
  const void* q_weight;        // optional bf16 [dim]
  const void* k_weight;
  bool normalize_v;
  float eps;
  void* q_out;                 // bf16 [tokens, heads, dim]
  void* k_out;                 // optional bf16 [tokens, kv_heads, dim], both or none
  void* v_out;
  int* status;
};
cudaError_t launch_kv_append(const AppendCall& call, int sm_count, cudaStream_t stream);

// out = rms_norm(x) * weight, or (residual + gate * rms_norm(x) * weight) * scale where there is a residual; next = rms_norm(out) *
// next_weight of the values before their rounding.
struct BlockNormCall {
  const void* x;
  const void* weight;
  const void* residual;     // optional
  const void* gate;         // optional
  const void* scale;        // optional
  const void* next_weight;  // optional, with next
  void* out;
  void* next;
  int rows, width;
  float eps;
};
cudaError_t launch_block_norm(const BlockNormCall& call, int sm_count, cudaStream_t stream);

}  // namespace gv
