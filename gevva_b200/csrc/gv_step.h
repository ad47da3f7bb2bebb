// Launchers of what a serving step has around its layers: pages and slots (step_pages.cu), the append at given slots
// (attention_rows.cu), tokens from logits (sample.cu).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>

#include "gv_attention.h"

namespace gv {

// Requests and the pool that their pages come from; counts as the call finds them, the outputs may be the same memory.
struct PagesCall {
  const int* lengths;   // [sequences]
  const int* counts;    // [sequences]: new tokens (plan), tokens that stay (trim)
  const int* shift;     // plan, optional [sequences]
  int* table;           // [sequences, table_stride], the first table_width of each row in use
  int* pool;            // [pool_pages]: pages, of which the first `taken` are handed out
  const int* taken;     // [1]
  int sequences, table_width, table_stride, pool_pages, page_size;
  int tokens;           // plan: rows of slots and positions
  int* offsets_out;     // plan [sequences + 1]
  int* lengths_out;     // [sequences]
  int* slots;           // plan [tokens]
  int* positions;       // plan [tokens]
  int* taken_out;       // [1]
  int* status;
  bool trim;
};
constexpr int kMaxPlanSequences = 16384;
cudaError_t launch_step_pages(const PagesCall& call, cudaStream_t stream);

// kv_append at given places: slots[token] = page * page_size + slot in the page, below zero for a row that is no token;
// pair j turns by the sum over the axes of positions[axis * position_stride + token] * frequencies[axis * rotated / 2 + j].
struct PlacedCall {
  AppendCall rows;           // its token_offsets, sequences, lengths and table are not read
  const int* slots;          // [tokens]
  const int* positions;      // [axes, tokens], position_stride apart
  long long position_stride;
  int axes;
};
cudaError_t launch_kv_append_placed(const PlacedCall& call, int sm_count, cudaStream_t stream);

struct SampleCall {
  const void* logits;        // [rows, vocabulary], row_stride values apart
  long long row_stride;
  bool wide;                 // f32; else bf16
  const float* uniforms;     // [rows]
  const float* temperature;  // the rest optional, [rows]
  const int* top_k;
  const float* top_p;
  const float* min_p;
  float softcap;             // 0: none
  int rows, vocabulary;
  int* tokens;               // [rows]
  float* probabilities;      // optional [rows]
};
constexpr int kMaxVocabulary = 1 << 19;
cudaError_t launch_sample(const SampleCall& call, int sm_count, cudaStream_t stream);

}  // namespace gv
