// C ABI of what a serving step has around its layers (declared in include/gevva_moe.h): what a call may be, and what it launches.  (Its
// append stands beside the other one, in attention_abi.cu.)
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/gevva_moe.h"
#include "gv_launchers.h"
#include "gv_step.h"

namespace {

constexpr long long kMaxPositions = 1ll << 30;

// Memory that a call reads or writes; none of nothing.
struct Range {
  const void* at;
  long long bytes;
};
bool meet(const Range& a, const Range& b) { return gv::touch(a.at, a.bytes, b.at, b.bytes); }
Range words(const int* p, long long count) { return {p, 4 * count}; }

// Whether no output shares memory with another one or with what is read.
template <int kRead, int kWritten>
bool apart(const Range (&read)[kRead], const Range (&written)[kWritten]) {
  for (int i = 0; i < kWritten; ++i) {
    for (int j = 0; j < kRead; ++j)
      if (meet(written[i], read[j])) return false;
    for (int j = 0; j < i; ++j)
      if (meet(written[i], written[j])) return false;
  }
  return true;
}

bool aligned_to(const void* p, int bytes) { return p && reinterpret_cast<uintptr_t>(p) % bytes == 0; }
bool aligned_or_null(const void* p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// What both calls over the pool have.
template <class Args>
bool fill_pages(gv::PagesCall* call, const Args& a) {
  if (!aligned_to(a.lengths, 4) || !aligned_to(a.table, 4) || !aligned_to(a.pool, 4) || !aligned_to(a.taken, 4) || !aligned_to(a.lengths_out, 4) ||
      !aligned_to(a.taken_out, 4))
    return false;
  if (a.sequences < 1 || a.table_width < 1 || a.table_stride < a.table_width || a.pool_pages < 1 || a.page_size < 16 ||
      (a.page_size & (a.page_size - 1)) || static_cast<long long>(a.table_width) * a.page_size > kMaxPositions)
    return false;
  call->lengths = a.lengths;
  call->table = const_cast<int*>(a.table);
  call->pool = const_cast<int*>(a.pool);
  call->taken = a.taken;
  call->sequences = a.sequences;
  call->table_width = a.table_width;
  call->table_stride = a.table_stride;
  call->pool_pages = a.pool_pages;
  call->page_size = a.page_size;
  call->lengths_out = a.lengths_out;
  call->taken_out = a.taken_out;
  return true;
}
template <class Args>
Range table_of(const Args& a) {
  return words(a.table, static_cast<long long>(a.sequences - 1) * a.table_stride + a.table_width);
}
// An input that the output may be, whole: then it is none that the output has to be apart from.
Range unless(const int* in, const int* out, long long count) { return in == out ? Range{nullptr, 0} : words(in, count); }

int launch_pages(gv::PagesCall& call, int* device_status, gevva_stream_t stream) {
  if (call.sequences > gv::kMaxPlanSequences) return GEVVA_MOE_TOO_LARGE;
  const cudaError_t e = gv::status_word(device_status, &call.status);
  return gv::launched(e != cudaSuccess ? e : gv::launch_step_pages(call, stream));
}

}  // namespace

extern "C" {

int gevva_step_plan(const gevva_step_plan_args* a, gevva_stream_t stream) {
  gv::PagesCall call{};
  if (!a || !fill_pages(&call, *a) || !aligned_to(a->news, 4) || !aligned_or_null(a->shift, 4) || !aligned_to(a->token_offsets, 4) ||
      a->tokens < 0 || a->tokens > kMaxPositions || (a->tokens > 0 && (!aligned_to(a->slots, 4) || !aligned_to(a->positions, 4))))
    return GEVVA_MOE_BAD_ARGUMENT;
  const long long n = a->sequences;
  const Range read[] = {unless(a->lengths, a->lengths_out, n), words(a->news, n), words(a->shift, n), words(a->pool, a->pool_pages),
                        unless(a->taken, a->taken_out, 1)};
  const Range written[] = {table_of(*a), words(a->token_offsets, n + 1), words(a->lengths_out, n), words(a->slots, a->tokens),
                           words(a->positions, a->tokens), words(a->taken_out, 1)};
  if (!apart(read, written)) return GEVVA_MOE_BAD_ARGUMENT;
  call.counts = a->news;
  call.shift = a->shift;
  call.tokens = a->tokens;
  call.offsets_out = a->token_offsets;
  call.slots = a->slots;
  call.positions = a->positions;
  return launch_pages(call, a->device_status, stream);
}

int gevva_step_trim(const gevva_step_trim_args* a, gevva_stream_t stream) {
  gv::PagesCall call{};
  if (!a || !fill_pages(&call, *a) || !aligned_to(a->keep, 4) || a->reserved) return GEVVA_MOE_BAD_ARGUMENT;
  const long long n = a->sequences;
  const Range read[] = {unless(a->lengths, a->lengths_out, n), words(a->keep, n), table_of(*a), unless(a->taken, a->taken_out, 1)};
  const Range written[] = {words(a->pool, a->pool_pages), words(a->lengths_out, n), words(a->taken_out, 1)};
  if (!apart(read, written)) return GEVVA_MOE_BAD_ARGUMENT;
  call.trim = true;
  call.counts = a->keep;
  return launch_pages(call, a->device_status, stream);
}

int gevva_step_sample(const gevva_step_sample_args* a, gevva_stream_t stream) {
  if (!a || a->rows < 0 || a->vocabulary < 1 || (a->f32 != 0 && a->f32 != 1) || !(a->softcap >= 0.0f) || isinf(a->softcap)) return GEVVA_MOE_BAD_ARGUMENT;
  if (a->rows == 0) return GEVVA_MOE_OK;
  const int size = a->f32 ? 4 : 2;
  if (!aligned_to(a->logits, size) || !aligned_to(a->uniforms, 4) || !aligned_or_null(a->temperature, 4) || !aligned_or_null(a->top_k, 4) ||
      !aligned_or_null(a->top_p, 4) || !aligned_or_null(a->min_p, 4) || !aligned_to(a->tokens, 4) || !aligned_or_null(a->probabilities, 4) ||
      (a->rows > 1 && (a->row_stride < 0 || a->row_stride >= 1ll << 38)))
    return GEVVA_MOE_BAD_ARGUMENT;
  if (a->vocabulary > gv::kMaxVocabulary || a->rows >= 1 << 27) return GEVVA_MOE_TOO_LARGE;
  const long long rows = a->rows, stride = rows > 1 ? a->row_stride : 0;
  const Range read[] = {{a->logits, size * ((rows - 1) * stride + a->vocabulary)}, {a->uniforms, 4 * rows}, {a->temperature, 4 * rows},
                        words(a->top_k, rows), {a->top_p, 4 * rows}, {a->min_p, 4 * rows}};
  const Range written[] = {words(a->tokens, rows), {a->probabilities, 4 * rows}};
  if (!apart(read, written)) return GEVVA_MOE_BAD_ARGUMENT;
  gv::SampleCall call{};
  call.logits = a->logits;
  call.row_stride = stride;
  call.wide = a->f32 != 0;
  call.uniforms = a->uniforms;
  call.temperature = a->temperature;
  call.top_k = a->top_k;
  call.top_p = a->top_p;
  call.min_p = a->min_p;
  call.softcap = a->softcap;
  call.rows = a->rows;
  call.vocabulary = a->vocabulary;
  call.tokens = a->tokens;
  call.probabilities = a->probabilities;
  return gv::launched(gv::launch_sample(call, gv::current_sm_count(), stream));
}

}  // extern "C"
