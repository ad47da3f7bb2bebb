// The row kernels around attention (declared in include/gevva_moe.h): RMS norms in front of and behind a block, and what happens to queries, keys and
// values between their projection and attention.  All are bound by HBM, or by latency for a few tokens: a value is read once, held in registers in
// 32 bits and written once.
#include "gv_attention.h"
#include "gv_common.cuh"
#include "gv_gemm_parts.cuh"

namespace gv {
namespace {

__device__ __forceinline__ void unpack8(const uint4& v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = bf16_bits_to_float(w[i] & 0xffffu);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  return make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
}
__device__ __forceinline__ float squares(const float (&x)[8]) {
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) s = fmaf(x[i], x[i], s);
  return s;
}

// ---- RMS norms in front of and behind a block ------------------------------------------------------------
// A row is held by kLanes threads: a warp for rows of up to 512 values, else a block; each thread has kEach times eight values of it.
struct NormParams {
  const uint4 *x, *weight, *residual, *gate, *next_weight;
  const __nv_bfloat16* scale;
  uint4 *out, *next;
  int rows, vectors;  // of eight values in a row
  float inverse_width, eps;
};

// Sum over the threads that hold a row, the same in each of them.
template <bool kBlock>
__device__ __forceinline__ float row_sum(float v, float* warp_sums) {
#pragma unroll
  for (int d = 16; d > 0; d /= 2) v += __shfl_xor_sync(0xffffffffu, v, d);
  if constexpr (kBlock) {
    const int warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0) warp_sums[threadIdx.x >> 5] = v;
    __syncthreads();
    v = (threadIdx.x & 31) < warps ? warp_sums[threadIdx.x & 31] : 0.0f;
#pragma unroll
    for (int d = 16; d > 0; d /= 2) v += __shfl_xor_sync(0xffffffffu, v, d);
  }
  return v;
}

template <bool kBlock, int kEach>
__global__ void __launch_bounds__(1024) block_norm_kernel(const NormParams p) {
  __shared__ float sums[2][32];
  const int lane = kBlock ? threadIdx.x : threadIdx.x & 31, lanes = kBlock ? blockDim.x : 32;
  const int row = kBlock ? blockIdx.x : blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
  grid_launch_dependents();
  grid_dependency_wait();
  if (row >= p.rows) return;
  const size_t base = static_cast<size_t>(row) * p.vectors;
  uint4 in[kEach], residual[kEach];
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int at = lane + k * lanes;
    in[k] = residual[k] = make_uint4(0, 0, 0, 0);
    if (at < p.vectors) {
      in[k] = p.x[base + at];
      if (p.residual) residual[k] = p.residual[base + at];
    }
  }
  float s = 0.0f;
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    float x[8];
    unpack8(in[k], x);
    s += squares(x);
  }
  const float inverse = rsqrtf(fmaf(row_sum<kBlock>(s, sums[0]), p.inverse_width, p.eps));
  const float scale = p.scale ? __bfloat162float(*p.scale) : 1.0f;
  float y[kEach][8];
  s = 0.0f;
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int at = lane + k * lanes;
    if (at < p.vectors) {
      float x[8], w[8], r[8], g[8];
      unpack8(in[k], x);
      unpack8(p.weight[at], w);
      unpack8(residual[k], r);
      if (p.gate) unpack8(p.gate[at], g);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float v = x[i] * inverse * w[i];
        if (p.gate) v *= g[i];
        if (p.residual) v = (r[i] + v) * scale;
        y[k][i] = v;
      }
      p.out[base + at] = pack8(y[k]);
      s += squares(y[k]);
    }
  }
  if (p.next) {
    const float again = rsqrtf(fmaf(row_sum<kBlock>(s, sums[1]), p.inverse_width, p.eps));
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const int at = lane + k * lanes;
      if (at < p.vectors) {
        float w[8];
        unpack8(p.next_weight[at], w);
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] *= y[k][i] * again;
        p.next[base + at] = pack8(w);
      }
    }
  }
}

// ---- queries, keys and values: per-head norms, rotation, the cache -----------------------------------------
constexpr int kAppendThreads = 256;
constexpr int kMaxDim = 512;

struct AppendParams {
  AttnRows q, k, v;
  AttnPages pages;
  const int* token_offsets;
  int sequences, heads, kv_heads;
  const double* frequencies;
  int half;  // frequencies: the pairs (j, half + j) turn
  const uint4 *q_weight, *k_weight;
  bool normalize_v;
  float eps;
  __nv_bfloat16 *q_out, *k_out, *v_out;
  int* status;
};

// A CTA takes one token, so that an angle is worked out once for all heads.  A thread holds eight columns of a head (two times eight
// of a head of 512); the other half of a pair comes through shared memory.
template <int kDim>
__global__ void __launch_bounds__(kAppendThreads) kv_append_kernel(const AppendParams p) {
  constexpr int kLanes = kDim / 8 < 32 ? kDim / 8 : 32;  // lanes of a head
  constexpr int kEach = kDim / 8 / kLanes;
  constexpr int kHeads = 32 / kLanes;                    // heads of a warp
  __shared__ float2 turns[kMaxDim / 2];
  __shared__ float values[kAppendThreads / 32][kHeads * kDim];
  const int token = blockIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_launch_dependents();
  grid_dependency_wait();

  // the sequence: offsets up to the token's
  int upto = 0;
  for (int base = 0; base <= p.sequences; base += kAppendThreads) {
    const int s = base + static_cast<int>(threadIdx.x);
    upto += __syncthreads_count(s <= p.sequences && p.token_offsets[s] <= token);
  }
  if (upto == 0 || upto > p.sequences) return;  // a row in front of the first or behind the last sequence: left as it was
  const int sequence = upto - 1;
  const int position = p.pages.lengths[sequence] - p.token_offsets[upto] + token;
  const int page_index = position / p.pages.page_size;
  int page = -1;
  if (position >= 0 && page_index < p.pages.table_width)
    page = p.pages.table[static_cast<size_t>(sequence) * p.pages.table_stride + page_index];
  const bool stored = page >= 0 && page < p.pages.page_count;
  if (!stored && threadIdx.x == 0 && p.status) atomicExch(p.status, static_cast<int>(kBadPage));
  const long long slot = position - page_index * p.pages.page_size;

  // position * frequency in 64 bits, whole turns taken off there: far positions keep the accuracy of near ones
  for (int j = threadIdx.x; j < p.half; j += kAppendThreads) {
    const double angle = static_cast<double>(position) * p.frequencies[j] * 0.31830988618379067154;  // in half turns
    float sine, cosine;
    sincospif(static_cast<float>(angle - 2.0 * rint(0.5 * angle)), &sine, &cosine);
    turns[j] = make_float2(cosine, sine);
  }
  __syncthreads();

  const int total = p.heads + 2 * p.kv_heads;
  const int in_warp = lane / kLanes, in_head = lane % kLanes;
  float* shared_head = values[warp] + in_warp * kDim;
  for (int first = warp * kHeads; first < total; first += kAppendThreads / 32 * kHeads) {
    const int h = first + in_warp;
    const bool exists = h < total;
    const int kind = h < p.heads ? 0 : h < p.heads + p.kv_heads ? 1 : 2;  // query, key, value
    const int head = kind == 0 ? h : kind == 1 ? h - p.heads : h - p.heads - p.kv_heads;
    const AttnRows& from = kind == 0 ? p.q : kind == 1 ? p.k : p.v;
    const uint4* in = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(from.data) + token * from.token_stride +
                                                     head * from.head_stride);
    float x[kEach][8];
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      unpack8(exists ? in[in_head + k * kLanes] : make_uint4(0, 0, 0, 0), x[k]);
      s += squares(x[k]);
    }
    const uint4* weight = kind == 0 ? p.q_weight : kind == 1 ? p.k_weight : nullptr;
    const bool normal = kind == 2 ? p.normalize_v : weight != nullptr;
#pragma unroll
    for (int d = kLanes / 2; d > 0; d /= 2) s += __shfl_xor_sync(0xffffffffu, s, d);
    const float inverse = normal ? rsqrtf(fmaf(s, 1.0f / kDim, p.eps)) : 1.0f;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      float w[8];
      if (weight) unpack8(weight[in_head + k * kLanes], w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[k][i] *= inverse;
        if (weight) x[k][i] *= w[i];
      }
    }
    if (p.half > 0) {
      __syncwarp();
#pragma unroll
      for (int k = 0; k < kEach; ++k) {
        float4* to = reinterpret_cast<float4*>(shared_head + 8 * (in_head + k * kLanes));
        to[0] = make_float4(x[k][0], x[k][1], x[k][2], x[k][3]);
        to[1] = make_float4(x[k][4], x[k][5], x[k][6], x[k][7]);
      }
      __syncwarp();
      if (kind != 2) {
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
          const int column = 8 * (in_head + k * kLanes);
          if (column < 2 * p.half) {  // (half is a multiple of eight)
            const bool low = column < p.half;
            const int pair = low ? column : column - p.half;
            const float* other = shared_head + (low ? column + p.half : pair);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float2 turn = turns[pair + i];
              x[k][i] = x[k][i] * turn.x + (low ? -other[i] : other[i]) * turn.y;
            }
          }
        }
      }
    }
    if (!exists) continue;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const uint4 packed = pack8(x[k]);
      const int at = in_head + k * kLanes;
      const size_t row = static_cast<size_t>(token) * (kind == 0 ? p.heads : p.kv_heads) + head;
      if (kind == 0) {
        reinterpret_cast<uint4*>(p.q_out + row * kDim)[at] = packed;
      } else {
        __nv_bfloat16* out = kind == 1 ? p.k_out : p.v_out;
        if (out) reinterpret_cast<uint4*>(out + row * kDim)[at] = packed;
        if (stored) {
          __nv_bfloat16* cache = kind == 1 ? static_cast<__nv_bfloat16*>(p.pages.keys) + page * p.pages.key_page_stride +
                                                 slot * p.pages.key_slot_stride + head * p.pages.key_head_stride
                                           : static_cast<__nv_bfloat16*>(p.pages.values) + page * p.pages.value_page_stride +
                                                 slot * p.pages.value_slot_stride + head * p.pages.value_head_stride;
          reinterpret_cast<uint4*>(cache)[at] = packed;
        }
      }
    }
  }
}

}  // namespace

cudaError_t launch_block_norm(const BlockNormCall& call, int sm_count, cudaStream_t stream) {
  (void)sm_count;
  NormParams p{};
  p.x = static_cast<const uint4*>(call.x);
  p.weight = static_cast<const uint4*>(call.weight);
  p.residual = static_cast<const uint4*>(call.residual);
  p.gate = static_cast<const uint4*>(call.gate);
  p.next_weight = static_cast<const uint4*>(call.next_weight);
  p.scale = static_cast<const __nv_bfloat16*>(call.scale);
  p.out = static_cast<uint4*>(call.out);
  p.next = static_cast<uint4*>(call.next);
  p.rows = call.rows;
  p.vectors = call.width / 8;
  p.inverse_width = 1.0f / static_cast<float>(call.width);
  p.eps = call.eps;
  if (p.vectors <= 64) {
    const dim3 grid((call.rows + 7) / 8), block(256);
    if (p.vectors <= 32) return launch_chained(block_norm_kernel<false, 1>, grid, block, 0, stream, p);
    return launch_chained(block_norm_kernel<false, 2>, grid, block, 0, stream, p);
  }
  const dim3 grid(call.rows);
  if (p.vectors <= 512) return launch_chained(block_norm_kernel<true, 1>, grid, dim3((p.vectors + 31) / 32 * 32), 0, stream, p);
  if (p.vectors <= 1024) return launch_chained(block_norm_kernel<true, 2>, grid, dim3((p.vectors + 63) / 64 * 32), 0, stream, p);
  return launch_chained(block_norm_kernel<true, 4>, grid, dim3((p.vectors + 127) / 128 * 32), 0, stream, p);
}

cudaError_t launch_kv_append(const AppendCall& call, cudaStream_t stream) {
  AppendParams p{};
  p.q = call.q;
  p.k = call.k;
  p.v = call.v;
  p.pages = call.pages;
  p.token_offsets = call.token_offsets;
  p.sequences = call.sequences;
  p.heads = call.heads;
  p.kv_heads = call.kv_heads;
  p.frequencies = call.frequencies;
  p.half = call.rotated / 2;
  p.q_weight = static_cast<const uint4*>(call.q_weight);
  p.k_weight = static_cast<const uint4*>(call.k_weight);
  p.normalize_v = call.normalize_v;
  p.eps = call.eps;
  p.q_out = static_cast<__nv_bfloat16*>(call.q_out);
  p.k_out = static_cast<__nv_bfloat16*>(call.k_out);
  p.v_out = static_cast<__nv_bfloat16*>(call.v_out);
  p.status = call.status;
  const dim3 grid(call.tokens), block(kAppendThreads);
  switch (call.dim) {
    case 64: return launch_chained(kv_append_kernel<64>, grid, block, 0, stream, p);
    case 128: return launch_chained(kv_append_kernel<128>, grid, block, 0, stream, p);
    case 256: return launch_chained(kv_append_kernel<256>, grid, block, 0, stream, p);
    default: return launch_chained(kv_append_kernel<512>, grid, block, 0, stream, p);
  }
}

}  // namespace gv
