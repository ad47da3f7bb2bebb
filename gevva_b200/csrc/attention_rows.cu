// The row kernels around attention (declared in include/gevva_moe.h): RMS norms in front of and behind a block, and what happens to
// queries, keys and values between their projection and attention.  All are bound by HBM, or by latency for a few tokens: a value is read
// once, held in registers in 32 bits and written once.
#include "gv_attention.h"
#include "gv_common.cuh"
#include "gv_gemm_parts.cuh"
#include "gv_step.h"

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
// A row is held by a warp or by a block; each thread has kEach times eight values of it, as they came, in registers: the second norm
// works its row out again instead of keeping it in 32 bits.
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

template <bool kBlock, int kEach, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) block_norm_kernel(const NormParams p) {
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
  const auto value_of = [&](int k, int at, float (&y)[8]) {
    float w[8], r[8], g[8];
    unpack8(in[k], y);
    unpack8(p.weight[at], w);
    unpack8(residual[k], r);
    if (p.gate) unpack8(p.gate[at], g);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      y[i] = y[i] * inverse * w[i];
      if (p.gate) y[i] *= g[i];
      if (p.residual) y[i] = (r[i] + y[i]) * scale;
    }
  };
  s = 0.0f;
#pragma unroll
  for (int k = 0; k < kEach; ++k) {
    const int at = lane + k * lanes;
    if (at < p.vectors) {
      float y[8];
      value_of(k, at, y);
      p.out[base + at] = pack8(y);
      s += squares(y);
    }
  }
  if (p.next) {
    const float again = rsqrtf(fmaf(row_sum<kBlock>(s, sums[1]), p.inverse_width, p.eps));
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const int at = lane + k * lanes;
      if (at < p.vectors) {
        float y[8], w[8];
        value_of(k, at, y);
        unpack8(p.next_weight[at], w);
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] *= y[i] * again;
        p.next[base + at] = pack8(w);
      }
    }
  }
}

// ---- queries, keys and values: per-head norms, rotation, the cache -----------------------------------------
constexpr int kMaxDim = 512;

// Of queries, keys and values by number: what a head has is read by its kind, which costs an indexed read of the constants instead of a
// choice for each word of each.
struct AppendSide {
  const uint4* weight;
  __nv_bfloat16 *out, *cache;
  long long page_stride, slot_stride, head_stride;  // of the cache
  int first_head, heads, norm, turns;
};
struct AppendParams {
  AttnRows rows[3];
  AppendSide side[3];
  AttnPages pages;
  const int* token_offsets;
  int sequences, tokens, heads, kv_heads;
  const double* frequencies;
  int half;        // frequencies: the pairs (j, half + j) turn
  int page_shift;
  float eps;
  int* status;
  // at given places
  const int *slots, *positions;
  long long position_stride;
  int axes;
};

// A CTA takes a token, or one after the other where there are many, so that an angle is worked out once for all heads.  A thread holds
// eight pairs of a head: the two halves of a pair come from two 16-byte vectors, (u, half / 8 + u) where pairs turn and two neighbours
// behind them, so nothing is exchanged.  Its first vectors are asked for before the token's place is looked up, behind the last ones of
// the token before.
// 4608 tokens of 32 heads of 256, packed: 35.9 us, of which 28.8 are its bytes (38.7 with queries, keys and values told apart by choices
// and weights read as they are; with a CTA for each token 2 more).
// kPlaced: slots and positions are given, one read instead of the look-ups of sequence, length and page; a position for each axis, and
// frequencies for each, most of them zero: a pair's angle is their sum of products, exactly its axis's product where the others are zero.
// The next token's are asked for in front of a token's heads and worked out behind them, into the other half of the arrays: one barrier a token.
// 64 tokens 2.8 us, 4608 (as above, three axes) 37.1, 16384 of 48 heads of 128 90 of 62 for its bytes: 0.66 instructions a cycle and scheduler, at 20 warps an SM.
// (Multiplications two an instruction 94 us; six CTAs an SM with 80 registers 104.)
constexpr int kAppendThreads = 512, kAppendManyThreads = 128;
constexpr int kAppendManyCtas = 5;  // of an SM (with six: 80 registers, which do not hold it all)
template <int kDim, int kThreads, bool kPlaced>
__global__ void __launch_bounds__(kThreads, kThreads == kAppendManyThreads ? kAppendManyCtas : 1) kv_append_kernel(const AppendParams p) {
  constexpr int kLanes = kDim / 16;  // threads of a head
  constexpr bool kMany = kThreads == kAppendManyThreads;
  constexpr int kBuffers = kPlaced ? 2 : 1;
  __shared__ alignas(16) float all_cosines[kBuffers][kMaxDim / 2], all_sines[kBuffers][kMaxDim / 2];
  const int u = threadIdx.x % kLanes, in_block = threadIdx.x / kLanes, heads_at_once = blockDim.x / kLanes;
  const int eighth = p.half / 8;
  const bool turns = u < eighth;
  const int low = turns ? u : 2 * u, high = turns ? u + eighth : 2 * u + 1;  // vectors
  const int total = p.heads + 2 * p.kv_heads;
  // Many tokens: the weights of queries and of keys, of each lane its two vectors by halves, as numbers of 32 bits.
  __shared__ float4 weights[kMany ? 2 : 1][4][kMany ? kLanes : 1];
  grid_launch_dependents();
  grid_dependency_wait();
  if constexpr (kMany) {
    if (threadIdx.x < 2 * kLanes) {
      const int kind = threadIdx.x / kLanes;
      if (p.side[kind].weight) {
        float w[8], z[8];
        unpack8(p.side[kind].weight[low], w);
        unpack8(p.side[kind].weight[high], z);
        weights[kind][0][u] = make_float4(w[0], w[1], w[2], w[3]);
        weights[kind][1][u] = make_float4(w[4], w[5], w[6], w[7]);
        weights[kind][2][u] = make_float4(z[0], z[1], z[2], z[3]);
        weights[kind][3][u] = make_float4(z[4], z[5], z[6], z[7]);
      }
    }
  }

  const auto kind_of = [&](int h) { return (h >= p.heads) + (h >= p.heads + p.kv_heads); };
  const auto source = [&](int token, int h) {
    const int kind = kind_of(h);
    const AttnRows& from = p.rows[kind];
    return reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(from.data) + token * from.token_stride +
                                          (h - p.side[kind].first_head) * from.head_stride);
  };
  uint4 a[2], b[2];  // of two heads, asked for together
  const auto ask = [&](int token, int first) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int h = first + k * heads_at_once;
      a[k] = b[k] = make_uint4(0, 0, 0, 0);
      if (h < total) {
        const uint4* const from = source(token, h);
        a[k] = from[low];
        b[k] = from[high];
      }
    }
  };
  ask(blockIdx.x, in_block);

  // position * frequency in 64 bits, whole turns taken off there: far positions keep the accuracy of near ones.  Groups of four of a
  // thread's eight stand in the two halves of the arrays, so that a warp's 16-byte reads follow one another.
  const int quarters = p.half / 8;
  const auto turn = [&](int j, double turned, int buffer) {
    const double angle = turned * 0.31830988618379067154;  // in half turns
    float sine, cosine;
    sincospif(static_cast<float>(angle - 2.0 * rint(0.5 * angle)), &sine, &cosine);
    const int at = ((j >> 2) & 1) * 4 * quarters + (j >> 3) * 4 + (j & 3);
    all_cosines[buffer][at] = cosine;
    all_sines[buffer][at] = sine;
  };
  // of a given place: its slot, and its positions along the first axes
  constexpr int kAxes = 4;
  int place = 0, places[kAxes] = {0, 0, 0, 0}, buffer = 0;
  const auto look_up = [&](int token) {
    place = p.slots[token];
#pragma unroll
    for (int axis = 0; axis < kAxes; ++axis) places[axis] = axis < p.axes ? p.positions[axis * p.position_stride + token] : 0;
  };
  const auto turn_placed = [&](int token, int into) {
    for (int j = threadIdx.x; j < p.half; j += blockDim.x) {
      double turned = static_cast<double>(places[0]) * p.frequencies[j];
#pragma unroll
      for (int axis = 1; axis < kAxes; ++axis)
        if (axis < p.axes) turned += static_cast<double>(places[axis]) * p.frequencies[axis * p.half + j];
      for (int axis = kAxes; axis < p.axes; ++axis)
        turned += static_cast<double>(p.positions[axis * p.position_stride + token]) * p.frequencies[axis * p.half + j];
      turn(j, turned, into);
    }
  };
  if constexpr (kPlaced) {
    look_up(blockIdx.x);
    turn_placed(blockIdx.x, 0);
  }

#pragma unroll 1
  for (int token = blockIdx.x; token < p.tokens; token += gridDim.x) {
  const int next_token = kMany ? token + static_cast<int>(gridDim.x) : p.tokens;
  int position, page = -1, in_page;
  if constexpr (kPlaced) {
    const int at = place;
    const bool none = __syncthreads_or(at < 0);  // (and the token's angles are there)
    const bool again = next_token < p.tokens;
    if (again) look_up(next_token);
    if (none) {  // a row that is no token: left as it was
      if (again) {
        ask(next_token, in_block);
        buffer ^= 1;
        turn_placed(next_token, buffer);
      }
      continue;
    }
    page = at >> p.page_shift;
    in_page = at & (p.pages.page_size - 1);
    position = 0;
  } else {
  // the sequence: offsets up to the token's
  int upto = 0;
  for (int base = 0; base <= p.sequences; base += blockDim.x) {
    const int s = base + static_cast<int>(threadIdx.x);
    upto += __syncthreads_count(s <= p.sequences && p.token_offsets[s] <= token);
  }
  if (upto == 0 || upto > p.sequences) {  // a row in front of the first or behind the last sequence: left as it was
    if (next_token < p.tokens) ask(next_token, in_block);
    continue;
  }
  const int sequence = upto - 1;
  position = p.pages.lengths[sequence] - p.token_offsets[upto] + token;
  const int page_index = position >> p.page_shift;
  if (position >= 0 && page_index < p.pages.table_width)
    page = p.pages.table[static_cast<size_t>(sequence) * p.pages.table_stride + page_index];
  in_page = position & (p.pages.page_size - 1);
  }
  const bool stored = page >= 0 && page < p.pages.page_count;
  if (!stored && threadIdx.x == 0 && p.status) atomicExch(p.status, static_cast<int>(kBadPage));
  const long long slot = in_page;

  if constexpr (!kPlaced) {
    for (int j = threadIdx.x; j < p.half; j += blockDim.x) turn(j, static_cast<double>(position) * p.frequencies[j], 0);
    __syncthreads();
  }
  const float* const cosines = all_cosines[kPlaced ? buffer : 0];
  const float* const sines = all_sines[kPlaced ? buffer : 0];

#pragma unroll 1
  for (int first_head = in_block; first_head < total; first_head += 2 * heads_at_once) {
  const uint4 low_now[2] = {a[0], a[1]}, high_now[2] = {b[0], b[1]};
  const bool more = first_head + 2 * heads_at_once < total;
  if (more || next_token < p.tokens) ask(more ? token : next_token, more ? first_head + 2 * heads_at_once : in_block);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int h = first_head + k * heads_at_once;
    if (h >= total) break;
    const int kind = kind_of(h);
    const AppendSide& side = p.side[kind];
    const int head = h - side.first_head;
    float x[8], y[8];
    unpack8(low_now[k], x);
    unpack8(high_now[k], y);
    const uint4* weight = side.weight;
    if (side.norm) {  // (the same for all threads of a head, which are in one warp)
      float s = squares(x) + squares(y);
      const uint32_t mates = kLanes == 32 ? 0xffffffffu : ((1u << (kLanes & 31)) - 1u) << ((threadIdx.x & 31) / kLanes * kLanes);
#pragma unroll
      for (int d = kLanes / 2; d > 0; d /= 2) s += __shfl_xor_sync(mates, s, d);
      const float inverse = rsqrtf(fmaf(s, 1.0f / kDim, p.eps));
      float w[8], z[8];
      if (weight) {
        if constexpr (kMany) {
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const float4 first = weights[kind][g][u], second = weights[kind][2 + g][u];
            w[4 * g] = first.x, w[4 * g + 1] = first.y, w[4 * g + 2] = first.z, w[4 * g + 3] = first.w;
            z[4 * g] = second.x, z[4 * g + 1] = second.y, z[4 * g + 2] = second.z, z[4 * g + 3] = second.w;
          }
        } else {
          unpack8(weight[low], w);
          unpack8(weight[high], z);
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        x[i] *= inverse;
        y[i] *= inverse;
        if (weight) {
          x[i] *= w[i];
          y[i] *= z[i];
        }
      }
    }
    if (side.turns && turns) {
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const float4 c = *reinterpret_cast<const float4*>(cosines + g * 4 * quarters + 4 * u);
        const float4 s = *reinterpret_cast<const float4*>(sines + g * 4 * quarters + 4 * u);
        const float cs[4] = {c.x, c.y, c.z, c.w}, sn[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float first = x[4 * g + i], second = y[4 * g + i];
          x[4 * g + i] = first * cs[i] - second * sn[i];
          y[4 * g + i] = second * cs[i] + first * sn[i];
        }
      }
    }
    const uint4 first = pack8(x), second = pack8(y);
    const size_t row = static_cast<size_t>(token) * side.heads + head;
    __nv_bfloat16* out = side.out;
    if (out) {
      reinterpret_cast<uint4*>(out + row * kDim)[low] = first;
      reinterpret_cast<uint4*>(out + row * kDim)[high] = second;
    }
    __nv_bfloat16* cache = side.cache;
    if (cache && stored) {
      cache += page * side.page_stride + slot * side.slot_stride + head * side.head_stride;
      reinterpret_cast<uint4*>(cache)[low] = first;
      reinterpret_cast<uint4*>(cache)[high] = second;
    }
  }
  }
  if constexpr (kPlaced) {
    if (next_token < p.tokens) {
      buffer ^= 1;
      turn_placed(next_token, buffer);
    }
  } else if constexpr (kMany) {
    __syncthreads();  // (the angles are another token's next)
  }
  }
}

}  // namespace

cudaError_t launch_block_norm(const BlockNormCall& call, int sm_count, cudaStream_t stream) {
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
  if (p.vectors <= 32) return launch_chained(block_norm_kernel<false, 1, 128>, dim3((static_cast<unsigned>(call.rows) + 3) / 4), dim3(128), 0, stream, p);
  const dim3 grid(call.rows);
  // Four warps a row where there are rows for all SMs several times over: sixteen rows of an SM at a time have more bytes on their way
  // than five of eleven warps.
  if (p.vectors <= 512 && call.rows >= 4 * sm_count) {
    if (p.vectors <= 128) return launch_chained(block_norm_kernel<true, 1, 128>, grid, dim3(128), 0, stream, p);
    if (p.vectors <= 256) return launch_chained(block_norm_kernel<true, 2, 128>, grid, dim3(128), 0, stream, p);
    if (p.vectors <= 384) return launch_chained(block_norm_kernel<true, 3, 128>, grid, dim3(128), 0, stream, p);
    return launch_chained(block_norm_kernel<true, 4, 128>, grid, dim3(128), 0, stream, p);
  }
  if (p.vectors <= 512) return launch_chained(block_norm_kernel<true, 1, 512>, grid, dim3((p.vectors + 31) / 32 * 32), 0, stream, p);
  if (p.vectors <= 1024) return launch_chained(block_norm_kernel<true, 2, 1024>, grid, dim3((p.vectors + 63) / 64 * 32), 0, stream, p);
  return launch_chained(block_norm_kernel<true, 4, 1024>, grid, dim3((p.vectors + 127) / 128 * 32), 0, stream, p);
}

namespace {

AppendParams append_params(const AppendCall& call) {
  AppendParams p{};
  p.rows[0] = call.q;
  p.rows[1] = call.k;
  p.rows[2] = call.v;
  const AttnPages& c = call.pages;
  p.side[0] = {static_cast<const uint4*>(call.q_weight), static_cast<__nv_bfloat16*>(call.q_out), nullptr, 0, 0, 0, 0, call.heads, call.q_weight != nullptr, 1};
  p.side[1] = {static_cast<const uint4*>(call.k_weight), static_cast<__nv_bfloat16*>(call.k_out), static_cast<__nv_bfloat16*>(c.keys),
               c.key_page_stride, c.key_slot_stride, c.key_head_stride, call.heads, call.kv_heads, call.k_weight != nullptr, 1};
  p.side[2] = {nullptr, static_cast<__nv_bfloat16*>(call.v_out), static_cast<__nv_bfloat16*>(c.values),
               c.value_page_stride, c.value_slot_stride, c.value_head_stride, call.heads + call.kv_heads, call.kv_heads, call.normalize_v, 0};
  p.pages = c;
  p.token_offsets = call.token_offsets;
  p.sequences = call.sequences;
  p.tokens = call.tokens;
  p.heads = call.heads;
  p.kv_heads = call.kv_heads;
  p.frequencies = call.frequencies;
  p.half = call.rotated / 2;
  p.eps = call.eps;
  p.status = call.status;
  while ((1 << p.page_shift) < call.pages.page_size) ++p.page_shift;
  return p;
}

template <bool kPlaced>
cudaError_t launch_append(const AppendCall& call, const AppendParams& p, int sm_count, cudaStream_t stream) {
  // Threads for all heads of a token at once; with tokens for all SMs several times over four warps a token, so that more
  // tokens' chains of look-ups run side by side (64 tokens 4.3 and 5.6 us, 4608 tokens 47 and 41 us with up to eight warps and four).
  const int wanted = ((call.heads + 2 * call.kv_heads) * (call.dim / 16) + 31) / 32 * 32;
  const bool many = call.tokens >= 4 * sm_count;
  const int most = many ? kAppendManyThreads : kAppendThreads;
  const int ctas = kAppendManyCtas * sm_count;
  const dim3 grid(many && call.tokens > ctas ? ctas : call.tokens), block(wanted < most ? wanted : most);
#define GV_APPEND(dim) \
  launch_chained(many ? kv_append_kernel<dim, kAppendManyThreads, kPlaced> : kv_append_kernel<dim, kAppendThreads, kPlaced>, grid, block, 0, stream, p)
  switch (call.dim) {
    case 64: return GV_APPEND(64);
    case 128: return GV_APPEND(128);
    case 256: return GV_APPEND(256);
    default: return GV_APPEND(512);
  }
#undef GV_APPEND
}

}  // namespace

cudaError_t launch_kv_append(const AppendCall& call, int sm_count, cudaStream_t stream) {
  return launch_append<false>(call, append_params(call), sm_count, stream);
}

cudaError_t launch_kv_append_placed(const PlacedCall& call, int sm_count, cudaStream_t stream) {
  AppendParams p = append_params(call.rows);
  p.slots = call.slots;
  p.positions = call.positions;
  p.position_stride = call.position_stride;
  p.axes = call.axes;
  return launch_append<true>(call.rows, p, sm_count, stream);
}

}  // namespace gv
