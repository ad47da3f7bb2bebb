// Causal attention with grouped heads: whole prompts over packed keys, or new tokens over a paged cache (declared in
// include/gevva_moe.h as gevva_attn_prompt and gevva_attn_chunk).
//
//   o_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(scale * q_i.k_j - m_i),   i - window < j <= i
//
// in one pass over the keys: a row keeps a reference m_i, the sum of its p and the sum of p * v.  The sums may be taken against any
// reference, so m_i follows the row's maximum only when that has grown by more than 8 binary orders (p stays below 256); only then is what
// has been summed scaled down.  p is rounded to bf16 for its product with v (2^-8 of each term at most, as v itself was), and its sum is of the
// rounded values: the result is then a mean of v whose weights are off, and what is off cancels where few keys have all the weight (scores of
// deviation 4 over 1024 keys: 8.1e-4 of the result's size, with the sum of the unrounded 1.42e-3; of deviation 1: 1.58e-3 and 1.59e-3).
//
// A query tile is 128 rows: floor(128 / group) tokens times the query heads of one key head, so that a key tile of 128 keys is read
// once for all of them, with one token as with many.  Scores and outputs are products of the tensor pipe (tcgen05.mma, M = 128): S = Q K^T
// with both operands in shared memory, O += P V with P in tensor memory, where the softmax threads leave it over the scores it came from.
//   warp 0    fetches Q, K and V by TMA, a page's slots at a time where the keys are paged
//   warp 1    issues the products, by one thread: the tensor pipe holds few of them ahead, so an issuer's votes and branches are time
//             that it stands still (heads of 512: 1190 -> 1068 us; with a second issuer for the outputs 1295, since the two kinds of
//             product then alternate)
//   warp 2    works out the pieces of work, a step ahead of the others
//   warps 4+  softmax and epilogue, a row per thread, by two warpgroups
// Tensor memory holds two score tiles (three with heads of 64) and the outputs.  Heads of 256 and 512 (the value columns of 512 in two
// items): one query tile. Its key tiles are taken by the warpgroups in turn, and the scores of the next are worked out while the softmax
// of this one runs, over the end of a piece too; a key tile takes the tensor pipe 2048 cycles, and half as much again for 512, whose
// scores both items work out.
// Heads of 64 and 128: two query tiles, a warpgroup each, since there a tile's exponentials take as long as its products or longer.
//
// Work is dealt out in key tiles (gv_attention_plan.h).  Prompts: an item, one query tile of one head, is never cut; CTAs take the
// items, a sequence's last and longest first, further ones by cancelling launches that have not started (clusterlaunchcontrol).  Chunks:
// a CTA takes an equal run of key tiles, whatever the sequences' lengths, which only the device knows; an item that a run's end cuts
// leaves sums in the workspace, and attention_join_kernel adds them up in the order of the keys: no atomics, and the same bits every time.
//
// What bounds it (B200, of 1658 TFLOP/s and 6.56 TB/s measured; in a graph, on a cool GPU and, behind it, under its power limit, where the clock is
// 1.6 GHz).  Prompts: 8192 tokens causal, 16 heads of 256 405 and 425 us (1360 and 1290 TFLOP/s), 32 of 64 339 and 405 (810 and 680), 8191
// tokens, 32 of 128 454 and 534 (1210 and 1030), 4608 tokens, 16 of 512 361 to 373 (960 to 930, half as much again with the scores that are worked
// out twice).  Neither L2 nor shared memory bounds them: with boxes outside the tensors, which TMA fills with zeros and reads nothing for, 674 k
// cycles become 656 k (256), 860 k 839 k (128) and 602 k 568 k (512), without the writes too 680 k, 860 k and 538 k.  Heads of 256 and 512: the
// tensor pipe, at work for 71 and 76 % of the cycles, and what lies between its batches.  Heads of 128: a query tile's chain of softmax, outputs
// and next scores.  Heads of 64: the softmax warps' instructions.  Decoding: HBM, 5.7 to 6.2 TB/s in a graph at 64 sequences of 8 key heads of 256
// (by where a process's caches lie; 5.1 over 6 GB of them in turn); a single short one is a chain of latencies, 14.6 us (launch and plan
// 3, first keys 2.5, softmax of cold code 1.5, outputs 2, second launch 4).
#include <cuda.h>
#include <math_constants.h>

#include "gv_attention.h"
#include "gv_attention_plan.h"
#include "gv_common.cuh"
#include "gv_gemm_parts.cuh"
#include "gv_launchers.h"

namespace gv {
namespace {

constexpr int kRows = 128;         // rows of a query tile
constexpr int kKeys = kAttnKeys;   // keys of a key tile
constexpr int kPieceSlots = 3;     // pieces in work: one whose outputs are read, one whose scores are, one whose operands are fetched
// Items that CTAs take from one another are better not taken far ahead (1500, 1, 2049 and 1058 tokens through a window of 1024: 67.7 ->
// 65.7 us), but with two query tiles the time to the next counts more (8192 tokens, heads of 64: 383 and 391 us).
template <int kTiles, bool kPaged>
constexpr uint32_t kSlotsOf = kPaged || kTiles == 2 ? kPieceSlots : 2;
constexpr int kColumnBytes = kKeys * 128;  // 64 columns of a tile: 128 rows of 128 bytes, one swizzle row each
constexpr float kGrowth = 8.0f;    // binary orders by which a row's maximum may exceed its reference
constexpr int kLeastRun = 1;       // key tiles of the shortest run that a CTA is given (one reply of 700 tokens, 8 key heads of 256:
                                   // 16.0 us, with 2 16.4, with 4 20.8)

// One run of key tiles of one item.
struct Piece {
  int tiles;       // 0: there are no more pieces
  int first_tile;
  int query0;      // row in q of the query tile's first token
  int tokens;      // its tokens
  int position0;   // of the first token
  int key_origin;  // prompt: row in k of the sequence's first key
  int sequence;
  int kv_head, half;
  int slot;        // where its sums go; -1: the whole item, which goes to the output
};

// Keys of a piece's j-th tile that some row of its item sees: [from, to) within the tile.  What stands elsewhere is other sequences' or
// stale (behind the sequence's end, in front of the window), and zero times a value need not be zero: those rows of V are cleared.
struct Seen {
  int from, to;
  __device__ bool all() const { return from <= 0 && to >= kKeys; }
};
__device__ __forceinline__ Seen seen_keys(const Piece& piece, int j, int window) {
  const int key0 = (piece.first_tile + j) * kKeys;
  return Seen{(window > 0 ? max(piece.position0 - window + 1, 0) : 0) - key0, max(piece.position0 + piece.tokens, 0) - key0};
}

template <int kDim, int kTiles>
struct Shape {
  static constexpr int kValueDim = kDim < 256 ? kDim : 256;
  static constexpr int kHalves = kDim / kValueDim;
  static constexpr int kStageDim = kDim < 128 ? kDim : 128;
  static constexpr int kStageBytes = kKeys * kStageDim * 2;
  static constexpr int kKeyStages = kDim / kStageDim;
  static constexpr int kValueStages = kValueDim / kStageDim;
  static constexpr int kQueryTileBytes = kRows * kDim * 2;
  static constexpr int kControlBytes = 3 << 10;
  static constexpr int kRoom = (232448 - kControlBytes - kTiles * kQueryTileBytes) / kStageBytes;
  static constexpr int kStages = kRoom < 8 ? kRoom : 8;
  static constexpr int kSoftmaxWarps = 8;
  static constexpr int kThreads = 128 + 32 * kSoftmaxWarps;
  // Whether a tile's values and the next one's keys fit side by side: scores of the next piece may then be asked for before this one's end.
  static constexpr bool kAhead = kTiles == 1 && kStages >= kKeyStages + kValueStages;
  // Two query tiles of heads of 64 leave tensor memory for a third score tile: scores are then asked for half a round earlier, and the
  // chain of a query tile is its softmax alone (8192 tokens, 32 heads: 389 -> 347 us; 339 now, with one exponential of eight instead of three on
  // the multiply-add units).  Score tile 2 * (key tile) + (query tile), modulo three.
  static constexpr bool kSpare = kTiles == 2 && kDim == 64;
  static constexpr uint32_t kOutputs = kSpare ? 384 : 256;  // first tensor-memory column of the outputs
  static_assert(!kSpare || (kStages & (kStages - 1)) == 0, "stages are found by position");
  static_assert(kStages > kValueStages, "the values of a tile are in shared memory at the same time");
  static_assert(kTiles == 1 || kDim <= 128, "two query tiles need 2 * (128 + dim) columns of tensor memory");
};

template <int kDim, int kTiles>
struct AttnSmem {
  using S = Shape<kDim, kTiles>;
  uint8_t queries[kTiles][S::kQueryTileBytes];
  uint8_t stage[S::kStages][S::kStageBytes];
  uint64_t full[S::kStages], empty[S::kStages];
  uint64_t q_full, q_empty;
  // Scores are there, P is, outputs of a key tile are summed up: by key tile in turn (one query tile), by query tile (two), or by both
  // (three score tiles, 2 * query tile + turn: the next scores do not wait for all warps' P there, so that a warp whose rows do not exist
  // may be a key tile ahead).
  uint64_t acc_full[4], p_ready[4], pv_done[4];
  uint64_t o_free[kTiles];    // the outputs of the last piece have been read
  uint64_t piece_full[kPieceSlots], piece_empty[kPieceSlots];
  uint64_t v_landed[2];       // values of a tile that has rows to be cleared, by softmax warpgroup
  // One query tile: the warpgroups take the key tiles in turn, and hand each row's reference and sum on (a barrier for each quarter's
  // warps).
  uint64_t reference_ready[2][4], sum_ready[2][4];
  uint64_t next_full;
  alignas(16) uint4 next_item;  // answer to a request for another item
  Piece pieces[kPieceSlots];
  uint32_t tmem_base;
  volatile int abort;
  float references[kTiles == 1 ? 2 : 1][kTiles == 1 ? kRows : 1], sums[kTiles == 1 ? 2 : 1][kTiles == 1 ? kRows : 1];
};

struct AttnParams {
  const int* token_offsets;
  const int* lengths;
  const int* table;
  int table_width, table_stride, page_shift, page_count;
  int sequences, tokens;
  int group, kv_heads;
  int step;        // tokens of one 128-row tile: 128 / group
  int window;
  float scale_log2;
  __nv_bfloat16* out;
  long long out_token_stride, out_head_stride;
  float* partial;  // [2 * CTAs][kTiles * 128][value columns]
  float* partial_stats;  // [2 * CTAs][kTiles * 128][2]: reference (binary orders), sum
  int* records;    // [CTAs][8]
  int* status;
};

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The same for two exponents on the multiply-add units: 2^n of the nearest whole n, times the polynomial of degree four with the
// smallest largest relative error for what is left, in [-1/2, 1/2] (2.7e-6; exp2_minimax in fit_transcendentals.py), far below
// the rounding of p to bf16.  Zero below 2^-126, as from the other; what is no number stays none (2^n put into the exponent by adding
// whole numbers would make it the largest finite one).
__device__ __forceinline__ void exp2_by_polynomial(unsigned long long x, float& a, float& b) {
  constexpr float kShift = 12582912.0f;  // 1.5 * 2^23: adding it rounds to a whole number, which then stands in the low bits
  const unsigned long long t = add2(x, two(kShift, kShift));
  const unsigned long long f = fma2(add2(t, two(-kShift, -kShift)), two(-1.0f, -1.0f), x);
  unsigned long long p = fma2(two(0.009570102207362652f, 0.009570102207362652f), f, two(0.05591786280274391f, 0.05591786280274391f));
  p = fma2(p, f, two(0.240247443318367f, 0.240247443318367f));
  p = fma2(p, f, two(0.6931217908859253f, 0.6931217908859253f));
  p = fma2(p, f, two(0.9999992847442627f, 0.9999992847442627f));
  p = mul2(p, two(__uint_as_float((static_cast<uint32_t>(t) << 23) + 0x3f800000u),
                  __uint_as_float((static_cast<uint32_t>(t >> 32) << 23) + 0x3f800000u)));
  a = low_of(x) < -126.0f ? 0.0f : low_of(p);
  b = high_of(x) < -126.0f ? 0.0f : high_of(p);
}

// sum += both halves of a pair of bf16, each into its own.
__device__ __forceinline__ void add_bf16x2(float& low_sum, float& high_sum, uint32_t pair) {
  asm("{\n\t.reg .b16 low, high;\n\tmov.b32 {low, high}, %2;\n\tadd.rn.f32.bf16 %0, low, %0;\n\tadd.rn.f32.bf16 %1, high, %1;\n\t}"
      : "+f"(low_sum), "+f"(high_sum)
      : "r"(pair));
}

__device__ __forceinline__ void tma_load_4d(void* smem_dst, const void* tensor_map, uint64_t* bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(smem_dst)),
      "l"(tensor_map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

__device__ __forceinline__ void tmem_store_32x32(uint32_t tmem_address, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(tmem_address),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]),
      "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
      "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 bytes, to an address that is a multiple of that.
__device__ __forceinline__ void store_32(void* to, const uint32_t (&v)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
               "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
// D (+)= A B^T, bf16 operands, fp32 sums, K = 16; A from shared memory or from tensor memory.
__device__ __forceinline__ void mma_shared(uint32_t d, uint64_t a, uint64_t b, uint32_t descriptor, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
               "l"(a), "l"(b), "r"(descriptor), "r"(accumulate)
               : "memory");
}
__device__ __forceinline__ void mma_tensor(uint32_t d, uint32_t a, uint64_t b, uint32_t descriptor, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
               "r"(a), "l"(b), "r"(descriptor), "r"(accumulate)
               : "memory");
}

// Instruction descriptors: fp32 sums (bit 4), bf16 operands (1 at [7,10) and [10,13)), B with its rows (keys) along K instead of N for
// the values (bit 16), N at [17,23) in units of 8, M at [24,29) in units of 16.
constexpr uint32_t kIdescScores = (1u << 4) | (1u << 7) | (1u << 10) | ((kKeys >> 3) << 17) | ((kRows >> 4) << 24);
template <int kColumns>
constexpr uint32_t kIdescValues = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((kColumns >> 3) << 17) | ((kRows >> 4) << 24);

// A softmax thread holds more registers than the launch gives every thread: 168 a thread at launch, and
// 128 x 88 + 256 x 208 = 384 x 168.  (At the top of each role: that is what the compiler goes by.)
__device__ __forceinline__ void fewer_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
}
__device__ __forceinline__ void more_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
}

template <int kDim, int kTiles, bool kPaged>
__global__ void __launch_bounds__(Shape<kDim, kTiles>::kThreads, 1)
attention_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                 const __grid_constant__ CUtensorMap map_v, const AttnParams p) {
  using S = Shape<kDim, kTiles>;
  constexpr uint32_t kSlots = kSlotsOf<kTiles, kPaged>;
  using Smem = AttnSmem<kDim, kTiles>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Smem* smem = reinterpret_cast<Smem*>(smem_raw);
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(&smem->full[s], 1);
      mbar_init(&smem->empty[s], 1);
    }
    mbar_init(&smem->q_full, 1);
    mbar_init(&smem->q_empty, 1);
    for (int s = 0; s < 4; ++s) {
      mbar_init(&smem->acc_full[s], 1);
      mbar_init(&smem->p_ready[s], 4);
      mbar_init(&smem->pv_done[s], 1);
    }
    for (int t = 0; t < kTiles; ++t) mbar_init(&smem->o_free[t], 4);
    for (uint32_t s = 0; s < kSlots; ++s) {
      mbar_init(&smem->piece_full[s], 1);
      mbar_init(&smem->piece_empty[s], 2 + S::kSoftmaxWarps);  // fetching warp, MMA warp, softmax warps
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(&smem->v_landed[w], 1);
      for (int i = 0; i < 4; ++i) {
        mbar_init(&smem->reference_ready[w][i], 1);
        mbar_init(&smem->sum_ready[w][i], 1);
      }
    }
    mbar_init(&smem->next_full, 1);
    // shared memory that is not where the swizzle wants it: nothing is computed, and the status word says so
    smem->abort = (smem_u32(smem_raw) & 1023u) != 0;
    if (smem->abort && p.status) atomicExch(p.status, static_cast<int>(kCudaError));
    fence_barrier_init();
    prefetch_tensor_map(&map_q);
    prefetch_tensor_map(&map_k);
    prefetch_tensor_map(&map_v);
  }
  if (warp == 1) {
    tmem_alloc(&smem->tmem_base, 512);
    tmem_relinquish();
  }
  grid_launch_dependents();
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = smem->tmem_base;
  grid_dependency_wait();

  const int step = p.step * kTiles;  // tokens of an item
  if (warp < 4) {
  fewer_registers();  // (a warpgroup's four warps at the same place)
  if (warp == 2) {
    // ---------------- what to do next ----------------
    uint32_t count = 0;  // pieces handed out
    bool ok = true;
    const auto room = [&] {  // waits until the next piece's slot is free
      return __all_sync(0xffffffffu, wait_or_abort(&smem->piece_empty[count % kSlots], ((count / kSlots) & 1u) ^ 1u, smem, p.status));
    };
    const auto hand_out = [&](const Piece& piece) {
      if (lane == 0) {
        smem->pieces[count % kSlots] = piece;
        mbar_arrive(&smem->piece_full[count % kSlots]);
      }
      __syncwarp();
      ++count;
    };
    if constexpr (kPaged) {
      int record[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      // All sequences' work, 32 at a time, a lane each; then the sequence that this CTA's run begins in.
      const int heads = p.kv_heads * S::kHalves;
      const int capacity = p.table_width << p.page_shift;
      int lane_from = 0, lane_news = 0, lane_length = 0, loaded = -1;  // of the 32 sequences from `loaded` on
      const auto load_sequences = [&](int first) {
        if (first == loaded) return;
        loaded = first;
        lane_from = lane_news = lane_length = 0;
        if (first + lane < p.sequences) {
          lane_from = max(p.token_offsets[first + lane], 0);
          lane_news = max(min(p.token_offsets[first + lane + 1], p.tokens) - lane_from, 0);
          const int length = p.lengths[first + lane];
          if (length > capacity && blockIdx.x == 0 && p.status) atomicExch(p.status, static_cast<int>(kBadPage));
          lane_length = min(max(length, 0), capacity);
        }
      };
      const auto upto_lane = [&] {  // key tiles of one head in the loaded sequences up to the lane's
        long long upto = 0;
        if (lane_news > 0) {
          const AttnSequence q = attn_sequence(lane_news, lane_length, step);
          upto = attn_tiles_before(q, q.query_tiles, step, p.window);
        }
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
          const long long other = __shfl_up_sync(0xffffffffu, upto, d);
          if (lane >= d) upto += other;
        }
        return upto;
      };
      long long of_head = 0, upto = 0;
      for (int first = 0; first < p.sequences; first += 32) {
        load_sequences(first);
        upto = upto_lane();
        of_head += __shfl_sync(0xffffffffu, upto, 31);
      }
      // Head after head, each through all sequences: with as many runs for each head, the heads of a page are read at the same time.
      const long long work = heads * of_head;
      const int parts = attn_parts(work, static_cast<int>(gridDim.x), heads, kLeastRun);
      if (static_cast<int>(blockIdx.x) < parts) {
        const long long run_begin = attn_part_begin(work, parts, blockIdx.x), run_end = attn_part_begin(work, parts, blockIdx.x + 1);
        const int head = attn_quotient(run_begin, of_head);
        const long long in_head = run_begin - head * of_head;
        long long before = 0;
        int s = 0;
        for (; s < p.sequences; s += 32) {
          if (loaded != s) {
            load_sequences(s);
            upto = upto_lane();
          }
          const long long all = __shfl_sync(0xffffffffu, upto, 31);
          if (before + all > in_head) break;
          before += all;
        }
        const int owner = __ffs(__ballot_sync(0xffffffffu, before + upto > in_head)) - 1;
        const long long in_front = __shfl_sync(0xffffffffu, upto, (owner + 31) & 31);
        const long long offset = in_head - before - (owner > 0 ? in_front : 0);
        const long long of_first = __shfl_sync(0xffffffffu, upto, owner) - (owner > 0 ? in_front : 0);  // of the run's first sequence
        s += owner;
        int from = 0, past = 0, news = 0;
        const auto load = [&](int sequence, int* of_news, int* length) {
          load_sequences(sequence & ~31);
          from = __shfl_sync(0xffffffffu, lane_from, sequence & 31);
          news = *of_news = __shfl_sync(0xffffffffu, lane_news, sequence & 31);
          *length = __shfl_sync(0xffffffffu, lane_length, sequence & 31);
          past = *length - news;
        };
        const auto share_out = [&](const AttnShare& share) {
          const AttnSequence q = {news, past, 0};
          Piece piece;
          piece.tiles = share.take;
          piece.first_tile = attn_first_tile(q, share.tile, step, p.window) + share.skip;
          piece.query0 = from + share.tile * step;
          piece.tokens = min(step, news - share.tile * step);
          piece.position0 = past + share.tile * step;
          piece.key_origin = 0;
          piece.sequence = share.sequence;
          piece.kv_head = share.head / S::kHalves;
          piece.half = share.head % S::kHalves;
          piece.slot = share.slot;
          if (share.behind > 0) {  // what attention_join_kernel has to add up
            record[0] = share.behind;
            record[1] = piece.query0;
            record[2] = piece.tokens;
            record[3] = piece.kv_head;
            record[4] = piece.half;
          }
          if (!room()) return false;
          hand_out(piece);
          return true;
        };
        ok = attn_walk(work, parts, blockIdx.x, run_begin, run_end, heads, head, s, offset, of_first, p.sequences, step, p.window, load, share_out);
      }
      if (lane == 0) {
        int4* slot = reinterpret_cast<int4*>(p.records + 8 * static_cast<size_t>(blockIdx.x));
        slot[0] = make_int4(record[0], record[1], record[2], record[3]);
        slot[1] = make_int4(record[4], 0, 0, 0);
      }
    } else {
      const int heads = p.kv_heads * S::kHalves;
      uint32_t asked = 0;
      int item = blockIdx.x;
      for (;;) {
        // The item's sequence and query tile: rank in the list of all query tiles, each sequence's last one first.
        int rank = item / heads;
        Piece piece;
        piece.tiles = 0;
        for (int base = 0; base < p.sequences; base += 32) {
          const int s = base + lane;
          int from = 0, news = 0;
          if (s < p.sequences) {
            from = max(p.token_offsets[s], 0);
            news = max(min(p.token_offsets[s + 1], p.tokens) - from, 0);
          }
          const int mine = (news + step - 1) / step;
          int upto = mine;
#pragma unroll
          for (int d = 1; d < 32; d *= 2) {
            const int other = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= d) upto += other;
          }
          const uint32_t holds = __ballot_sync(0xffffffffu, upto > rank);
          if (holds == 0) {
            rank -= __shfl_sync(0xffffffffu, upto, 31);
            continue;
          }
          const int owner = __ffs(holds) - 1;
          rank -= __shfl_sync(0xffffffffu, upto - mine, owner);
          from = __shfl_sync(0xffffffffu, from, owner);
          news = __shfl_sync(0xffffffffu, news, owner);
          const AttnSequence q = attn_sequence(news, news, step);
          const int tile = q.query_tiles - 1 - rank;
          const int head = item % heads;
          piece.tiles = attn_tiles(q, tile, step, p.window);
          piece.first_tile = attn_first_tile(q, tile, step, p.window);
          piece.query0 = from + tile * step;
          piece.tokens = min(step, news - tile * step);
          piece.position0 = tile * step;
          piece.key_origin = from;
          piece.sequence = base + owner;
          piece.kv_head = head / S::kHalves;
          piece.half = head % S::kHalves;
          piece.slot = -1;
          break;
        }
        if (piece.tiles > 0) {
          ok = room();
          if (!ok) break;
          hand_out(piece);
        }
        // Another item is asked for once its slot is free, so that no CTA holds more than one that it does not work on.
        ok = room();
        if (!ok) break;
        if (lane == 0) {
          fence_proxy_async_smem();  // (the last answer has been read)
          mbar_arrive_expect_tx(&smem->next_full, 16);
          asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                           smem_u32(&smem->next_item)),
                       "r"(smem_u32(&smem->next_full))
                       : "memory");
        }
        __syncwarp();
        ok = __all_sync(0xffffffffu, wait_or_abort(&smem->next_full, asked & 1u, smem, p.status));
        if (!ok) {
          if (lane == 0) mbar_wait_bounded(&smem->next_full, asked & 1u, 40000000ll);  // shared memory is given up only behind the answer
          break;
        }
        ++asked;
        uint32_t granted, next;
        asm volatile(
            "{\n\t.reg .b128 answer;\n\t.reg .pred p;\n\t.reg .b32 y, z, w;\n\t"
            "ld.shared.b128 answer, [%2];\n\t"
            "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, answer;\n\t"
            "selp.u32 %0, 1, 0, p;\n\tmov.u32 %1, 0;\n\t"
            "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, y, z, w}, answer;\n\t}"
            : "=r"(granted), "=r"(next)
            : "r"(smem_u32(&smem->next_item))
            : "memory");
        __syncwarp();
        if (!granted) break;
        item = static_cast<int>(next);
      }
    }
    if (ok && room()) {
      Piece none;
      none.tiles = 0;
      none.first_tile = none.query0 = none.tokens = none.position0 = none.key_origin = none.sequence = 0;
      none.kv_head = none.half = 0;
      none.slot = -1;
      hand_out(none);
    }
  } else if (warp == 0) {
    // ---------------- operands ----------------
    uint32_t stage = 0, phase = 0, issued = 0;
    bool ok = true;
    const int page_boxes = kPaged && p.page_shift < 7 ? kKeys >> p.page_shift : 1;  // boxes of one tile's 64 columns
    const int box_rows = kKeys / page_boxes;
    const int box = lane & (page_boxes - 1), column = lane / page_boxes;
    uint32_t q_issued = 0;
    for (uint32_t count = 0;; ++count) {
      const int slot = count % kSlots;
      ok = __all_sync(0xffffffffu, wait_or_abort(&smem->piece_full[slot], (count / kSlots) & 1u, smem, p.status));
      if (!ok) break;
      const Piece piece = smem->pieces[slot];
      if (piece.tiles == 0) break;
      const int* table = kPaged ? p.table + static_cast<size_t>(piece.sequence) * p.table_stride : nullptr;
      const auto page_of = [&](int tile) {  // of this lane's box
        if constexpr (!kPaged) return 0;
        const int index = (tile * kKeys + box * box_rows) >> p.page_shift;
        return table[min(index, p.table_width - 1)];
      };
      const auto fetch = [&](const CUtensorMap* map, int x, int tile, int page) {
        ok = __all_sync(0xffffffffu, wait_or_abort(&smem->empty[stage], phase ^ 1u, smem, p.status));
        if (!ok) return;
        if (lane == 0) mbar_arrive_expect_tx(&smem->full[stage], S::kStageBytes);
        __syncwarp();
        if (column < S::kStageDim / 64) {
          uint8_t* to = smem->stage[stage] + column * kColumnBytes + box * box_rows * 128;
          const int row = kPaged ? (tile * kKeys + box * box_rows) & ((1 << p.page_shift) - 1) : piece.key_origin + tile * kKeys;
          tma_load_4d(to, map, &smem->full[stage], x + 64 * column, row, piece.kv_head, page);
        }
        __syncwarp();
        ++issued;
        if (++stage == S::kStages) {
          stage = 0;
          phase ^= 1u;
        }
      };
      const auto fetch_keys = [&](int tile, int page) {
        if (kPaged && static_cast<unsigned>(page) >= static_cast<unsigned>(p.page_count)) {
          // (read as zeros, wherever that is; reported where some row sees it)
          const Seen seen = seen_keys(piece, tile - piece.first_tile, p.window);
          if (seen.to > box * box_rows && seen.from < (box + 1) * box_rows && p.status) atomicExch(p.status, static_cast<int>(kBadPage));
        }
#pragma unroll
        for (int i = 0; i < S::kKeyStages; ++i)
          if (ok) fetch(&map_k, i * S::kStageDim, tile, page);
      };
      const auto fetch_values = [&](int tile, int page) {
#pragma unroll
        for (int i = 0; i < S::kValueStages; ++i)
          if (ok) fetch(&map_v, piece.half * S::kValueDim + i * S::kStageDim, tile, page);
      };
      int page = page_of(piece.first_tile), next_page = page_of(piece.first_tile + 1);
      ok = __all_sync(0xffffffffu, wait_or_abort(&smem->q_empty, (count & 1u) ^ 1u, smem, p.status));
      if (!ok) break;
      if (lane == 0) {
        constexpr int kBoxes = kTiles * kDim / 64;
        mbar_arrive_expect_tx(&smem->q_full, kBoxes * 128 * p.step * p.group);
#pragma unroll
        for (int i = 0; i < kBoxes; ++i) {
          const int t = i / (kDim / 64), c = i % (kDim / 64);
          tma_load_3d(smem->queries[t] + c * kColumnBytes, &map_q, &smem->q_full, 64 * c, piece.kv_head * p.group,
                      piece.query0 + t * p.step);
        }
      }
      __syncwarp();
      ++q_issued;
      constexpr bool kKeysFirst = kTiles == 1 || S::kSpare;  // K0 K1 V0 K2 V1 .., otherwise K0 V0 K1 V1 ..
      if constexpr (kKeysFirst) fetch_keys(piece.first_tile, page);
      for (int j = 0; ok && j < piece.tiles; ++j) {
        const int tile = piece.first_tile + j;
        const int page_after = page_of(tile + 2);
        if constexpr (kKeysFirst) {
          if (j + 1 < piece.tiles) fetch_keys(tile + 1, next_page);
        } else {
          fetch_keys(tile, page);
        }
        if (ok) fetch_values(tile, page);
        page = next_page;
        next_page = page_after;
      }
      if (!ok) break;
      if (lane == 0) mbar_arrive(&smem->piece_empty[slot]);
      __syncwarp();
    }
    if (!ok && lane == 0) {
      // let the copies already issued land before shared memory is given up
      const uint32_t pending = issued < static_cast<uint32_t>(S::kStages) ? issued : S::kStages;
      uint32_t s = stage, ph = phase;
      for (uint32_t i = 0; i < pending; ++i) {
        if (s == 0) {
          s = S::kStages;
          ph ^= 1u;
        }
        --s;
        mbar_wait_bounded(&smem->full[s], ph, 40000000ll);
      }
      if (q_issued) mbar_wait_bounded(&smem->q_full, (q_issued - 1) & 1u, 40000000ll);
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    if (elect_one()) {
    // The tensor pipe holds few instructions ahead, so what lies between two batches of products is time that it stands still: one wait
    // for all that a batch needs (a lane for each barrier), and few, wide products.
    const uint64_t q_desc = make_smem_desc(smem_u32(smem->queries[0]), 1024, 2);
    const uint64_t k_desc = make_smem_desc(smem_u32(smem->stage[0]), 1024, 2);
    // values: 64 columns a swizzle row, the next 64 a column block further (leading offset), keys eight rows a group (stride offset)
    const uint64_t v_desc = k_desc | (static_cast<uint64_t>(kColumnBytes >> 4) << 16);
    constexpr int kTogether = S::kStages > 3 ? 2 : 1;  // stages of a batch: of three, one has to be free for the next
    uint32_t stage = 0, phase = 0;
    bool ok = true;
    const auto skip_stages = [&](uint32_t count) {
      stage += count;
      if (stage >= S::kStages) {
        stage -= S::kStages;
        phase ^= 1u;
      }
    };
    // Waits until the next `count` stages are there, and `other`'s phase is over (null: nothing else); all are looked at before any is
    // waited for.
    const auto ready = [&](uint32_t count, uint64_t* other, uint32_t other_parity) {
      const uint32_t behind = stage + 1 == S::kStages ? 0 : stage + 1, behind_phase = stage + 1 == S::kStages ? phase ^ 1u : phase;
      const bool first = mbar_try_wait(&smem->full[stage], phase);
      const bool second = count < 2 || mbar_try_wait(&smem->full[behind], behind_phase);
      const bool third = !other || mbar_try_wait(other, other_parity);
      if (first && second && third) return true;
      return wait_or_abort(&smem->full[stage], phase, smem, p.status) &&
             (count < 2 || wait_or_abort(&smem->full[behind], behind_phase, smem, p.status)) &&
             (!other || wait_or_abort(other, other_parity, smem, p.status));
    };
    const auto wait_for = [&](uint64_t* bar, uint32_t parity) { return wait_or_abort(bar, parity, smem, p.status); };
    // The products of one stage: 128 (64) of the columns that scores sum over; or of the outputs' columns, of one stage or of two that
    // lie side by side.
    const auto scores_of_stage = [&](uint32_t d, int tile, int part) {
      const uint64_t b = k_desc + stage * (S::kStageBytes >> 4);
#pragma unroll
      for (int i = 0; i < S::kStageDim / 16; ++i) {
        const uint32_t at = (i / 4) * kColumnBytes + (i % 4) * 32;
        mma_shared(d, q_desc + ((tile * S::kQueryTileBytes + part * 2 * kColumnBytes + at) >> 4), b + (at >> 4), kIdescScores,
                   part > 0 || i > 0 ? 1u : 0u);
      }
    };
    const auto values_of_stage = [&](uint32_t d, uint32_t at_stage, uint32_t a, uint32_t accumulate, uint32_t descriptor) {
      const uint64_t b = v_desc + at_stage * (S::kStageBytes >> 4);
#pragma unroll
      for (int i = 0; i < kKeys / 16; ++i) mma_tensor(d, a + 8 * i, b + ((i * 2048) >> 4), descriptor, i > 0 ? 1u : accumulate);
    };
    uint32_t done = 0;    // key tiles of the pieces before
    bool scored = false;  // the piece's first scores have been asked for at the end of the one before
    for (uint32_t count = 0; ok; ++count) {
      const int slot = count % kSlots;
      ok = wait_for(&smem->piece_full[slot], (count / kSlots) & 1u);
      if (!ok) break;
      const Piece piece = smem->pieces[slot];
      const int tiles = piece.tiles;
      if (tiles == 0) break;
      if (!scored) ok = wait_for(&smem->q_full, count & 1u);
      if (!ok) break;
      if constexpr (kTiles == 1) {
        // Of key tile n, the piece's last one or not: its queries may be replaced behind the last one's.
        const auto scores = [&](uint32_t n, bool last) {
#pragma unroll
          for (int i = 0; i < S::kKeyStages; i += kTogether) {
            constexpr int kBatch = kTogether < S::kKeyStages ? kTogether : S::kKeyStages;
            ok = ok && ready(kBatch, nullptr, 0);
            if (!ok) break;
#pragma unroll
            for (int k = 0; k < kBatch; ++k) {
              {
                scores_of_stage(tmem_base + (n & 1u) * kKeys, 0, i + k);
                tc_commit(&smem->empty[stage]);
                if (i + k + 1 == S::kKeyStages) {
                  tc_commit(&smem->acc_full[n & 1u]);
                  if (last) tc_commit(&smem->q_empty);
                }
              }
              skip_stages(1);
            }
          }
        };
        if (!scored) scores(done, tiles == 1);
        scored = false;
        for (int j = 0; ok && j < tiles; ++j) {
          const uint32_t n = done + j;
          if (j + 1 < tiles) scores(n + 1, j + 2 == tiles);
          if (j == 0) ok = ok && wait_for(&smem->o_free[0], (count & 1u) ^ 1u);
          if (ok && !seen_keys(piece, j, p.window).all()) {
            // the softmax warps clear rows of these values before they say that P is there
            ok = ready(S::kValueStages, nullptr, 0);
            if (ok) mbar_arrive(&smem->v_landed[n & 1u]);
          }
          if (S::kAhead && ok && j + 1 == tiles) {
            // While the last softmax runs: the first scores of the next piece, if its operands are there before P is.
            const uint32_t value_stage = stage, value_phase = phase;
            const int next_slot = (count + 1) % kSlots;
            const uint32_t next_parity = ((count + 1) / kSlots) & 1u;
            const long long start = clock64();
            skip_stages(S::kValueStages);
            while (!scored && !mbar_try_wait(&smem->p_ready[n & 1u], (n >> 1) & 1u)) {
              if (mbar_try_wait(&smem->piece_full[next_slot], next_parity) && smem->pieces[next_slot].tiles > 0 &&
                  mbar_try_wait(&smem->q_full, (count + 1) & 1u)) {
                bool there = true;
                uint32_t s = stage, parity = phase;
                for (int i = 0; i < S::kKeyStages; ++i) {
                  there = there && mbar_try_wait(&smem->full[s], parity);
                  if (++s == S::kStages) {
                    s = 0;
                    parity ^= 1u;
                  }
                }
                if (there) {
                  scores(n + 1, smem->pieces[next_slot].tiles == 1);
                  scored = true;
                }
              }
              // (the wait below says that P does not come; this loop only has to end)
              if (smem->abort || clock64() - start > kWaitLimitCycles) break;
            }
            stage = value_stage;
            phase = value_phase;
          }
          constexpr int kBatch = kTogether < S::kValueStages ? kTogether : S::kValueStages;
          ok = ok && ready(kBatch, &smem->p_ready[n & 1u], (n >> 1) & 1u);
          if (!ok) break;
          tc_fence_after_sync();
          const uint32_t weights = tmem_base + (n & 1u) * kKeys, accumulate = j > 0 ? 1u : 0u;
          if (kBatch == 2 && stage + 1 < S::kStages) {
            {
              values_of_stage(tmem_base + 256, stage, weights, accumulate, kIdescValues<2 * S::kStageDim>);
              tc_commit(&smem->empty[stage]);
              tc_commit(&smem->empty[stage + 1]);
              tc_commit(&smem->pv_done[n & 1u]);
            }
            skip_stages(2);
          } else {
#pragma unroll
            for (int i = 0; i < S::kValueStages; ++i) {
              if (i >= kBatch) ok = ok && ready(1, nullptr, 0);
              if (!ok) break;
              {
                values_of_stage(tmem_base + 256 + i * S::kStageDim, stage, weights, accumulate, kIdescValues<S::kStageDim>);
                tc_commit(&smem->empty[stage]);
                if (i + 1 == S::kValueStages) tc_commit(&smem->pv_done[n & 1u]);
              }
              skip_stages(1);
            }
            if (!ok) break;
          }
          if (scored) skip_stages(S::kKeyStages);  // the next piece's keys stand behind these values, and have been used
        }
      } else if constexpr (S::kSpare) {
        // Score tiles are free again behind the products that read their P: the second query tile's next scores follow the first one's
        // outputs, the first one's next but one the second one's.
        const uint32_t ring = 2 * done;  // stages of the pieces before
        const auto stage_at = [&](uint32_t at) {
          stage = (ring + at) % S::kStages;
          phase = ((ring + at) / S::kStages) & 1u;
        };
        const auto keys_at = [&](uint32_t j) { stage_at(j > 0 ? 2 * j - 1 : 0); };
        const auto scores = [&](uint32_t j, int t) {  // (the keys are there)
          const uint32_t n = done + j;
          scores_of_stage(tmem_base + (2 * n + t) % 3 * kKeys, t, 0);
          tc_commit(&smem->acc_full[2 * t + (n & 1u)]);
          if (t == 1) tc_commit(&smem->empty[stage]);
        };
        keys_at(0);
        ok = ready(1, nullptr, 0);
        if (!ok) break;
        scores(0, 0);
        scores(0, 1);
        if (tiles > 1) {
          keys_at(1);
          ok = ready(1, nullptr, 0);
          if (!ok) break;
          scores(1, 0);
        }
        for (int j = 0; ok && j < tiles; ++j) {
          const uint32_t n = done + j;
          const uint32_t accumulate = j > 0 ? 1u : 0u;
          if (j == 0) ok = wait_for(&smem->o_free[0], (count & 1u) ^ 1u) && wait_for(&smem->o_free[1], (count & 1u) ^ 1u);
          stage_at(min(j + 2, tiles) + j);
          const uint32_t value_stage = stage;
          if (ok && !seen_keys(piece, j, p.window).all()) {
            ok = ready(1, nullptr, 0);
            if (ok) mbar_arrive(&smem->v_landed[0]);
          }
          ok = ok && ready(1, &smem->p_ready[n & 1u], (n >> 1) & 1u);
          if (!ok) break;
          tc_fence_after_sync();
          values_of_stage(tmem_base + S::kOutputs, value_stage, tmem_base + 2 * n % 3 * kKeys, accumulate, kIdescValues<S::kStageDim>);
          tc_commit(&smem->pv_done[n & 1u]);
          if (j + 1 < tiles) {
            keys_at(j + 1);
            scores(j + 1, 1);
          }
          if (j + 2 < tiles) keys_at(j + 2);
          ok = j + 2 < tiles ? ready(1, &smem->p_ready[2 + (n & 1u)], (n >> 1) & 1u)
                             : wait_for(&smem->p_ready[2 + (n & 1u)], (n >> 1) & 1u);
          if (!ok) break;
          tc_fence_after_sync();
          values_of_stage(tmem_base + S::kOutputs + kDim, value_stage, tmem_base + (2 * n + 1) % 3 * kKeys, accumulate,
                          kIdescValues<S::kStageDim>);
          tc_commit(&smem->pv_done[2 + (n & 1u)]);
          tc_commit(&smem->empty[value_stage]);
          if (j + 2 < tiles) scores(j + 2, 0);
          if (j + 2 == tiles || tiles == 1) tc_commit(&smem->q_empty);
        }
      } else {
        // one stage holds a tile's keys, another its values
        ok = ready(1, nullptr, 0);
        if (!ok) break;
        {
#pragma unroll
          for (int t = 0; t < kTiles; ++t) {
            scores_of_stage(tmem_base + t * kKeys, t, 0);
            tc_commit(&smem->acc_full[t]);
          }
          tc_commit(&smem->empty[stage]);
        }
        skip_stages(1);
        for (int j = 0; ok && j < tiles; ++j) {
          const uint32_t n = done + j;
          const uint32_t accumulate = j > 0 ? 1u : 0u;
          const bool more = j + 1 < tiles;
          if (j == 0) ok = wait_for(&smem->o_free[0], (count & 1u) ^ 1u) && wait_for(&smem->o_free[1], (count & 1u) ^ 1u);
          if (ok && !seen_keys(piece, j, p.window).all()) {
            ok = ready(1, nullptr, 0);
            if (ok) mbar_arrive(&smem->v_landed[0]);
          }
          // P of the first tile, the values and the next keys; then P of the second
          ok = ok && ready(more ? 2 : 1, &smem->p_ready[0], n & 1u);
          if (!ok) break;
          tc_fence_after_sync();
          const uint32_t value_stage = stage;
          skip_stages(1);
          {
            values_of_stage(tmem_base + 256, value_stage, tmem_base, accumulate, kIdescValues<S::kStageDim>);
            tc_commit(&smem->pv_done[0]);
            if (more) {
              scores_of_stage(tmem_base, 0, 0);
              tc_commit(&smem->acc_full[0]);
            }
          }
          ok = wait_for(&smem->p_ready[1], n & 1u);
          if (!ok) break;
          tc_fence_after_sync();
          {
            values_of_stage(tmem_base + 256 + kDim, value_stage, tmem_base + kKeys, accumulate, kIdescValues<S::kStageDim>);
            tc_commit(&smem->pv_done[1]);
            tc_commit(&smem->empty[value_stage]);
            if (more) {
              scores_of_stage(tmem_base + kKeys, 1, 0);
              tc_commit(&smem->acc_full[1]);
              tc_commit(&smem->empty[stage]);
            } else {
              tc_commit(&smem->q_empty);
            }
          }
          if (more) skip_stages(1);
        }
      }
      done += tiles;
      if (ok) mbar_arrive(&smem->piece_empty[slot]);
    }
    }
    __syncwarp();
  }
  } else {
    // ---------------- softmax and epilogue ----------------
    more_registers();
    // This warpgroup's query tile; or, of the one query tile there is, the key tiles that are its turn: those whose scores stand in its
    // half of the score columns.
    const int own = (warp - 4) / 4;
    const int tile_of_rows = kTiles == 2 ? own : 0;
    const int quarter = warp & 3;              // the tensor-memory lanes this warp may read
    const int row = quarter * 32 + lane;
    const int row_token = row / p.group, row_head = row - row_token * p.group;
    const uint32_t lanes = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t outputs = lanes + S::kOutputs + tile_of_rows * kDim;
    const float c = p.scale_log2;
    uint32_t done = 0, ring = 0;  // key tiles and operand stages of the pieces before
    uint32_t cleared = 0;         // tiles with values that this warpgroup has cleared
    bool ok = true;
    for (uint32_t count = 0; ok; ++count) {
      const int slot = count % kSlots;
      ok = __all_sync(0xffffffffu, wait_or_abort(&smem->piece_full[slot], (count / kSlots) & 1u, smem, p.status));
      if (!ok) break;
      const Piece piece = smem->pieces[slot];
      if (piece.tiles == 0) break;
      const int token = tile_of_rows * p.step + row_token;
      const bool valid = row_token < p.step && token < piece.tokens;
      // keys that the row sees: [row_begin, row_end)
      const int position = piece.position0 + token;
      const int row_end = valid && position >= 0 ? position + 1 : 0;
      const int row_begin = p.window > 0 && position - p.window + 1 > 0 ? position - p.window + 1 : 0;
      const bool active = __any_sync(0xffffffffu, valid);
      const int least_end = __reduce_min_sync(0xffffffffu, valid ? row_end : 0x7fffffff);
      const int most_begin = __reduce_max_sync(0xffffffffu, valid ? row_begin : 0);
      float reference = -CUDART_INF_F, sum = 0.0f;
      const int first = kTiles == 2 ? 0 : static_cast<int>((done & 1u) ^ static_cast<uint32_t>(own));
#pragma unroll 1
      for (int j = first; j < piece.tiles; j += kTiles == 2 ? 1 : 2) {
        const uint32_t n = done + j;
        const uint32_t scores = lanes + (S::kSpare ? (2 * n + own) % 3 : own) * kKeys;
        const uint32_t barrier = S::kSpare ? 2 * own + (n & 1u) : own;
        const uint32_t turn = kTiles == 2 && !S::kSpare ? n : n >> 1;  // of that barrier
        ok = __all_sync(0xffffffffu, wait_or_abort(&smem->acc_full[barrier], turn & 1u, smem, p.status));
        if (!ok) break;
        tc_fence_after_sync();
        const int key0 = (piece.first_tile + j) * kKeys;
        float factor = 1.0f, tile_sum = 0.0f;
        const uint32_t turn_before = ((n - 1) >> 1) & 1u;  // of the other warpgroup, for the tile before
        if (!active && kTiles == 1) {
          if (n > 0) ok = __all_sync(0xffffffffu, wait_or_abort(&smem->reference_ready[own ^ 1][quarter], turn_before, smem, p.status));
          if (!ok) break;
          if (lane == 0) mbar_arrive(&smem->reference_ready[own][quarter]);
        }
        if (active) {
          uint32_t s0[32], s1[32], s2[32], s3[32];
          tmem_load_32x32(scores, s0);
          tmem_load_32x32(scores + 32, s1);
          tmem_load_32x32(scores + 64, s2);
          tmem_load_32x32(scores + 96, s3);
          tmem_load_wait(s0, s1, s2, s3);
          if (key0 + kKeys > least_end || key0 < most_begin) {
            const int from = row_begin - key0, to = row_end - key0;
            const auto hide = [&](uint32_t (&s)[32], int base) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (base + i < from || base + i >= to) s[i] = 0xff800000u;  // -inf
            };
            hide(s0, 0);
            hide(s1, 32);
            hide(s2, 64);
            hide(s3, 96);
          }
          float top0 = -CUDART_INF_F, top1 = top0, top2 = top0, top3 = top0;
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            top0 = fmaxf(top0, __uint_as_float(s0[i]));
            top1 = fmaxf(top1, __uint_as_float(s1[i]));
            top2 = fmaxf(top2, __uint_as_float(s2[i]));
            top3 = fmaxf(top3, __uint_as_float(s3[i]));
          }
          const float top = fmaxf(fmaxf(top0, top1), fmaxf(top2, top3));
          if constexpr (kTiles == 1) {
            // (waited for at a piece's first tile too: then nothing is read, but what this warp writes next has been read)
            if (n > 0) ok = __all_sync(0xffffffffu, wait_or_abort(&smem->reference_ready[own ^ 1][quarter], turn_before, smem, p.status));
            if (!ok) break;
            reference = j > 0 ? smem->references[own ^ 1][row] : -CUDART_INF_F;
          }
          // (false where nothing has been seen yet: the difference of two infinities is no number)
          const bool grow = (top - reference) * c > kGrowth;
          const bool any_grow = __any_sync(0xffffffffu, grow);
          if (grow) {
            factor = exp2_approx((reference - top) * c);
            reference = top;
          }
          if constexpr (kTiles == 1) {
            smem->references[own][row] = reference;
            __syncwarp();
            if (lane == 0) mbar_arrive(&smem->reference_ready[own][quarter]);
          }
          if (any_grow && j > 0) {
            // (A wait can tell a phase from the one before it, not from the one after the next: each of these barriers is one phase
            // behind at most, since the scores at hand were asked for behind the outputs of two tiles before, and one ahead at most.)
            const uint32_t before = kTiles == 2 && !S::kSpare ? n - 1 : (n - 1) >> 1;
            const uint32_t summed = S::kSpare ? 2 * own + ((n - 1) & 1u) : kTiles == 2 ? own : own ^ 1;
            ok = __all_sync(0xffffffffu, wait_or_abort(&smem->pv_done[summed], before & 1u, smem, p.status));
            if (!ok) break;
            tc_fence_after_sync();
#pragma unroll 1
            for (int i = 0; i < S::kValueDim; i += 32) {
              uint32_t o[32];
              tmem_load_32x32(outputs + i, o);
              tmem_load_wait(o);
#pragma unroll
              for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * factor);
              tmem_store_32x32(outputs + i, o);
            }
          }
          const float shift = reference == -CUDART_INF_F ? 0.0f : -reference * c;
          const unsigned long long c2 = two(c, c), shift2 = two(shift, shift);
          float low_sum = 0.0f, high_sum = 0.0f;
          uint32_t packed[32];
          const auto exponentials = [&](const uint32_t (&s)[32], int first) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const unsigned long long v = fma2(two(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), c2, shift2);
              float a, b;
              // Heads of 64: the exponentials of two query tiles take twice as long as their products; one of eight by the other units, of
              // more the instructions cost more than they spare (8192 tokens, 32 heads: none 335 us, one 326, two 338, four 392; heads of
              // 128, a quarter: 451 and 452).
              if (kTiles == 2 && kDim == 64 && (i % 8 == 3)) {
                exp2_by_polynomial(v, a, b);
              } else {
                a = exp2_approx(low_of(v));
                b = exp2_approx(high_of(v));
              }
              // (the sums of the unrounded values, in pairs, took 1 % less: 8192 tokens, heads of 64 336 and 339 us, 8191 of 128 452 and 454,
              // 4608 of 512 360 and 365; unpacked by shifts 369, 468 and 368)
              packed[first + i] = pack_bf16x2(a, b);
              add_bf16x2(low_sum, high_sum, packed[first + i]);
            }
          };
          exponentials(s0, 0);
          exponentials(s1, 16);
          tmem_store_32x32(scores, packed);
          exponentials(s2, 0);
          exponentials(s3, 16);
          tmem_store_32x32(scores + 32, packed);
          tile_sum = low_sum + high_sum;
          tmem_store_wait();
        }
        tc_fence_before_sync();
        const Seen seen = seen_keys(piece, j, p.window);
        if ((kTiles == 1 || own == 0) && !seen.all()) {
          // (the MMA warp says when they have landed: these threads do not follow the stages' phases)
          ok = __all_sync(0xffffffffu, wait_or_abort(&smem->v_landed[own], cleared & 1u, smem, p.status));
          if (!ok) break;
          ++cleared;
          const uint32_t at = ring + (kTiles == 2 && !S::kSpare ? j * (S::kKeyStages + S::kValueStages) + S::kKeyStages
                                                  : min(j + 2, piece.tiles) * S::kKeyStages + j * S::kValueStages);
          if (row < seen.from || row >= seen.to)
            for (int i = 0; i < S::kValueStages; ++i)
              for (int x = 0; x < S::kStageDim / 64; ++x)
#pragma unroll
                for (int y = 0; y < 8; ++y)  // (a row of the tile is 128 bytes in a row, whatever the swizzle does within them)
                  *reinterpret_cast<uint4*>(smem->stage[(at + i) % S::kStages] + x * kColumnBytes + row * 128 + ((y ^ (row & 7)) << 4)) =
                      make_uint4(0, 0, 0, 0);
          fence_proxy_async_smem();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&smem->p_ready[barrier]);
        if constexpr (kTiles == 1) {
          if (n > 0) ok = __all_sync(0xffffffffu, wait_or_abort(&smem->sum_ready[own ^ 1][quarter], turn_before, smem, p.status));
          if (!ok) break;
          sum = j > 0 ? fmaf(smem->sums[own ^ 1][row], factor, tile_sum) : tile_sum;
          smem->sums[own][row] = sum;
          __syncwarp();
          if (lane == 0) mbar_arrive(&smem->sum_ready[own][quarter]);
        } else {
          sum = fmaf(sum, factor, tile_sum);
        }
      }
      if (!ok) break;
      const bool finishes = kTiles == 2 || ((done + piece.tiles - 1) & 1u) == static_cast<uint32_t>(own);
      done += piece.tiles;
      ring += piece.tiles * (S::kKeyStages + S::kValueStages);
      if (!finishes) {  // the other warpgroup has the last tile, and so the outputs
        if (lane == 0) mbar_arrive(&smem->piece_empty[slot]);
        continue;
      }
      const uint32_t summed = S::kSpare ? 2 * own + ((done - 1) & 1u) : own;
      const uint32_t sums_before = kTiles == 2 && !S::kSpare ? done - 1 : (done - 1) >> 1;
      ok = __all_sync(0xffffffffu, wait_or_abort(&smem->pv_done[summed], sums_before & 1u, smem, p.status));
      if (!ok) break;
      tc_fence_after_sync();
      if (active) {
        const float inverse = sum != 0.0f ? 1.0f / sum : 0.0f;  // a row that sees nothing: zeros
        const int column0 = piece.half * S::kValueDim;
        __nv_bfloat16* out = p.out + static_cast<long long>(piece.query0 + token) * p.out_token_stride +
                             static_cast<long long>(piece.kv_head * p.group + row_head) * p.out_head_stride + column0;
        const size_t partial_row = (static_cast<size_t>(piece.slot < 0 ? 0 : piece.slot) * kTiles + tile_of_rows) * kRows + row;
        // A store of a row per lane keeps the store unit busy for 32 lines whatever it stores.  So lanes work in pairs: each has 64 bytes
        // of a row, and they store first the one's, then the other's, 32 bytes each.
        const bool odd = lane & 1;
        __nv_bfloat16* other_out =
            reinterpret_cast<__nv_bfloat16*>(__shfl_xor_sync(0xffffffffu, reinterpret_cast<unsigned long long>(out), 1));
        const bool other_valid = __shfl_xor_sync(0xffffffffu, valid ? 1 : 0, 1) != 0;
        __nv_bfloat16* const first_out = odd ? other_out + 16 : out;
        __nv_bfloat16* const second_out = odd ? out + 16 : other_out;
        const bool first_valid = odd ? other_valid : valid, second_valid = odd ? valid : other_valid;
        const auto finish = [&](const uint32_t (&o)[32], int i) {
          if (piece.slot < 0) {
            uint32_t mine[16], theirs[8];
#pragma unroll
            for (int k = 0; k < 16; ++k)
              mine[k] = pack_bf16x2(__uint_as_float(o[2 * k]) * inverse, __uint_as_float(o[2 * k + 1]) * inverse);
#pragma unroll
            for (int k = 0; k < 8; ++k) theirs[k] = __shfl_xor_sync(0xffffffffu, odd ? mine[k] : mine[8 + k], 1);
            uint32_t first[8], second[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              first[k] = odd ? theirs[k] : mine[k];
              second[k] = odd ? mine[8 + k] : theirs[k];
            }
            if (first_valid) store_32(first_out + i, first);
            if (second_valid) store_32(second_out + i, second);
          } else if (valid) {
            float* to = p.partial + partial_row * S::kValueDim + i;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t v[8] = {o[8 * k],     o[8 * k + 1], o[8 * k + 2], o[8 * k + 3],
                                     o[8 * k + 4], o[8 * k + 5], o[8 * k + 6], o[8 * k + 7]};
              store_32(to + 8 * k, v);
            }
          }
          __syncwarp();
        };
#pragma unroll 1
        for (int i = 0; i < S::kValueDim; i += 64) {
          uint32_t o0[32], o1[32];
          tmem_load_32x32(outputs + i, o0);
          tmem_load_32x32(outputs + i + 32, o1);
          tmem_load_wait(o0, o1);
          finish(o0, i);
          finish(o1, i + 32);
        }
        if (valid && piece.slot >= 0) {
          float2* stats = reinterpret_cast<float2*>(p.partial_stats) + partial_row;
          *stats = make_float2(reference == -CUDART_INF_F ? -CUDART_INF_F : reference * c, sum);
        }
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&smem->o_free[tile_of_rows]);
        mbar_arrive(&smem->piece_empty[slot]);
      }
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    __syncwarp();
    tmem_dealloc(tmem_base, 512);
  }
}

// Adds up the sums of the items that the ends of runs have cut: CTA x takes the item that begins in run x and does not end there, its
// rows dealt out over the warps of gridDim.y CTAs.  Bound by latency: the record says where the parts are, and what of them is asked for,
// four at a time, waits for nothing else.
template <int kValueDim>
__global__ void __launch_bounds__(256) attention_join_kernel(const AttnParams p, int tiles) {
  grid_dependency_wait();
  const int4 first = *reinterpret_cast<const int4*>(p.records + 8 * static_cast<size_t>(blockIdx.x));
  const int half = p.records[8 * static_cast<size_t>(blockIdx.x) + 4];
  const int parts = first.x + 1;
  if (parts == 1) return;
  const int lane = threadIdx.x & 31;
  const int query0 = first.y, tokens = first.z, kv_head = first.w;
  const size_t slot_rows = static_cast<size_t>(tiles) * kRows;
  const auto row_of = [&](int part) {  // first row of the item's part
    return static_cast<size_t>(2 * (static_cast<int>(blockIdx.x) + part) + (part == 0 ? 1 : 0)) * slot_rows;
  };
  const int rows = tokens * p.group;
  constexpr int kEach = kValueDim / 32, kVector = kEach < 4 ? kEach : 4, kVectors = kEach / kVector;
  for (int r = blockIdx.y * 8 + (threadIdx.x >> 5); r < rows; r += gridDim.y * 8) {
    const int token = r / p.group, head = r - token * p.group;
    const int row = (token / p.step) * kRows + (token % p.step) * p.group + head;
    float top = -CUDART_INF_F, sum = 0.0f, acc[kEach] = {};
    for (int part = 0; part < parts; part += 4) {
      float2 stats[4];
      float v[4][kEach];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const size_t at = row_of(min(part + i, parts - 1)) + row;
        stats[i] = reinterpret_cast<const float2*>(p.partial_stats)[at];
        if (part + i >= parts) stats[i] = make_float2(-CUDART_INF_F, 0.0f);
        const float* from = p.partial + at * kValueDim;
#pragma unroll
        for (int k = 0; k < kVectors; ++k) {
          if constexpr (kVector == 2) {
            const float2 x = reinterpret_cast<const float2*>(from)[lane];
            v[i][0] = x.x;
            v[i][1] = x.y;
          } else {
            const float4 x = reinterpret_cast<const float4*>(from)[k * 32 + lane];
            v[i][4 * k] = x.x;
            v[i][4 * k + 1] = x.y;
            v[i][4 * k + 2] = x.z;
            v[i][4 * k + 3] = x.w;
          }
        }
      }
      const float now = fmaxf(fmaxf(fmaxf(stats[0].x, stats[1].x), fmaxf(stats[2].x, stats[3].x)), top);
      const float shift = now == -CUDART_INF_F ? 0.0f : now;  // (nothing seen: every weight is zero)
      const float keep = exp2_approx(top - shift);
      sum *= keep;
#pragma unroll
      for (int k = 0; k < kEach; ++k) acc[k] *= keep;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float weight = exp2_approx(stats[i].x - shift);
        sum = fmaf(stats[i].y, weight, sum);
        // (a part that is not there, or has seen nothing, adds nothing, whatever its sums hold)
#pragma unroll
        for (int k = 0; k < kEach; ++k) acc[k] = weight > 0.0f || weight != weight ? fmaf(v[i][k], weight, acc[k]) : acc[k];
      }
      top = now;
    }
    const float inverse = sum != 0.0f ? 1.0f / sum : 0.0f;
    __nv_bfloat16* out = p.out + static_cast<long long>(query0 + token) * p.out_token_stride +
                         static_cast<long long>(kv_head * p.group + head) * p.out_head_stride + half * kValueDim;
#pragma unroll
    for (int k = 0; k < kVectors; ++k) {
      if constexpr (kVector == 2)
        reinterpret_cast<uint32_t*>(out)[lane] = pack_bf16x2(acc[0] * inverse, acc[1] * inverse);
      else
        reinterpret_cast<uint2*>(out)[k * 32 + lane] = make_uint2(pack_bf16x2(acc[4 * k] * inverse, acc[4 * k + 1] * inverse),
                                                                  pack_bf16x2(acc[4 * k + 2] * inverse, acc[4 * k + 3] * inverse));
    }
  }
}

constexpr int kJoinColumns = 8;  // CTAs that share an item's rows

bool make_map(CUtensorMap* map, const void* base, int rank, const uint64_t* dims, const long long* strides, const uint32_t* box) {
  uint64_t bytes[3];
  for (int i = 0; i + 1 < rank; ++i) bytes[i] = static_cast<uint64_t>(strides[i]) * 2;
  return make_bf16_tensor_map(map, base, rank, dims, bytes, box);
}

template <int kDim, int kTiles, bool kPaged>
cudaError_t launch_shape(const AttnCall& call, cudaStream_t stream) {
  using S = Shape<kDim, kTiles>;
  const auto kernel = attention_kernel<kDim, kTiles, kPaged>;
  constexpr int kSmemBytes = static_cast<int>(sizeof(AttnSmem<kDim, kTiles>));
  static_assert(kSmemBytes <= 232448, "shared memory of an SM");
  static bool prepared[64] = {};
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  if (device < 0 || device >= 64 || !prepared[device]) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
    if (e != cudaSuccess) return e;
    if (device >= 0 && device < 64) prepared[device] = true;
  }
  const int group = call.heads / call.kv_heads;
  AttnParams p{};
  p.token_offsets = call.token_offsets;
  p.sequences = call.sequences;
  p.tokens = call.tokens;
  p.group = group;
  p.kv_heads = call.kv_heads;
  p.step = kRows / group;
  p.window = call.window;
  p.scale_log2 = call.scale * 1.4426950408889634f;
  p.out = static_cast<__nv_bfloat16*>(call.out);
  p.out_token_stride = call.out_token_stride;
  p.out_head_stride = call.out_head_stride;
  p.status = call.status;
  CUtensorMap map_q, map_k, map_v;
  {
    const uint64_t dims[3] = {kDim, static_cast<uint64_t>(call.heads), static_cast<uint64_t>(call.tokens)};
    const long long strides[2] = {call.q.head_stride, call.q.token_stride};
    const uint32_t box[3] = {64, static_cast<uint32_t>(group), static_cast<uint32_t>(p.step)};
    if (!make_map(&map_q, call.q.data, 3, dims, strides, box)) return cudaErrorInvalidValue;
  }
  long long items;
  if constexpr (kPaged) {
    const AttnPages& c = call.pages;
    p.lengths = c.lengths;
    p.table = c.table;
    p.table_width = c.table_width;
    p.table_stride = c.table_stride;
    p.page_count = c.page_count;
    while ((1 << p.page_shift) < c.page_size) ++p.page_shift;
    const uint64_t dims[4] = {kDim, static_cast<uint64_t>(c.page_size), static_cast<uint64_t>(call.kv_heads),
                              static_cast<uint64_t>(c.page_count)};
    const uint32_t box[4] = {64, static_cast<uint32_t>(c.page_size < kKeys ? c.page_size : kKeys), 1, 1};
    const long long key_strides[3] = {c.key_slot_stride, c.key_head_stride, c.key_page_stride};
    const long long value_strides[3] = {c.value_slot_stride, c.value_head_stride, c.value_page_stride};
    if (!make_map(&map_k, c.keys, 4, dims, key_strides, box) || !make_map(&map_v, c.values, 4, dims, value_strides, box))
      return cudaErrorInvalidValue;
    items = call.sm_count;
    const size_t rows = 2 * static_cast<size_t>(call.sm_count) * kTiles * kRows;
    p.partial = static_cast<float*>(call.workspace);
    p.partial_stats = p.partial + rows * S::kValueDim;
    p.records = reinterpret_cast<int*>(p.partial_stats + 2 * rows);
  } else {
    const uint64_t dims[4] = {kDim, static_cast<uint64_t>(call.tokens), static_cast<uint64_t>(call.kv_heads), 1};
    const uint32_t box[4] = {64, kKeys, 1, 1};
    const long long key_strides[3] = {call.k.token_stride, call.k.head_stride, kDim};  // (the last is of one page that there is)
    const long long value_strides[3] = {call.v.token_stride, call.v.head_stride, kDim};
    if (!make_map(&map_k, call.k.data, 4, dims, key_strides, box) || !make_map(&map_v, call.v.data, 4, dims, value_strides, box))
      return cudaErrorInvalidValue;
    // as many query tiles as sequences of any lengths can have
    const long long step = static_cast<long long>(p.step) * kTiles;
    items = (call.tokens + call.sequences * (step - 1)) / step * call.kv_heads * S::kHalves;
    if (items > 0x7fffffff) return cudaErrorInvalidConfiguration;
  }
  e = launch_chained(kernel, dim3(static_cast<unsigned>(items)), dim3(S::kThreads), kSmemBytes, stream, map_q, map_k, map_v, p);
  if (e != cudaSuccess) return e;
  if constexpr (kPaged)
    e = launch_chained(attention_join_kernel<S::kValueDim>, dim3(static_cast<unsigned>(items), kJoinColumns), dim3(256), 0, stream, p,
                       kTiles);
  return e;
}

}  // namespace

size_t attention_workspace_bytes(int dim, int sm_count) {
  const size_t tiles = dim <= 128 ? 2 : 1;
  const size_t rows = 2 * static_cast<size_t>(sm_count) * tiles * kRows;
  return rows * ((dim < 256 ? dim : 256) + 2) * sizeof(float) + static_cast<size_t>(sm_count) * 8 * sizeof(int);
}

cudaError_t launch_attention(const AttnCall& call, cudaStream_t stream) {
  // Two query tiles where there are rows for them: below, half of the products and exponentials would be of rows that do not exist.
  const long long rows = static_cast<long long>(call.tokens) * (call.heads / call.kv_heads);
  const bool two_tiles = rows > static_cast<long long>(call.sequences) * kRows;
  if (call.paged) {
    switch (call.dim) {
      case 64: return two_tiles ? launch_shape<64, 2, true>(call, stream) : launch_shape<64, 1, true>(call, stream);
      case 128: return two_tiles ? launch_shape<128, 2, true>(call, stream) : launch_shape<128, 1, true>(call, stream);
      case 256: return launch_shape<256, 1, true>(call, stream);
      default: return launch_shape<512, 1, true>(call, stream);
    }
  }
  switch (call.dim) {
    case 64: return two_tiles ? launch_shape<64, 2, false>(call, stream) : launch_shape<64, 1, false>(call, stream);
    case 128: return two_tiles ? launch_shape<128, 2, false>(call, stream) : launch_shape<128, 1, false>(call, stream);
    case 256: return launch_shape<256, 1, false>(call, stream);
    default: return launch_shape<512, 1, false>(call, stream);
  }
}

}  // namespace gv
