// Tokens from logits (declared in include/gevva_moe.h): temperature, top-k, top-p and min-p, from one given random number a row.
//
// With y = x, or cap * tanh(x / cap), a token's share is w = exp((y - y_max) / T).  Tokens are ranked by x, ties by index; kept are the ranks below
// top_k, those whose better ranks have less than top_p of what top_k leaves, and those with w >= min_p.  The token is the first of the
// vocabulary at which the sum of kept shares passes u times the sum of all kept ones.
//
// A row is gone through a few times, by a CTA or a cluster of up to 16, from HBM first and from L2 afterwards:
//   1. the largest value, and for groups of threads of every size the smallest of their largest values: with at least k groups, at least k
//      values are not below that, and with about k groups only some k ln k are.  Those go to a list.
//   2. where top_p has to cut a whole row, or a large top_k: how many values lie in each of 1024 bins, and the shares' sum in 32 bits.  From these
//      the border is known to a few bins.
//   3. all shares in 64 bits, their sum and that of those above the border's bins; what lies in the bins goes to the list.  Sorted, it tells the border
//      exactly; a border that is not there (the counts told wrong, or too many values in the bins) is looked for closer, at last by halving.
//   4. the kept shares are summed by CTAs, warps and pieces of a warp in the order of the vocabulary, down to the piece that holds the token.
// A list that has all that may be kept (most rows that are not flat) is cut by rank and walked over by index in the first CTA instead.
// All sums are taken in an order that sizes alone give: the same inputs give the same token.
//
// Floors are a row's bytes, read once: 64 rows of 262144 in bf16 5.1 us, 256 of 50257 in f32 7.9, of 128000 20.  None of them bounds, and no
// pipe does: a pass over values in L2 takes 30 to 60 issue slots a value and warp for shares in 64 bits (8 for the largest value, about 10 cycles of
// the shared-memory atomics a count in a bin), and an SM's 13 to 14 warps fill a quarter (best token) to a half (tokens as they are, top_p) of the slots
// between waits for memory, fixed latencies and barriers.  For 22 (tokens as they are) to 57 % of the time (rows with settings of their own) an
// SM has no CTA, since rows take different times.  In a graph over inputs larger than L2, f32 64 x 262144: the largest alone 18.9 us (3.6 TB/s),
// as they are 46, above a floor of 0.1 59 and of 0.01 86, by a count of 50 49, of 300 89, of 1000 103, by top_p 155 to 163; bf16 with settings of
// their own and a cap 75 to 184 by what is drawn, 108 on most; 256 x 50257 as they are 38.8, 256 x 128000 by top_p 220 to 260; one row of 262144
// 4.8, 14.0, by a count of 50 14, of 1000 34, by top_p 38, of which about half is cluster barriers and the first CTA's work on lists and bins.  With borders found by
// halving instead of bins, conversions of values where they are used and half the CTAs for rows with rules (the first form) the 64 rows with
// settings of their own took 424 us, the 256 of 50257 70 and the 256 of 128000 720.
//
// The parts are functions of their own that find what they share in shared memory: inlined where they are called they were 360 KB of code.
#include "gv_common.cuh"
#include "gv_shares.h"
#include "gv_step.h"

namespace gv {
namespace {

constexpr int kMostCtas = 16;
constexpr int kLevels = 10;       // groups of 2^level threads
constexpr int kSums = 3;
constexpr int kBins = 1024;       // of equal width over a range of values
constexpr int kEdges = 8;        // of four windows in the bins
constexpr int kAhead = 8;         // vectors that a thread has on their way: an L2 read takes as long as a warp works on these
constexpr int kTableCopies = 16;  // of the table of 2^(j/32), one for each lane of half a warp: no two lanes of a read meet in a bank

struct SampleParams {
  SampleCall call;
  int ctas;         // of a row's cluster
  int cta_vectors;  // 16-byte vectors of a row that a CTA goes through
};

// What the counts say of a border: it lies in bins first .. last.
enum BinsSay : int { kNotHere, kLookCloser, kInList, kListHasAll };  // (all: the list has everything from the largest value on, first is 0)
struct BinWindow {
  int first, last;
  BinsSay says;
  int sure_first, sure_last;  // what holds it in any case (kBins: that may be behind all bins)
};
// Bins of equal width from `high` (bin 0's middle) down to `low`; a bin's values are the nearest to its middle.  Half of a distance is a number of 32
// bits wherever both ends are; infinite values are in the first bin, and `high` is the largest number then.
struct Bins {
  float low, high, per_two;  // bins for two
  __device__ __forceinline__ float middle(float bin) const { return __fmaf_rn(bin / per_two, -2.0f, high); }  // (twice that may be more than a number says)
};

// How shares are worked out: from 32 bits' whole part where temperature and values are of ordinary size, of capped values where cap and
// temperature are, or of any.
enum ShareForm : int { kPlain, kCapped, kAny };
// cap * tanh(x / cap), with e = exp(-2 |x| / cap): cap * (1 - e) / (1 + e).
struct Cap {
  double cap, scale;      // scale: of |x| in 32nds of an octave of e
  float scale32, most32;  // beyond `most32` e is not noticed
};

// What all threads of a CTA know of its row.
struct RowState {
  const uint4* source;  // the row from the 16-byte boundary at or in front of its first value
  int lead;             // values in front of it there
  int vocabulary;
  int vectors;          // that have values of the row
  int cta_begin, cta_end, warp_vectors;  // the CTA's part of them, and how many a warp has of it
  int ctas, rank;
  ShareForm form;
  int bounded;          // whether top_k or top_p have a border: order above border_key, or equal to it and index up to border_index
  uint32_t border_key, border_index;
  float border;         // border_key's
  float scale32, top32, cut;  // kPlain: values below `cut` have no share
  float largest;
  double scale, top;    // of y
  Cap cap;
};

template <int kThreads>
struct SampleShared {
  static constexpr int kEach = 4;  // a thread's entries of the list
  static_assert(kBins % (4 * kThreads) == 0, "a thread adds up its bins four at a time");
  static constexpr int kCap = kEach * kThreads;
  static constexpr int kWarps = kThreads / 32;
  static constexpr int kFew = 128;
  uint4 ring[kWarps][kAhead][32];  // vectors on their way, of each lane its own
  double table[kExp2Entries * kTableCopies];
  RowState row;
  double few[kFew];
  union {
    unsigned long long mine[kCap];   // candidates of this CTA
    int4 bins4[kBins / 4];
    int bins[kBins + 32];            // (behind them one for each lane that has nothing to count: no branch, no conflict)
  };
  unsigned long long list[kCap];     // the cluster's, in its first CTA
  uint4 first[kMostCtas][4];       // largest key, levels, settings
  double slots[2][kMostCtas][kSums];
  double warp_sums[kWarps][kSums];
  uint4 window[2];                 // a BinWindow, from the first CTA, by turns
  unsigned long long border, kept; // from the first CTA: the border's entry, and how many of the list are up to it
  uint32_t warp_key[kWarps], warp_index[kWarps], warp_levels[kWarps][5];
  int mine_count, list_count, base, found;
  int edges[kEdges];
};
extern __shared__ uint4 sample_memory[];
template <int kThreads>
__device__ __forceinline__ SampleShared<kThreads>& shared() {
  return *reinterpret_cast<SampleShared<kThreads>*>(sample_memory);
}

__device__ __forceinline__ void cluster_store_double(uint32_t address, double v) {
  asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(address), "l"(__double_as_longlong(v)) : "memory");
}
__device__ __forceinline__ void cluster_store_u64(uint32_t address, unsigned long long v) {
  asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(address), "l"(v) : "memory");
}
__device__ __forceinline__ int4 cluster_load4(uint32_t address) {
  int4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(address) : "memory");
  return v;
}
__device__ __forceinline__ unsigned long long cluster_load_u64(uint32_t address) {
  unsigned long long v;
  asm volatile("ld.shared::cluster.b64 %0, [%1];" : "=l"(v) : "r"(address) : "memory");
  return v;
}
__device__ __forceinline__ int cluster_add(uint32_t address, int v) {
  int old;
  asm volatile("atom.relaxed.cluster.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(old) : "r"(address), "r"(v) : "memory");
  return old;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int d = 16; d > 0; d /= 2) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}
// Sum over the lanes up to this one.
__device__ __forceinline__ double warp_upto(double v) {
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const double w = __shfl_up_sync(0xffffffffu, v, d);
    if ((threadIdx.x & 31) >= d) v += w;
  }
  return v;
}

// The numbers next to one in order; the one that would stand for minus zero is left out.
__device__ __forceinline__ uint32_t order_below(uint32_t order) { return order == 0x80000000u ? 0x7ffffffeu : order - 1; }
__device__ __forceinline__ uint32_t order_above(uint32_t order) { return order == 0x7ffffffeu ? 0x80000000u : order + 1; }

static __constant__ double g_exp2_table[kExp2Entries] = GV_EXP2_TABLE_INIT;

// One step of a bitonic sort between lanes, or between a lane's two values.
__device__ __forceinline__ void order_lanes(unsigned long long& x, int stride, bool up) {
  const unsigned long long y = __shfl_xor_sync(0xffffffffu, x, stride);
  const bool lower = (threadIdx.x & stride) == 0;
  x = (x < y) == (lower == up) ? x : y;
}
// Bitonic, ascending; entries from `count` on up to a power of two, at least 64, are made the largest.  Strides below 64 are between
// the lanes of a warp, two values each, the others in shared memory.
template <int kThreads>
__device__ __noinline__ void sort_list(unsigned long long* list, int count) {
  constexpr int kWarps = kThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int whole = 64;
  while (whole < count && whole < SampleShared<kThreads>::kCap) whole *= 2;
  for (int i = count + threadIdx.x; i < whole; i += kThreads) list[i] = ~0ull;
  __syncthreads();
  for (int size = 64; size <= whole; size *= 2) {
    for (int stride = size / 2; stride >= 64; stride /= 2) {
      for (int i = threadIdx.x; i < whole / 2; i += kThreads) {
        const int a = 2 * i - (i & (stride - 1)), b = a + stride;
        const unsigned long long x = list[a], y = list[b];
        if ((x > y) == ((a & size) == 0)) {
          list[a] = y;
          list[b] = x;
        }
      }
      __syncthreads();
    }
    for (int block = warp; block < whole / 64; block += kWarps) {
      unsigned long long* const values = list + 64 * block;
      unsigned long long x = values[lane], y = values[lane + 32];
      if (size == 64) {
#pragma unroll
        for (int inner = 2; inner <= 32; inner *= 2) {
#pragma unroll
          for (int stride = inner / 2; stride > 0; stride /= 2) {
            order_lanes(x, stride, (lane & inner) == 0);           // (at 32: x up, y down)
            order_lanes(y, stride, inner == 32 ? false : (lane & inner) == 0);
          }
        }
      }
      const bool up = (64 * block & size) == 0;
      if ((x > y) == up) {
        const unsigned long long z = x;
        x = y;
        y = z;
      }
#pragma unroll
      for (int stride = 16; stride > 0; stride /= 2) {
        order_lanes(x, stride, up);
        order_lanes(y, stride, up);
      }
      values[lane] = x;
      values[lane + 32] = y;
    }
    __syncthreads();
  }
}

__device__ __forceinline__ float ranked_value(unsigned long long entry) { return value_of(~static_cast<uint32_t>(entry >> 32)); }
// What top_k and top_p leave: values above `value`, and those equal to it up to `index`.
struct Border {
  float value;
  uint32_t index;
  __device__ __forceinline__ bool inside(float x, uint32_t i) const { return (x > value) | ((x == value) & (i <= index)); }
};
__device__ __forceinline__ Border border_of(const RowState& row) { return {row.border, row.border_index}; }

// ---- shares

__device__ __forceinline__ float power_of_two(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float reciprocal(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// cap * tanh(x / cap) in both precisions.
struct Softened {
  double y;
  float y32;
};
__device__ __forceinline__ Softened softened(float x, const Cap& c, float cap32, const double* table) {
  const float size = fminf(fabsf(x), c.most32);
  const double e = share_with<true>(-wide_of(size), c.scale, share_whole(-size, c.scale32), table, kTableCopies);
  const float e32 = power_of_two(-size * (c.scale32 * (1.0f / kExp2Entries))), r32 = reciprocal(1.0f + e32);
  // 1 / (1 + e) by two steps of Newton's from 32 bits (2^-21: 2^-42, 2^-84)
  const double d = 1.0 + e;
  double r = wide_of(r32);
  r = __fma_rn(r, __fma_rn(-d, r, 1.0), r);
  r = __fma_rn(r, __fma_rn(-d, r, 1.0), r);
  const double y = c.cap * ((1.0 - e) * r);
  return {x < 0.0f ? -y : y, copysignf(cap32 * ((1.0f - e32) * r32), x)};
}
// A cap of at most this many times the temperature is of ordinary size: y in 32 bits is off by cap * 2^-22, so that a distance's whole part is
// by 2 * 128 * 46 * 2^-22 = 0.003 32nds, and y in 64 bits by cap * 2^-51.3, a share's exponent by 2^-43: no more than the series leaves.
constexpr double kMostCap = 128.0;
// So is a temperature of at least this many: zero and what is next to it come from wide_of off by up to 2^-126, 2^-46 of a temperature here.
constexpr float kLeastCappedDegrees = 1e-24f;
// By its distance from the largest in y, at most two caps (12 thousand 32nds of an octave), whose whole part needs 32 bits only: none beyond kShareOctaves.
__device__ __forceinline__ double capped_share(float x, double scale, float scale32, double top, float top32, const Cap& cap, float cap32, const double* table) {
  const Softened it = softened(x, cap, cap32, table);
  const float octaves = (it.y32 - top32) * scale32;
  const double share = share_with(it.y - top, scale, share_whole(it.y32 - top32, scale32), table, kTableCopies);
  return octaves > -kShareOctaves * kExp2Entries ? share : 0.0;
}
// cap * tanh(x / cap) for any cap, to a few steps of 64 bits: 1 - e keeps too little of a value that is small next to its cap.  There the series
// x (1 - z^2 / 3 + 2 z^4 / 15 - 17 z^6 / 315) is off by 62 z^8 / 2835, 2^-65 at z = ln 2 / 128, where e's exponent is half a 32nd.
__device__ __noinline__ double softened_any(float x, const Cap& c, const double* table) {
  const double size = fmin(fabs(static_cast<double>(x)), 24.0 * c.cap), octaves = size * c.scale;
  double y;
  if (octaves <= 0.5) {
    const double z = size / c.cap, q = z * z;
    y = size * (1.0 - q * (1.0 / 3.0 - q * (2.0 / 15.0 - q * (17.0 / 315.0))));
  } else {
    const double e = share_with<true>(-size, c.scale, share_whole(-static_cast<float>(octaves), 1.0f), table, kTableCopies);
    y = c.cap * ((1.0 - e) / (1.0 + e));
  }
  return x < 0.0f ? -y : y;
}
// A little below the value with the largest one's y and so many temperatures less: where there is a cap, below where its inverse is.
__device__ __noinline__ double value_below(const RowState& row, double degrees, double temperatures) {
  double y = row.top - degrees * temperatures;
  if (row.cap.cap > 0.0) {
    const double z = y / row.cap.cap - 1e-12;
    y = z > -1.0 ? row.cap.cap * 0.5 * log((1.0 + z) / fmax(1.0 - z, 1e-30)) : -INFINITY;
  }
  return y - 1e-6 * (fabs(y) + fabs(static_cast<double>(row.largest)));
}
template <int kThreads>
__device__ __forceinline__ const double* lane_table() {
  return shared<kThreads>().table + (threadIdx.x & (kTableCopies - 1));
}

// Shares of the plain form.  Values below `cut`, and what is no number, have the share of `cut`, 2^-200: a sum does not notice it, and a comparison
// and a choice for each value are saved (comparisons, choices and logic run at half the rate of the rest, and bound a pass).
struct PlainShares {
  double scale, top;
  float scale32, top32, cut;
  uint32_t table;  // address of this lane's copy
  template <int kThreads>
  static __device__ __forceinline__ PlainShares of() {
    const RowState& row = shared<kThreads>().row;
    return {row.scale, row.top, row.scale32, row.top32, row.cut, smem_u32(lane_table<kThreads>())};
  }
  __device__ __forceinline__ double operator()(float value) const {
    const float x = fmaxf(value, cut);
    const uint32_t n = share_whole(x - top32, scale32);
    double entry;
    asm("ld.shared.f64 %0, [%1];" : "=d"(entry) : "r"((n & (kExp2Entries - 1)) * (8 * kTableCopies) + table));
    const double whole = __hiloint2double(0x43300000, static_cast<int>(n)) - (0x1p52 + kShareWhole);
    return scaled_by(exp2_rest(__fma_rn(static_cast<double>(x) - top, scale, -whole)) * entry, n);
  }
};

// The share of any value that may be taken.
template <int kThreads>
__device__ __noinline__ double share(float x) {
  const RowState& row = shared<kThreads>().row;
  const double* table = lane_table<kThreads>();
  if (row.form == kPlain) return x >= row.cut ? PlainShares::of<kThreads>()(x) : 0.0;
  if (row.form == kCapped) return capped_share(x, row.scale, row.scale32, row.top, row.top32, row.cap, static_cast<float>(row.cap.cap), table);
  if (row.cap.cap > 0.0) return share_of(softened_any(x, row.cap, table) - row.top, row.scale, table, kTableCopies);
  if (isinf(x)) return 1.0;  // (the largest value is infinite then, and so is this one)
  return isinf(row.top) ? 0.0 : share_of(static_cast<double>(x) - row.top, row.scale, table, kTableCopies);
}

struct Eight {
  double w[8];
};
// Of eight values, side by side (a share is a chain of a dozen operations that wait for one another), where the form is not the plain one.
template <int kThreads>
__device__ __noinline__ Eight other_shares(float a, float b, float c, float d, float e, float f, float g, float h) {
  const RowState& row = shared<kThreads>().row;
  const float x[8] = {a, b, c, d, e, f, g, h};
  Eight out;
  if (row.form == kCapped) {
    const Cap cap = row.cap;
    const double scale = row.scale, top = row.top;
    const float scale32 = row.scale32, top32 = row.top32, cap32 = static_cast<float>(cap.cap);
    const double* table = lane_table<kThreads>();
#pragma unroll
    for (int i = 0; i < 8; ++i) out.w[i] = capped_share(x[i], scale, scale32, top, top32, cap, cap32, table);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) out.w[i] = x[i] > -INFINITY ? share<kThreads>(x[i]) : 0.0;
  }
  return out;
}

// ---- going through a row

template <typename T>
struct Vector;
template <>
struct Vector<float> {
  static constexpr int kValues = 4;
  static __device__ __forceinline__ void unpack(const uint4& v, float* x) {
    x[0] = __uint_as_float(v.x);
    x[1] = __uint_as_float(v.y);
    x[2] = __uint_as_float(v.z);
    x[3] = __uint_as_float(v.w);
  }
};
template <>
struct Vector<__nv_bfloat16> {
  static constexpr int kValues = 8;
  static __device__ __forceinline__ void unpack(const uint4& v, float* x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};

// A thread's way through its warp's part of a row, vectors that follow one another in steps of 32, eight values at a time.
template <typename T, int kThreads>
struct Walk {
  static constexpr int kE = Vector<T>::kValues;
  static constexpr int kGroup = 8 / kE;
  const uint4* source;
  int begin, end;  // vectors
  int last;        // the row's last one
  int lead;
  unsigned limit;  // indexes that are the row's, and of vectors up to the end

  __device__ __forceinline__ Walk(int begin, int end) : begin(begin), end(end) {
    const RowState& row = shared<kThreads>().row;
    source = row.source;
    last = row.vectors - 1;
    lead = row.lead;
    limit = static_cast<unsigned>(max(0, min(row.vocabulary, end * kE - lead)));
  }
  // This warp's part.
  static __device__ __forceinline__ Walk mine() {
    const RowState& row = shared<kThreads>().row;
    const int begin = min(row.cta_end, row.cta_begin + static_cast<int>(threadIdx.x >> 5) * row.warp_vectors);
    return Walk(begin, min(row.cta_end, begin + row.warp_vectors));
  }
  __device__ __forceinline__ int index_of(int v) const { return v * kE - lead; }
  // Values that are not of these vectors, or none of the row's, are minus infinity.
  __device__ __forceinline__ void mask(int v, float* x) const {
#pragma unroll
    for (int i = 0; i < kE; ++i) x[i] = static_cast<unsigned>(index_of(v) + i) < limit ? x[i] : -INFINITY;
  }
  // f(value, index) of vector v's.
  template <class F>
  __device__ __forceinline__ void one_vector(int v, F&& f) const {
    float x[kE];
    Vector<T>::unpack(source[v], x);
    mask(v, x);
#pragma unroll
    for (int i = 0; i < kE; ++i) f(x[i], index_of(v) + i);
  }
  // f(values, the first vector's number): value i is of vector + 32 * (i / kE).  The next values are on their way meanwhile, by asynchronous copies
  // that a lane waits for and reads itself.
  template <class F>
  __device__ __forceinline__ void each_eight(F&& f) const {
    constexpr int kDepth = kAhead / kGroup;
    const int lane = threadIdx.x & 31;
    uint4* const ring = &shared<kThreads>().ring[threadIdx.x >> 5][0][lane];
    const uint32_t to = smem_u32(ring);
    const auto ask = [&](int at, int slot) {
      if (at < end) {
#pragma unroll
        for (int g = 0; g < kGroup; ++g)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + 512 * (slot * kGroup + g)), "l"(source + min(at + lane + 32 * g, last)) : "memory");
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int d = 0; d < kDepth; ++d) ask(begin + 32 * kGroup * d, d);
    int slot = 0;
#pragma unroll 1
    for (int at = begin; at < end; at += 32 * kGroup) {
      const int v = at + lane;
      float x[8];
      asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
#pragma unroll
      for (int g = 0; g < kGroup; ++g) Vector<T>::unpack(ring[32 * (slot * kGroup + g)], x + g * kE);
      if (at == 0 || at + 32 * kGroup >= end) {  // (the ends; the same for the whole warp)
#pragma unroll
        for (int g = 0; g < kGroup; ++g) mask(v + 32 * g, x + g * kE);
      }
      f(x, v);
      ask(at + 32 * kGroup * kDepth, slot);  // (its values have been read: they have been worked on)
      slot = (slot + 1) & (kDepth - 1);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }
  __device__ __forceinline__ int index_in(int v, int i) const { return index_of(v + 32 * (i / kE)) + i % kE; }
};

template <int kThreads>
__device__ __forceinline__ void cluster_barrier() {
  __syncwarp();
  if (shared<kThreads>().row.ctas > 1) cluster_sync_all();
  else __syncthreads();
}

struct Three {
  double a, b, c;
};
// Sums over the cluster, in every thread the same; slots[which][rank] has the CTAs' own, warp_sums the warps' of this one.
template <int kThreads>
__device__ __noinline__ Three cluster_sums(double a, double b, double c, int which) {
  SampleShared<kThreads>& sh = shared<kThreads>();
  constexpr int kWarps = kThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, ctas = sh.row.ctas;
  a = warp_sum(a);
  b = warp_sum(b);
  c = warp_sum(c);
  if (lane == 0) {
    sh.warp_sums[warp][0] = a;
    sh.warp_sums[warp][1] = b;
    sh.warp_sums[warp][2] = c;
  }
  __syncthreads();
  if (warp == 0 && lane < ctas) {
    const uint32_t peer = cluster_map_shared(smem_u32(&sh.slots[which][sh.row.rank][0]), lane);
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      double sum = 0.0;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) sum += sh.warp_sums[w][i];
      cluster_store_double(peer + 8 * i, sum);
    }
  }
  cluster_barrier<kThreads>();
  const double* slot = sh.slots[which][lane & (kMostCtas - 1)];
  const bool mine = lane < ctas;
  return {warp_sum(mine ? slot[0] : 0.0), warp_sum(mine ? slot[1] : 0.0), warp_sum(mine ? slot[2] : 0.0)};
}

// ---- passes

template <typename T, int kThreads>
__device__ __noinline__ float largest_value() {
  const auto walk = Walk<T, kThreads>::mine();
  float a = -INFINITY, b = -INFINITY;
  walk.each_eight([&](const float (&x)[8], int) {  // (fmaxf of a number and none is the number)
    a = fmaxf(fmaxf(a, fmaxf(x[0], x[1])), fmaxf(x[2], x[3]));
    b = fmaxf(fmaxf(b, fmaxf(x[4], x[5])), fmaxf(x[6], x[7]));
  });
  return fmaxf(a, b);
}

template <typename T, int kThreads>
__device__ __noinline__ uint32_t first_index_of(float value) {
  const auto walk = Walk<T, kThreads>::mine();
  uint32_t index = 0xffffffffu;
  walk.each_eight([&](const float (&x)[8], int v) {
#pragma unroll
    for (int i = 0; i < 8; ++i) index = x[i] == value ? min(index, static_cast<uint32_t>(walk.index_in(v, i))) : index;
  });
  return index;
}

// (of what is not in the range any: sums tell whether the border is where counts say)
__device__ __forceinline__ int bin_of(const Bins& bins, float x) { return bin_at(half_distance(bins.high, x), bins.per_two, kBins); }
__device__ __forceinline__ Bins bins_between(float low, float high) {
  const float finite = fminf(high, 3.402823466e38f);
  return {low, finite, bins_for_one(kBins, half_distance(finite, low))};
}

template <int kThreads>
__device__ __forceinline__ void clear_bins() {
  for (int i = threadIdx.x; i < kBins; i += kThreads) shared<kThreads>().bins[i] = 0;
  __syncthreads();
}

// softened(), in 32 bits.
__device__ __forceinline__ float capped_in_32_bits(float x, float cap, float rate) {
  const float e = power_of_two(-fabsf(x) * rate);
  return copysignf(cap * ((1.0f - e) * reciprocal(1.0f + e)), x);
}

// Counts what is inside by bins; with `shares` also this lane's sum of shares, in 32 bits: where to look, no more.
template <typename T, int kThreads>
__device__ __noinline__ float look(Bins bins, bool shares) {
  SampleShared<kThreads>& sh = shared<kThreads>();
  const auto walk = Walk<T, kThreads>::mine();
  const Border border = border_of(sh.row);
  const int nothing = kBins + (threadIdx.x & 31);
  const bool all = !sh.row.bounded;
  const ShareForm form = sh.row.form;
  const float top32 = sh.row.top32, rate = sh.row.scale32 * (1.0f / kExp2Entries);
  const float cap = static_cast<float>(sh.row.cap.cap), cap_rate = sh.row.cap.scale32 * (1.0f / kExp2Entries);
  float sum = 0.0f;
  walk.each_eight([&](const float (&x)[8], int v) {
    bool in[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) in[i] = true;
    if (!all) {
#pragma unroll
      for (int i = 0; i < 8; ++i) in[i] = border.inside(x[i], walk.index_in(v, i));
    }
    if (shares) {
      if (form != kAny) {
        float w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          w[i] = fmaxf(x[i], -3.402823466e38f);  // (no number: none)
          if (form == kCapped) w[i] = capped_in_32_bits(w[i], cap, cap_rate);
          w[i] = power_of_two((w[i] - top32) * rate);
          w[i] = in[i] & (x[i] > -INFINITY) ? w[i] : 0.0f;
        }
        sum += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
      } else {
        const Eight eight = other_shares<kThreads>(x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]);
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += in[i] & (x[i] > -INFINITY) ? static_cast<float>(eight.w[i]) : 0.0f;
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) atomicAdd(&sh.bins[in[i] & (x[i] >= bins.low) ? bin_of(bins, x[i]) : nothing], 1);
  });
  return sum;
}

// Of what is inside: what lies from `low` to `high` is put on this CTA's list or, with bins, counted in them.  Measured for this lane: what is above
// `high` and not above `before`, by shares or by how many; and with `whole`, the shares of all.
struct Sifted {
  double above, all;
};
template <typename T, int kThreads, bool kGeneral>
__device__ __noinline__ Sifted sift(bool binned, float low, float high, float before, bool measured, bool shares, bool whole, Bins bins) {
  SampleShared<kThreads>& sh = shared<kThreads>();
  constexpr int kCap = SampleShared<kThreads>::kCap;
  const auto walk = Walk<T, kThreads>::mine();
  constexpr int kE = Walk<T, kThreads>::kE, kGroup = Walk<T, kThreads>::kGroup;
  const Border border = border_of(sh.row);
  const int nothing = kBins + (threadIdx.x & 31);
  const PlainShares plain_share = PlainShares::of<kThreads>();
  const bool all_before = before >= sh.row.largest;
  Sifted sifted{0.0, 0.0};
  // Hits are a few of thousands: which values they are is noted in bits, and they are put on the list behind some rounds of the loop together.
  unsigned long long noted = 0;
  int noted_from = walk.begin + (threadIdx.x & 31), rounds = 0;
  const auto put = [&]() {
    if (noted == 0) return;
    int to = atomicAdd(&sh.mine_count, __popcll(noted));
    while (noted != 0) {
      const int bit = __ffsll(noted) - 1, i = bit & 7;
      noted &= noted - 1;
      const int v = noted_from + (bit >> 3) * 32 * kGroup + i / kE * 32;
      const float x = static_cast<float>(reinterpret_cast<const T*>(walk.source + v)[i % kE]);
      if (to < kCap) sh.mine[to] = static_cast<unsigned long long>(~order_of(x)) << 32 | static_cast<uint32_t>(walk.index_of(v) + i % kE);
      ++to;
    }
  };
  walk.each_eight([&](const float (&x)[8], int v) {
    // (most often nothing is between `low` and `high`: bits only where something is)
    bool any = false, over[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      over[i] = x[i] > high;
      any |= (x[i] >= low) & !over[i];
    }
    if (!all_before) {
#pragma unroll
      for (int i = 0; i < 8; ++i) over[i] &= x[i] <= before;
    }
    uint32_t hits = 0;
    if (any || binned) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        bool in = (x[i] >= low) & (x[i] <= high);
        if (kGeneral) in &= border.inside(x[i], walk.index_in(v, i));
        hits |= in ? 1u << i : 0u;
      }
    }
    if (kGeneral) {
#pragma unroll
      for (int i = 0; i < 8; ++i) over[i] &= border.inside(x[i], walk.index_in(v, i));
    }
    if (whole || measured) {
      bool higher = false;
#pragma unroll
      for (int i = 0; i < 8; ++i) higher |= over[i];
      if (!shares) {
#pragma unroll
        for (int i = 0; i < 8; ++i) sifted.above += over[i] ? 1.0 : 0.0;
      } else if (whole || higher) {
        double w[8];
        if (!kGeneral || sh.row.form == kPlain) {
#pragma unroll
          for (int i = 0; i < 8; ++i) w[i] = plain_share(x[i]);
        } else {
          const Eight eight = other_shares<kThreads>(x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]);
#pragma unroll
          for (int i = 0; i < 8; ++i) w[i] = eight.w[i];
        }
        if (kGeneral) {
#pragma unroll
          for (int i = 0; i < 8; ++i) w[i] = border.inside(x[i], walk.index_in(v, i)) ? w[i] : 0.0;
        }
        sifted.all += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = over[i] ? w[i] : 0.0;
        sifted.above += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
      }
    }
    if (binned) {
#pragma unroll
      for (int i = 0; i < 8; ++i) atomicAdd(&sh.bins[hits >> i & 1 ? bin_of(bins, x[i]) : nothing], 1);
    } else {
      noted |= static_cast<unsigned long long>(hits) << (8 * rounds);
      if (++rounds == 8) {
        put();
        noted_from += 8 * 32 * kGroup;
        rounds = 0;
      }
    }
  });
  if (!binned) put();
  return sifted;
}
template <typename T, int kThreads>
__device__ __forceinline__ Sifted sift_row(bool binned, float low, float high, float before, bool measured, bool shares, bool whole, const Bins& bins) {
  const RowState& row = shared<kThreads>().row;
  if (row.form == kPlain && !row.bounded) return sift<T, kThreads, false>(binned, low, high, before, measured, shares, whole, bins);
  return sift<T, kThreads, true>(binned, low, high, before, measured, shares, whole, bins);
}

// This lane's sum of the shares, of vectors begin .. end - 1, that are inside and not below `least`.
template <typename T, int kThreads>
__device__ __noinline__ double sum_shares(int begin, int end, double least) {
  SampleShared<kThreads>& sh = shared<kThreads>();
  const Walk<T, kThreads> walk(begin, end);
  const PlainShares plain_share = PlainShares::of<kThreads>();
  const Border border = border_of(sh.row);
  double sum = 0.0;
  if (sh.row.form == kPlain && !sh.row.bounded && !(least > 0.0)) {  // the ordinary case by itself: a dozen instructions a value fewer
    walk.each_eight([&](const float (&x)[8], int) {
      double w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = plain_share(x[i]);
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = x[i] >= plain_share.cut ? w[i] : 0.0;  // (none at all: a random number of zero finds the first that has some)
      sum += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
    });
    return sum;
  }
  const bool plain = sh.row.form == kPlain;
  walk.each_eight([&](const float (&x)[8], int v) {
    double w[8];
    if (plain) {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = plain_share(x[i]);
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = x[i] >= plain_share.cut ? w[i] : 0.0;
    } else {
      const Eight eight = other_shares<kThreads>(x[0], x[1], x[2], x[3], x[4], x[5], x[6], x[7]);
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = eight.w[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = border.inside(x[i], walk.index_in(v, i)) & (w[i] >= least) & (x[i] > -INFINITY) ? w[i] : 0.0;
    sum += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
  });
  return sum;
}

// How many of them are inside and equal to `value`.
template <typename T, int kThreads>
__device__ __noinline__ double count_ties(int begin, int end, float value) {
  const Border border = border_of(shared<kThreads>().row);
  const Walk<T, kThreads> walk(begin, end);
  int count = 0;
  walk.each_eight([&](const float (&x)[8], int v) {
#pragma unroll
    for (int i = 0; i < 8; ++i) count += (x[i] == value) & border.inside(x[i], walk.index_in(v, i)) ? 1 : 0;
  });
  return count;
}

// This lane's sum of the shares that the first CTA's list has up to the border, of values in this warp's part.
template <typename T, int kThreads>
__device__ __noinline__ double sum_listed() {
  SampleShared<kThreads>& sh = shared<kThreads>();
  const auto walk = Walk<T, kThreads>::mine();
  const int kept = static_cast<int>(sh.kept), rank = sh.row.rank;
  const unsigned long long* list = sh.list;
  if (rank > 0) {  // (the first CTA waits for all at the next exchange)
    list = sh.mine;
    const uint32_t from = cluster_map_shared(smem_u32(sh.list), 0);
    for (int i = threadIdx.x; i < kept; i += kThreads) sh.mine[i] = cluster_load_u64(from + 8 * i);
    __syncthreads();
  }
  const int first = walk.index_of(walk.begin), behind = walk.index_of(walk.end);
  double sum = 0.0;
  for (int i = threadIdx.x & 31; i < kept; i += 32) {
    const unsigned long long entry = list[i];
    const int index = static_cast<int>(entry);
    if (index >= first && index < behind) sum += share<kThreads>(ranked_value(entry));
  }
  return sum;
}

// The first CTA's list gets what lies from `low` to `high` in order and is inside; `count` of them (more than kCap: the list is not whole).
struct Gathered {
  int count;
  Sifted sifted;  // this lane's
  Sifted sums;    // the cluster's
};
template <typename T, int kThreads>
__device__ __noinline__ Gathered gather(uint32_t low, uint32_t high, float before, bool measured, bool shares, bool whole, int which) {
  SampleShared<kThreads>& sh = shared<kThreads>();
  constexpr int kCap = SampleShared<kThreads>::kCap;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, ctas = sh.row.ctas;
  if (threadIdx.x == 0) sh.mine_count = 0;
  __syncthreads();
  Gathered got;
  got.sifted = sift_row<T, kThreads>(false, value_of(low), value_of(high), before, measured, shares, whole, Bins{});
  const double above = warp_sum(got.sifted.above), all = warp_sum(got.sifted.all);
  if (lane == 0) {
    sh.warp_sums[warp][0] = above;
    sh.warp_sums[warp][1] = all;
  }
  __syncthreads();
  const int count = sh.mine_count;
  if (warp == 0) {
    if (lane < ctas) {  // (the sums go with the count: no exchange of their own)
      double own[2] = {0.0, 0.0};
#pragma unroll
      for (int w = 0; w < kThreads / 32; ++w) {
        own[0] += sh.warp_sums[w][0];
        own[1] += sh.warp_sums[w][1];
      }
      const uint32_t peer = cluster_map_shared(smem_u32(&sh.slots[which][sh.row.rank][0]), lane);
      cluster_store_double(peer, static_cast<double>(count));
      cluster_store_double(peer + 8, own[0]);
      cluster_store_double(peer + 16, own[1]);
    }
    if (lane == 0) sh.base = count > 0 && count <= kCap ? cluster_add(cluster_map_shared(smem_u32(&sh.list_count), 0), count) : kCap;
  }
  __syncthreads();
  if (count <= kCap) {
    const uint32_t list = cluster_map_shared(smem_u32(sh.list), 0);
    const int base = sh.base;
    for (int i = threadIdx.x; i < count; i += kThreads)
      if (base + i < kCap) cluster_store_u64(list + 8 * (base + i), sh.mine[i]);
  }
  cluster_barrier<kThreads>();
  const double* slot = sh.slots[which][lane & (kMostCtas - 1)];
  const bool one = lane < ctas;
  if (threadIdx.x == 0) sh.list_count = 0;  // (for the next gathering, which a barrier comes before)
  got.count = static_cast<int>(warp_sum(one ? slot[0] : 0.0));
  got.sums = {warp_sum(one ? slot[1] : 0.0), warp_sum(one ? slot[2] : 0.0)};
  return got;
}

// ---- the first CTA's list

// The entries of the list, which has more than `ranks`, up to the bin of their value that the last of the first `ranks` is in: to
// `mine`; returns how many.
template <int kThreads>
__device__ __noinline__ int prune(int count, int ranks, float highest) {
  SampleShared<kThreads>& sh = shared<kThreads>();
  constexpr int kFewBins = kThreads, kEach = SampleShared<kThreads>::kEach, kWarps = kThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  sh.bins[threadIdx.x] = 0;
  if (threadIdx.x == 0) {
    sh.edges[0] = kFewBins - 1;
    sh.edges[1] = 0;
  }
  float lowest = highest;
  unsigned long long entries[kEach];
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int i = threadIdx.x + j * kThreads;
    entries[j] = i < count ? sh.list[i] : 0;
    if (i < count) lowest = fminf(lowest, ranked_value(entries[j]));
  }
  const uint32_t low = __reduce_min_sync(0xffffffffu, order_of(lowest));
  if (lane == 0) sh.warp_index[warp] = low;
  __syncthreads();
  uint32_t least = sh.warp_index[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) least = min(least, sh.warp_index[w]);
  const float finite = fminf(highest, 3.402823466e38f), per_two = bins_for_one(kFewBins, half_distance(finite, value_of(least)));
  const auto bin = [&](unsigned long long entry) { return bin_at(half_distance(finite, ranked_value(entry)), per_two, kFewBins); };
#pragma unroll
  for (int j = 0; j < kEach; ++j)
    if (threadIdx.x + j * kThreads < count) atomicAdd(&sh.bins[bin(entries[j])], 1);
  __syncthreads();
  int upto = sh.bins[threadIdx.x];
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int more = __shfl_up_sync(0xffffffffu, upto, d);
    if (lane >= d) upto += more;
  }
  if (lane == 31) sh.warp_index[warp] = upto;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) upto += w < warp ? sh.warp_index[w] : 0;
  if (upto >= ranks) atomicMin(&sh.edges[0], static_cast<int>(threadIdx.x));
  __syncthreads();
  const int last = sh.edges[0];
  uint32_t keep = 0;
#pragma unroll
  for (int j = 0; j < kEach; ++j) keep |= threadIdx.x + j * kThreads < count && bin(entries[j]) <= last ? 1u << j : 0u;
  int to = keep ? atomicAdd(&sh.edges[1], __popc(keep)) : 0;  // (sorted afterwards: any order will do)
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kEach; ++j)
    if (keep >> j & 1) sh.mine[to++] = entries[j];
  __syncthreads();
  return sh.edges[1];
}

// Sums up to each of a thread's entries, over the whole CTA.
template <int kThreads>
struct Upto {
  double upto[SampleShared<kThreads>::kEach], in_front, all;
};
template <int kThreads>
__device__ __forceinline__ Upto<kThreads> list_upto(const double (&w)[SampleShared<kThreads>::kEach]) {
  SampleShared<kThreads>& sh = shared<kThreads>();
  constexpr int kEach = SampleShared<kThreads>::kEach, kWarps = kThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  Upto<kThreads> out;
  double mine = 0.0;
#pragma unroll
  for (int j = 0; j < kEach; ++j) mine += w[j];
  const double inclusive = warp_upto(mine);
  if (lane == 31) sh.warp_sums[warp][0] = inclusive;
  __syncthreads();
  double before = 0.0;
  out.all = 0.0;
#pragma unroll
  for (int v = 0; v < kWarps; ++v) {
    if (v == warp) before = out.all;
    out.all += sh.warp_sums[v][0];
  }
  const double previous = __shfl_up_sync(0xffffffffu, inclusive, 1);
  out.in_front = before + (lane > 0 ? previous : 0.0);
  double sum = out.in_front;
#pragma unroll
  for (int j = 0; j < kEach; ++j) out.upto[j] = sum += w[j];
  __syncthreads();
  return out;
}

// The border out of the first CTA's list of `count`, in all CTAs: the first entry by rank at which `above` and the measure of the entries up to it come
// to `target`.  False: it is not there.  (`surely`: the last entry where rounding leaves none.)
template <int kThreads>
__device__ __noinline__ bool border_from_list(int count, bool shares, double above, double target, bool surely) {
  SampleShared<kThreads>& sh = shared<kThreads>();
  constexpr int kEach = SampleShared<kThreads>::kEach;
  if (sh.row.rank == 0) {
    sort_list<kThreads>(sh.list, count);
    double w[kEach];
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int i = kEach * threadIdx.x + j;
      w[j] = i >= count ? 0.0 : shares ? share<kThreads>(ranked_value(sh.list[i])) : 1.0;
    }
    if (threadIdx.x == 0) sh.found = count;
    const Upto<kThreads> sums = list_upto<kThreads>(w);
    if (above < target || surely) {
#pragma unroll
      for (int j = kEach - 1; j >= 0; --j) {
        const int i = kEach * threadIdx.x + j;
        if (i < count && above + sums.upto[j] >= target) atomicMin(&sh.found, i);
      }
    }
    __syncthreads();
    int at = sh.found;
    if (surely && count > 0) at = min(at, count - 1);
    const unsigned long long entry = at < count ? sh.list[at] : 0;
    if (threadIdx.x < sh.row.ctas) {
      cluster_store_u64(cluster_map_shared(smem_u32(&sh.border), threadIdx.x), entry);
      cluster_store_u64(cluster_map_shared(smem_u32(&sh.kept), threadIdx.x), at < count ? at + 1 : 0);
    }
  }
  cluster_barrier<kThreads>();
  const unsigned long long entry = sh.border;
  if (entry == 0) return false;  // (no value that may be taken has the complement of zero for its order)
  if (threadIdx.x == 0) {
    sh.row.border_key = ~static_cast<uint32_t>(entry >> 32);
    sh.row.border_index = static_cast<uint32_t>(entry);
    sh.row.border = ranked_value(entry);
    sh.row.bounded = 1;
  }
  __syncthreads();
  return true;
}

// ---- where counts say that a border is

// The smallest order from `low` on (up to `high`, for which it holds) with a bin of at most `bin`; searched by 32 lanes at a time.
__device__ __noinline__ uint32_t order_with(Bins bins, int bin, uint32_t low, uint32_t high) {
  const int lane = threadIdx.x & 31;
  if (low < high) {  // most often it is among the 32 numbers about the bin's edge
    const uint32_t edge = order_of(bins.middle(static_cast<float>(bin) + 0.5f));
    const uint32_t begin = edge > low + 16 && edge < high ? edge - 16 : low, at = min(begin + lane, high);
    const uint32_t yes = __ballot_sync(0xffffffffu, at == high || bin_of(bins, value_of(at)) <= bin);
    if (yes != 0 && (yes & 1) == 0) return min(begin + __ffs(yes) - 1, high);
    if (yes & 1) high = begin;  // (begin is not below low)
    else low = begin + 32;
  }
  while (low < high) {
    const uint32_t step = (high - low) / 32 + 1, at = min(low + step * lane, high);
    const uint32_t yes = __ballot_sync(0xffffffffu, at == high || bin_of(bins, value_of(at)) <= bin);  // ascending: none, then all
    if (yes & 1) return low;
    const int first = yes ? __ffs(yes) - 1 : 32;
    const uint32_t next = min(low + step * first, high);
    low = min(low + step * (first - 1) + 1, next);
    high = next;
  }
  return low;
}

// Where the counts say that `target` is reached, with `above` in front of the bins.  Counts times the shares of their bins' middles are off by a factor of
// up to exp(off) either way: the border lies between where they reach the target with that much less and with that much more.  Where
// that is more than the list holds, it is looked at with a quarter, a sixteenth or a 64th of it (errors of many bins cancel; sums will tell), or
// closer.  `surely`: it is in the bins, whatever the counts say.  (With a sixteenth as the least 48 of 256 rows of 128000 by top_p were looked at again.)
template <int kThreads>
__device__ __noinline__ BinWindow window_of_bins(Bins bins, bool shares, double above, double target, double off, bool surely, int turn) {
  SampleShared<kThreads>& sh = shared<kThreads>();
  constexpr int kCap = SampleShared<kThreads>::kCap, kWarps = kThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, ctas = sh.row.ctas, rank = sh.row.rank;
  if (rank == 0) {
    constexpr int kOf = kBins / kThreads;
    const float rate = sh.row.scale32 * (1.0f / kExp2Entries), top32 = sh.row.top32;
    const bool plain = sh.row.form == kPlain;
    // A thread adds up its bins of all CTAs, which a barrier has been behind: 16 reads of 16 bytes from as many SMs on their way together.
    int count[kOf], counted = 0;
    float mass[kOf], massed = 0.0f;
#pragma unroll
    for (int i = 0; i < kOf; i += 4) {
      const int4* const own = &sh.bins4[(threadIdx.x * kOf + i) / 4];
      int4 sum = *own;
      const uint32_t at = smem_u32(own);
#pragma unroll 5
      for (int r = 1; r < ctas; ++r) {
        const int4 four = cluster_load4(cluster_map_shared(at, r));
        sum.x += four.x;
        sum.y += four.y;
        sum.z += four.z;
        sum.w += four.w;
      }
      count[i] = sum.x;
      count[i + 1] = sum.y;
      count[i + 2] = sum.z;
      count[i + 3] = sum.w;
    }
#pragma unroll
    for (int i = 0; i < kOf; ++i) {
      const int bin = threadIdx.x * kOf + i;
      const float middle = fmaxf(bins.middle(static_cast<float>(bin)), bins.low);
      mass[i] = 0.0f;
      if (shares && count[i] > 0) mass[i] = count[i] * (plain ? exp2f((middle - top32) * rate) : static_cast<float>(share<kThreads>(middle)));
      counted += count[i];
      massed += mass[i];
    }
    int counts = counted;
    float masses = massed;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int c = __shfl_up_sync(0xffffffffu, counts, d);
      const float m = __shfl_up_sync(0xffffffffu, masses, d);
      if (lane >= d) {
        counts += c;
        masses += m;
      }
    }
    if (lane == 31) {
      sh.warp_index[warp] = counts;
      sh.warp_key[warp] = __float_as_uint(masses);
    }
    if (threadIdx.x < kEdges) sh.edges[threadIdx.x] = kBins;
    __syncthreads();
    int count_upto = counts - counted;
    float mass_upto = masses - massed;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      count_upto += w < warp ? sh.warp_index[w] : 0;
      mass_upto += w < warp ? __uint_as_float(sh.warp_key[w]) : 0.0f;
    }
    // the target for counts' sums, by each edge: in which bin it is reached first
    const float rest = shares ? static_cast<float>(target - above) : static_cast<float>(ceil(target - above)), o = shares ? static_cast<float>(off) : 0.0f;
    float edge[kEdges] = {rest * expf(-o), rest * expf(o)};  // (counts: the target itself)
    int hit[kEdges];
#pragma unroll
    for (int e = 2; e < kEdges; e += 2) {
      const float less = fminf(o, 1.0f) * (e == 2 ? 1.0f / 4 : e == 4 ? 1.0f / 16 : 1.0f / 64);
      edge[e] = __fdividef(rest, 1.0f + less);
      edge[e + 1] = __fdividef(rest, 1.0f - less);
    }
#pragma unroll
    for (int e = 0; e < kEdges; ++e) hit[e] = kBins;
#pragma unroll
    for (int i = 0; i < kOf; ++i) {
      const int bin = threadIdx.x * kOf + i;
      count_upto += count[i];
      mass_upto += mass[i];
      sh.bins[bin] = count_upto;
      const float upto = shares ? mass_upto : static_cast<float>(count_upto);
#pragma unroll
      for (int e = 0; e < kEdges; ++e) hit[e] = upto >= edge[e] ? min(hit[e], bin) : hit[e];
    }
    int first = kBins;  // lane e's: of edge e in this warp
#pragma unroll
    for (int e = 0; e < kEdges; ++e) {
      const int least = __reduce_min_sync(0xffffffffu, hit[e]);
      first = lane == e ? least : first;
    }
    if (lane < kEdges && first < kBins) atomicMin(&sh.edges[lane], first);
    __syncthreads();
    if (warp == 0) {
      const auto upto = [&](int bin) { return bin < 0 ? 0 : sh.bins[bin]; };
      const int sure_first = sh.edges[0], sure_last = surely ? min(sh.edges[1], kBins - 1) : sh.edges[1];
      BinWindow window{sure_first, min(sure_last, kBins - 1), kNotHere, sure_first, sure_last};
      if (window.first < kBins) {
        if (sh.edges[1] < kBins && above == 0.0 && upto(window.last) <= kCap) {
          window.first = 0;
          window.says = kListHasAll;
        } else if (upto(window.last) - upto(window.first - 1) <= kCap) {
          window.says = kInList;
        } else {
          if (window.first > 0 || window.last < kBins - 1) window.says = kLookCloser;  // (else it would see the same)
          for (int e = 2; e < kEdges; e += 2) {
            if (sh.edges[e + 1] < kBins && upto(sh.edges[e + 1]) - upto(sh.edges[e] - 1) <= kCap) {
              window.first = sh.edges[e];
              window.last = sh.edges[e + 1];
              window.says = kInList;
              break;
            }
          }
        }
      }
      if (lane < ctas)
        cluster_store_uint4(cluster_map_shared(smem_u32(&sh.window[turn & 1]), lane), make_uint4(window.first, window.last, window.says, sure_first << 16 | sure_last));
    }
  }
  cluster_barrier<kThreads>();
  const uint4 w = sh.window[turn & 1];
  return BinWindow{static_cast<int>(w.x), static_cast<int>(w.y), static_cast<BinsSay>(w.z), static_cast<int>(w.w >> 16), static_cast<int>(w.w & 0xffffu)};
}

// ---- the token

// The first value of the vocabulary at which the sum of weights passes `of` times the sum of all, in one thread; the others have index -1.
// A value's weight is its share where it is kept and not below `least`; or (ties) one where it is `value`, and the sum comes to `of`.  `mine` is
// the sum of the lane's weights.
struct Located {
  int index;
  double weight, all;
};
template <typename T, int kThreads>
__device__ __noinline__ Located locate(double mine, bool ties, float value, double least, double of, int which) {
  SampleShared<kThreads>& sh = shared<kThreads>();
  constexpr int kWarps = kThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, ctas = sh.row.ctas;
  const Border border = border_of(sh.row);
  const auto weight = [&](float x, int index) {
    if (!border.inside(x, index)) return 0.0;
    if (ties) return x == value ? 1.0 : 0.0;
    const double w = share<kThreads>(x);
    return w < least ? 0.0 : w;
  };
  Located it{-1, 0.0, 0.0};
  const double all = cluster_sums<kThreads>(mine, 0.0, 0.0, which).a;
  const double target = ties ? fmin(fmax(ceil(of), 1.0), all) - 0.5 : of * all;
  // In what order sums follow one another: the part that holds the target, the last one with any weight where rounding leaves the target above all.
  struct Part {
    int hit, last;
    double front, last_front, sum;
    __device__ __forceinline__ void add(int part, double own, double target) {
      if (own > 0.0) {
        last = part;
        last_front = sum;
      }
      if (hit < 0 && sum + own > target) {
        hit = part;
        front = sum;
      }
      sum += own;
    }
    __device__ __forceinline__ void end() {
      if (hit < 0) {
        hit = last;
        front = last_front;
      }
    }
  };
  Part cta{-1, 0, 0.0, 0.0, 0.0};
  for (int r = 0; r < ctas; ++r) cta.add(r, sh.slots[which][r][0], target);
  cta.end();
  if (sh.row.rank != cta.hit || !(all > 0.0)) return it;
  Part in_warp{-1, 0, cta.front, cta.front, cta.front};
  for (int w = 0; w < kWarps; ++w) in_warp.add(w, sh.warp_sums[w][0], target);
  in_warp.end();
  // The warp's part is cut into as many pieces as there are warps, the piece that holds the target again, down to the 32 vectors that one
  // warp walks over.
  int from = sh.row.cta_begin + in_warp.hit * sh.row.warp_vectors, upto = min(sh.row.cta_end, from + sh.row.warp_vectors);
  double reached = in_warp.front;
  while (upto - from > 32) {
    const int piece = ((upto - from + kWarps - 1) / kWarps + 31) / 32 * 32;
    const int mine_from = from + warp * piece, mine_upto = min(upto, mine_from + piece);
    const double own = warp_sum(ties ? count_ties<T, kThreads>(mine_from, mine_upto, value) : sum_shares<T, kThreads>(mine_from, mine_upto, least));
    if (lane == 0) sh.warp_sums[warp][1] = own;
    __syncthreads();
    Part in_piece{-1, 0, reached, reached, reached};
    for (int w = 0; w < kWarps; ++w) in_piece.add(w, sh.warp_sums[w][1], target);
    in_piece.end();
    __syncthreads();
    from += in_piece.hit * piece;
    upto = min(upto, from + piece);
    reached = in_piece.front;
  }
  if (warp == 0) {
    const Walk<T, kThreads> end(from, upto);
    const int v = from + lane;
    double own = 0.0;
    if (v < upto) end.one_vector(v, [&](float x, int index) { own += weight(x, index); });
    const double sums = warp_upto(own), previous = __shfl_up_sync(0xffffffffu, sums, 1);
    const uint32_t passing = __ballot_sync(0xffffffffu, own > 0.0 && reached + sums > target);
    const uint32_t some = __ballot_sync(0xffffffffu, own > 0.0);
    const int chosen = passing ? __ffs(passing) - 1 : 31 - __clz(some);
    if (lane == chosen) {
      double running = reached + (lane > 0 ? previous : 0.0);
      bool done = false;
      end.one_vector(v, [&](float x, int index) {
        const double w = weight(x, index);
        if (!done && w > 0.0) it = Located{index, w, all};
        running += w;
        done |= w > 0.0 && running > target;
      });
    }
  }
  return it;
}

// ---- a border by halving

// Where all else fails (too many values, too equal or too far apart for bins): the value, and among its ties the index, at which the measure (shares,
// or how many) of what is inside and ranks up to there comes to `target`; from `low` to `high`, above which it measures `above`.  Sets the
// border; none where all that is inside does not come to it.
template <typename T, int kThreads>
__device__ __noinline__ int find_border(bool shares, double target, uint32_t low, uint32_t high, double above, int which) {
  SampleShared<kThreads>& sh = shared<kThreads>();
  constexpr int kCap = SampleShared<kThreads>::kCap;
  double count = 2.0 * kCap;  // how many lie from `low` to `high` (at first: many)
  for (int step = 0; low < high && count > kCap; ++step) {  // (every other step halves the range of orders: it ends in 64)
    const float middle = 0.5f * value_of(low) + 0.5f * value_of(high);
    uint32_t mid = step & 1 ? low + (high - low) / 2 : order_of(middle);
    mid = max(low, min(mid, order_below(high)));
    if (mid == 0x7fffffffu) mid = high > 0x80000000u ? 0x80000000u : 0x7ffffffeu;
    const float from = value_of(mid), bottom = value_of(low), upto = value_of(high);
    double within = 0.0, upper = 0.0, measure = 0.0;
    const auto walk = Walk<T, kThreads>::mine();
    const Border border = border_of(sh.row);
    walk.each_eight([&](const float (&x)[8], int v) {
      uint32_t in = 0, up = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool hit = (x[i] >= bottom) & (x[i] <= upto) & border.inside(x[i], walk.index_in(v, i));
        in |= hit ? 1u << i : 0u;
        up |= hit & (x[i] > from) ? 1u << i : 0u;
      }
      within += __popc(in);
      upper += __popc(up);
      if (shares && up != 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (up >> i & 1) measure += share<kThreads>(x[i]);
      }
    });
    const Three sums = cluster_sums<kThreads>(within, upper, measure, which);
    which ^= 1;
    const double over = shares ? sums.c : sums.b;
    if (above + over >= target) {
      low = order_above(mid);
      count = sums.b;
    } else {
      high = mid;
      above += over;
      count = sums.a - sums.b;
      if (count == 0.0) return which;  // (there are not as many: all stay)
    }
  }
  if (low < high || count <= kCap) {
    const int gathered = gather<T, kThreads>(low, high, value_of(high), false, false, false, which).count;
    which ^= 1;
    if (gathered <= kCap) {
      border_from_list<kThreads>(gathered, shares, above, target, true);
      return which;
    }
  }
  // More ties than the list holds: so many of them, in the order of the vocabulary.
  const float value = value_of(low);
  const auto part = Walk<T, kThreads>::mine();
  const double mine = count_ties<T, kThreads>(part.begin, part.end, value);
  double ties = target - above;
  if (shares) ties /= share<kThreads>(value);
  const Located it = locate<T, kThreads>(mine, true, value, 0.0, ties, which);
  which ^= 1;
  if (it.index >= 0)
    for (int r = 0; r < sh.row.ctas; ++r)
      cluster_store_u64(cluster_map_shared(smem_u32(&sh.border), r), static_cast<unsigned long long>(static_cast<uint32_t>(it.index)));
  cluster_barrier<kThreads>();
  if (threadIdx.x == 0) {
    sh.row.border_key = low;
    sh.row.border_index = static_cast<uint32_t>(sh.border);
    sh.row.border = value;
    sh.row.bounded = 1;
  }
  __syncthreads();
  return which;
}

// What a list that has all that may be kept gives.  counted: by rank the first top_k stay; by_sum: those in front of which less than top_p of the sum has
// been (of `whole_sum`, or where that is negative of the list's own); by_floor: shares of at least min_p.
struct Rules {
  int top_k;
  bool by_count, by_sum, by_floor;
  double top_p, min_p, u;
};
struct Taken {
  int index;  // -1: another thread has it
  float probability;
};
template <int kThreads>
__device__ __noinline__ Taken finish(int count, double whole_sum, const Rules& rules, float most) {
  SampleShared<kThreads>& sh = shared<kThreads>();
  constexpr int kEach = SampleShared<kThreads>::kEach, kFew = SampleShared<kThreads>::kFew;
  const int thread = threadIdx.x;
  Taken taken{-1, 0.0f};
  unsigned long long* list = sh.list;
  if (rules.by_count && count > 64 && count > rules.top_k) {  // nothing behind the bin that holds the top_k-th
    list = sh.mine;
    count = prune<kThreads>(count, rules.top_k, most);
  }
  sort_list<kThreads>(list, count);
  const int ranks = rules.by_count ? min(count, rules.top_k) : count;
  double w[kEach];
  unsigned long long entries[kEach];
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int i = kEach * thread + j;
    entries[j] = i < ranks ? list[i] : ~0ull;
    w[j] = i < ranks ? share<kThreads>(ranked_value(entries[j])) : 0.0;
  }
  const Upto<kThreads> sums = list_upto<kThreads>(w);
  const double target = rules.top_p * (whole_sum >= 0.0 ? whole_sum : sums.all);
  if (thread == 0) sh.found = ranks;
  __syncthreads();
#pragma unroll
  for (int j = kEach - 1; j >= 0; --j) {
    const int i = kEach * thread + j;
    const bool stays = i == 0 || !((rules.by_sum && (j == 0 ? sums.in_front : sums.upto[j > 0 ? j - 1 : 0]) >= target) || (rules.by_floor && w[j] < rules.min_p));
    if (i < ranks && !stays) atomicMin(&sh.found, i);
    list[i] = entries[j] << 32 | entries[j] >> 32;  // by index now, with the order behind it
  }
  __syncthreads();
  const int kept = sh.found;  // by rank; what is behind the first that goes, goes
  __syncthreads();            // (all have read it)
  if (kept <= kFew) {
    // Each with the sum of all up to its index: of few, sooner than sorted.
#pragma unroll
    for (int j = 0; j < kEach; ++j)
      if (kEach * thread + j < kept) sh.few[kEach * thread + j] = w[j];
    if (thread == 0) sh.found = 0x7fffffff;
    __syncthreads();
    double mine = 0.0, all = 0.0;
    const unsigned long long own = thread < kept ? list[thread] : 0;
    if (thread < kFew) {
#pragma unroll 4
      for (int j = 0; j < kept; ++j) {
        const double one = sh.few[j];
        all += one;
        mine += list[j] <= own ? one : 0.0;
      }
      // (the last by index has the whole sum, in the same order)
      if (thread < kept && mine > rules.u * all) atomicMin(&sh.found, static_cast<int>(own >> 32));
    }
    __syncthreads();
    if (thread < kept && static_cast<int>(own >> 32) == sh.found) taken = Taken{sh.found, static_cast<float>(sh.few[thread] / all)};
    return taken;
  }
  sort_list<kThreads>(list, kept);
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int i = kEach * thread + j;
    entries[j] = i < kept ? list[i] : ~0ull;
    w[j] = i < kept ? share<kThreads>(value_of(~static_cast<uint32_t>(entries[j]))) : 0.0;
  }
  if (thread == 0) sh.found = kept - 1;
  const Upto<kThreads> again = list_upto<kThreads>(w);
#pragma unroll
  for (int j = kEach - 1; j >= 0; --j)
    if (kEach * thread + j < kept && again.upto[j] > rules.u * again.all) atomicMin(&sh.found, kEach * thread + j);
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kEach; ++j)
    if (sh.found == kEach * thread + j) taken = Taken{static_cast<int>(entries[j] >> 32), static_cast<float>(w[j] / again.all)};
  return taken;
}

template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads, 512 / kThreads) sample_kernel(const SampleParams params) {
  SampleShared<kThreads>& sh = shared<kThreads>();
  constexpr int kE = Vector<T>::kValues, kWarps = kThreads / 32, kCap = SampleShared<kThreads>::kCap;
  const SampleCall& p = params.call;
  const int ctas = params.ctas, at_row = blockIdx.x / ctas, rank = static_cast<int>(ctas > 1 ? cluster_cta_rank() : 0);
  const int thread = threadIdx.x, lane = thread & 31, warp = thread >> 5;
  if (ctas > 1) cluster_arrive();  // (a CTA writes to the others when all have begun)
  for (int i = thread; i < kExp2Entries * kTableCopies; i += kThreads) sh.table[i] = g_exp2_table[i / kTableCopies];
  if (thread == 0) {
    sh.list_count = 0;
    // The row from the 16-byte boundary at or in front of its first value: what a vector has of other rows, or of the bytes in front of
    // and behind the tensor (of the same 16, and so of the same allocation), counts as nothing.
    const T* const data = static_cast<const T*>(p.logits) + at_row * p.row_stride;
    RowState& row = sh.row;
    row.lead = static_cast<int>((reinterpret_cast<uintptr_t>(data) & 15) / sizeof(T));
    row.source = reinterpret_cast<const uint4*>(data - row.lead);
    row.vocabulary = p.vocabulary;
    row.vectors = (row.lead + p.vocabulary + kE - 1) / kE;
    row.cta_begin = min(row.vectors, rank * params.cta_vectors);
    row.cta_end = min(row.vectors, row.cta_begin + params.cta_vectors);
    row.warp_vectors = params.cta_vectors / kWarps;
    row.ctas = ctas;
    row.rank = rank;
    row.bounded = 0;
    row.border_key = kNothing + 1;
    row.border_index = 0xffffffffu;
    row.border = -3.402823466e38f;
  }
  __syncthreads();
  grid_launch_dependents();
  grid_dependency_wait();
  float temperature = p.temperature ? p.temperature[at_row] : 1.0f;
  int top_k = p.top_k ? p.top_k[at_row] : 0;
  float top_p = p.top_p ? p.top_p[at_row] : 1.0f, floor = p.min_p ? p.min_p[at_row] : 0.0f;
  const float uniform = p.uniforms[at_row];
  const auto answer = [&](int token, float probability) {
    p.tokens[at_row] = token;
    if (p.probabilities) p.probabilities[at_row] = probability;
  };
  if (rank == 0 && thread == 0) answer(-1, 0.0f);  // until there is one, which barriers come before

  // ---- the largest value, and the levels
  {
    const uint32_t key = order_of(largest_value<T, kThreads>());
    uint32_t group = key, levels[5];
    levels[0] = __reduce_min_sync(0xffffffffu, group);
#pragma unroll
    for (int l = 1; l < 5; ++l) {
      group = max(group, __shfl_xor_sync(0xffffffffu, group, 1 << (l - 1)));
      levels[l] = __reduce_min_sync(0xffffffffu, group);
    }
    const uint32_t most = __reduce_max_sync(0xffffffffu, key);
    if (lane == 0) {
      sh.warp_key[warp] = most;
#pragma unroll
      for (int l = 0; l < 5; ++l) sh.warp_levels[warp][l] = levels[l];
    }
  }
  __syncthreads();
  if (ctas > 1) cluster_wait();
  if (warp == 0) {
    const bool mine = lane < kWarps;
    uint32_t out[16];
    uint32_t group = mine ? sh.warp_key[lane] : 0;
    out[0] = __reduce_max_sync(0xffffffffu, group);
    out[1] = 0;
#pragma unroll
    for (int l = 0; l < 5; ++l) out[2 + l] = __reduce_min_sync(0xffffffffu, mine ? sh.warp_levels[lane][l] : 0xffffffffu);
#pragma unroll
    for (int l = 5; l < kLevels; ++l) {  // groups of whole warps, as far as the CTA has them
      if (l > 5 && (1 << (l - 5)) <= kWarps) group = max(group, __shfl_xor_sync(0xffffffffu, group, 1 << (l - 6)));
      out[2 + l] = __reduce_min_sync(0xffffffffu, mine ? group : 0xffffffffu);
    }
    out[12] = __float_as_uint(temperature);
    out[13] = static_cast<uint32_t>(top_k);
    out[14] = __float_as_uint(top_p);
    out[15] = __float_as_uint(floor);
    if (lane < ctas) {
      const uint32_t peer = cluster_map_shared(smem_u32(&sh.first[rank][0]), lane);
#pragma unroll
      for (int i = 0; i < 4; ++i) cluster_store_uint4(peer + 16 * i, make_uint4(out[4 * i], out[4 * i + 1], out[4 * i + 2], out[4 * i + 3]));
    }
  }
  cluster_barrier<kThreads>();

  // The first CTA's settings are those of all: what CTAs meet at barriers by has to be the same in each, whatever another stream writes.
  const uint4 settings = sh.first[0][3];
  temperature = __uint_as_float(settings.x);
  top_k = static_cast<int>(settings.y);
  top_p = __uint_as_float(settings.z);
  floor = __uint_as_float(settings.w);
  const bool sampled = temperature > 0.0f;
  Rules rules;
  rules.top_k = top_k;
  rules.by_count = sampled && top_k > 0 && top_k < p.vocabulary;
  rules.by_sum = sampled && top_p < 1.0f;
  rules.by_floor = sampled && floor > 0.0f;
  rules.top_p = static_cast<double>(top_p);
  rules.min_p = rules.by_floor ? fmin(static_cast<double>(floor), 1.0) : 0.0;
  rules.u = fmin(fmax(static_cast<double>(uniform), 0.0), 1.0 - 0x1p-24);  // (not a number: zero)

  uint32_t largest, lower = kNothing + 1;  // at least top_k values are not below `lower`
  {
    const uint32_t* entry = reinterpret_cast<const uint32_t*>(&sh.first[lane < ctas ? lane : 0][0]);
    largest = __reduce_max_sync(0xffffffffu, entry[0]);
    if (rules.by_count) {
      int level = -1;
      for (int l = 0; l < kLevels && (1 << l) <= kThreads; ++l)
        if ((ctas * kThreads >> l) >= top_k) level = l;
      if (level >= 0) lower = max(lower, __reduce_min_sync(0xffffffffu, entry[2 + level]));
    }
  }
  if (largest <= kNothing) return;  // nothing to take
  const float most = value_of(largest);
  if (!sampled) {  // the best: the lowest index that has it, of the first CTA that has one
    bool before = false;
    for (int r = 0; r < rank; ++r) before |= sh.first[r][0].x == largest;
    if (before || sh.first[rank][0].x != largest) return;
    uint32_t index = __reduce_min_sync(0xffffffffu, first_index_of<T, kThreads>(most));
    if (lane == 0) sh.warp_index[warp] = index;
    __syncthreads();
    if (thread < kWarps) index = sh.warp_index[thread];
    if (warp == 0) index = __reduce_min_sync(0xffffffffu, index);
    if (thread == 0) answer(static_cast<int>(index), 1.0f);
    return;
  }
  const bool capped = p.softcap > 0.0f;
  const double degrees = static_cast<double>(temperature);
  if (thread == 0) {
    RowState& row = sh.row;
    constexpr double octave = 1.4426950408889634074 * kExp2Entries;
    row.cap = Cap{};
    if (capped) {
      const double rate = 2.0 * octave / p.softcap;
      row.cap = Cap{p.softcap, rate, static_cast<float>(rate), 24.0f * p.softcap};  // (2^-69 of one)
    }
    row.scale = octave / degrees;
    row.scale32 = static_cast<float>(row.scale);
    row.largest = most;
    const PlainRange plain = plain_range(most, degrees);
    const bool ordinary = (capped ? p.softcap > 1e-30f && p.softcap <= kMostCap * temperature && temperature >= kLeastCappedDegrees : plain.fits) &&
                          temperature > 1e-30f && temperature < 1e30f;
    row.top = static_cast<double>(most);
    row.top32 = most;
    if (capped && ordinary) {
      const Softened it = softened(most, row.cap, p.softcap, sh.table);
      row.top = it.y;
      row.top32 = it.y32;
    } else if (capped) {
      row.top = softened_any(most, row.cap, sh.table);
    }
    row.cut = plain.cut;
    // (sizes at which 32 bits hold the whole part of every share that there is)
    row.form = !ordinary ? kAny : capped ? kCapped : kPlain;
  }
  __syncthreads();

  // Where the list may have all that may be kept: from which order on.  Up to kCap / 8 groups give some kCap / 8 * ln(kCap / 8) candidates,
  // which a list holds; of more groups it would not.
  uint32_t from = 0;
  if (p.vocabulary <= kCap && (rules.by_count || rules.by_sum)) {
    from = kNothing + 1;
  } else if (rules.by_count) {
    if (top_k <= kCap / 8) from = lower;
  } else if (rules.by_floor) {
    // Nothing further below the largest than this has a share of min_p (a share next to it may be rounded to it: at high temperatures many are one).
    const double y = value_below(sh.row, degrees, 1e-12 - log(rules.min_p));
    const float bound = y > static_cast<double>(most) ? most : __double2float_rd(y);
    from = bound == bound ? max(order_of(bound), kNothing + 1) : kNothing + 1;
  }
  const auto part = Walk<T, kThreads>::mine();
  int which = 0;  // of the slots that the next exchange takes
  int listed = -1;  // entries of a list that has all
  double whole_sum = -1.0;
  if (from != 0) {
    const int count = gather<T, kThreads>(from, largest, most, false, false, false, which).count;
    which ^= 1;
    if (count <= kCap) listed = count;
    if (listed >= 0 && rules.by_sum && !rules.by_count && p.vocabulary > kCap) {  // (the list is what the floor leaves: top_p is of all)
      whole_sum = cluster_sums<kThreads>(sum_shares<T, kThreads>(part.begin, part.end, 0.0), 0.0, 0.0, which).a;
      which ^= 1;
    }
  }
  double above_mine = 0.0;  // this lane's part of the sum above what the list has
  bool begun = false;
#pragma unroll 1
  for (int rule = 0; rule < 2 && listed < 0; ++rule) {  // top_k, then top_p
    if (rule == 0 ? !rules.by_count : !rules.by_sum) continue;
    const bool shares = rule == 1;
    // Counts: from the bound that the groups gave.  Shares: n values below a share of (1 - top_p) / n have less than 1 - top_p together, which is less
    // than what top_p leaves out (the largest alone has a share of one), so the border is above that; but no further than 24 temperatures (2^-35 of the
    // largest), or bins would be wide: where the border is further down, halving finds it.
    const uint32_t border_key = sh.row.border_key;
    const double bottom = static_cast<double>(most) - 24.0 * degrees;
    const double reach = shares ? value_below(sh.row, degrees, logf((rules.by_count ? top_k : p.vocabulary) / (1.0f - top_p)) + 0.01f) : bottom;
    bool surely = reach >= bottom;
    const uint32_t near = max(order_of(__double2float_rd(fmax(reach, bottom))), border_key);
    uint32_t low = min(shares || value_of(lower) < -1e30f ? near : lower, largest), high = largest;
    uint32_t sure_low = border_key, sure_high = largest;  // the border lies between these
    double target = top_k, above = 0.0, all = 0.0;
    float seen = most;  // what is above has been measured
    bool done = false, known = !shares;  // (whether the target is)
    above_mine = 0.0;
#pragma unroll 1
    for (int turn = 0; turn < 5; ++turn) {
      const Bins bins = bins_between(value_of(low), value_of(high));
      if (turn == 0) {
        clear_bins<kThreads>();
        const float sum = look<T, kThreads>(bins, shares);
        all = cluster_sums<kThreads>(sum, 0.0, 0.0, which).a;
        which ^= 1;
        if (shares) target = rules.top_p * all;
      }
      // By how much, as an exponent, shares by middles are off.  A value is half a bin from its middle at most, and 0.005 for what the bin's number loses
      // (three roundings of 2^-24 of up to 1023); the middle is off by up to three roundings of at most `size`, or of 2^-149 where that is subnormal;
      // capped values in 32 bits by 5e-7 of the cap each, the largest and another (an exponential off by 2^-22 of up to one, of which a softened
      // value takes at most half, a reciprocal by 2^-23 and six roundings).  The rest is within 2.5e-5 of 1e-4: 259 additions of a lane and 21 of bins
      // (2^-24 each: 1.7e-5), exponents of up to 24 temperatures from three roundings (4.3e-6, and on a row's average, which is ln of its size,
      // 2.3e-6), exponentials (2^-22).
      const double size = fmax(fabs(static_cast<double>(bins.high)), fabs(static_cast<double>(bins.low)));
      const double off = shares ? (1.01 / static_cast<double>(bins.per_two) + 0x1p-22 * size + 0x1p-147 + (capped ? 1e-6 * p.softcap : 0.0)) / degrees + 1e-4 : 0.0;
      const BinWindow window = window_of_bins<kThreads>(bins, shares, above, target, off, surely, turn);
      if (window.says == kNotHere || low == high) break;
      if (window.says == kInList || window.says == kListHasAll) {
        const uint32_t next_low = order_with(bins, window.last, low, high);
        const uint32_t next_high = window.first > 0 ? order_below(order_with(bins, window.first - 1, low, high)) : high;
        const bool has_all = window.says == kListHasAll;
        const Gathered got = gather<T, kThreads>(next_low, next_high, seen, !has_all, shares, !known, which);
        which ^= 1;
        if (!known) {
          all = got.sums.all;
          target = rules.top_p * all;
          known = true;
        }
        if (has_all && got.count <= kCap) {
          listed = got.count;
          whole_sum = shares ? all : -1.0;
          break;
        }
        done = got.count > 0 && got.count <= kCap && border_from_list<kThreads>(got.count, shares, above + got.sums.above, target, false);
        if (done) {
          if (shares) {
            begun = !rules.by_floor || share<kThreads>(sh.row.border) >= rules.min_p;  // (else some above the border go too)
            above_mine += got.sifted.above;
          }
          break;
        }
      }
      // Closer.
      if (window.sure_last >= kBins) break;
      surely = true;
      const uint32_t next_low = order_with(bins, window.sure_last, low, high);
      const uint32_t next_high = window.sure_first > 0 ? order_below(order_with(bins, window.sure_first - 1, low, high)) : high;
      if (next_low == low && next_high == high) break;
      const float lowest = value_of(next_low), highest = value_of(next_high);
      clear_bins<kThreads>();
      const Sifted sifted = sift_row<T, kThreads>(true, lowest, highest, seen, true, shares, !known, bins_between(lowest, highest));
      const Three sums = cluster_sums<kThreads>(sifted.above, sifted.all, 0.0, which);
      which ^= 1;
      above_mine += sifted.above;
      above += sums.a;
      if (!known) {
        all = sums.b;
        target = rules.top_p * all;
        known = true;
      }
      seen = highest;
      sure_low = low = next_low;
      sure_high = high = next_high;
    }
    if (!done && listed < 0) {
      if (!known) {
        const double mine = sum_shares<T, kThreads>(part.begin, part.end, 0.0);
        target = rules.top_p * cluster_sums<kThreads>(mine, 0.0, 0.0, which).a;
        which ^= 1;
      }
      which = find_border<T, kThreads>(shares, target, sure_low, sure_high, above, which);
    }
  }
  if (listed >= 0) {
    if (rank == 0) {
      const Taken taken = finish<kThreads>(listed, whole_sum, rules, most);
      if (taken.index >= 0) answer(taken.index, taken.probability);
    }
    return;
  }
  // The kept shares in the order of the vocabulary; what is above the border's window has been summed.
  const double least = rules.by_floor ? rules.min_p : 0.0;
  const double mine = begun ? above_mine + sum_listed<T, kThreads>() : sum_shares<T, kThreads>(part.begin, part.end, least);
  const Located it = locate<T, kThreads>(mine, false, 0.0f, least, rules.u, which);
  if (it.index >= 0) answer(it.index, static_cast<float>(it.weight / it.all));
}

template <typename T, int kThreads>
cudaError_t launch_threads(const SampleCall& call, int ctas, cudaStream_t stream) {
  constexpr int kE = Vector<T>::kValues;
  SampleParams p{call, ctas, 0};
  // As many vectors for each warp (with the lead at its largest, where rows do not begin at a 16-byte boundary).
  const bool whole = (reinterpret_cast<uintptr_t>(call.logits) & 15) == 0 && (call.row_stride * sizeof(T) & 15) == 0;
  const int vectors = (call.vocabulary + (whole ? 0 : kE - 1) + kE - 1) / kE, warps = ctas * (kThreads / 32);
  p.cta_vectors = (vectors + warps - 1) / warps * (kThreads / 32);
  static std::atomic<unsigned long long> allowed{0};
  const cudaError_t e = allow_clusters(sample_kernel<T, kThreads>, sizeof(SampleShared<kThreads>), &allowed);
  if (e != cudaSuccess) return e;
  return launch_chained_clusters(sample_kernel<T, kThreads>, ctas, dim3(static_cast<unsigned>(call.rows) * ctas), dim3(kThreads),
                                 sizeof(SampleShared<kThreads>), stream, p);
}

template <typename T>
cudaError_t launch_type(const SampleCall& call, int sm_count, cudaStream_t stream) {
  const long long bytes = static_cast<long long>(call.vocabulary) * sizeof(T);
  if (bytes <= 4096) return launch_threads<T, 128>(call, 1, stream);
  // Two CTAs an SM take as many rows as there are; where there are fewer, as many CTAs a row as that leaves, down to 8 KB each.  With rules to find
  // borders for, rows take up to five times as long as one another: twice as many CTAs then (64 rows of 262144, each with rules of its
  // own, 243 -> 146 us when they took that; 256 rows of 128000 by top_p 300 -> 265; without rules 256 rows of 50257 would go 38 -> 47, which a call
  // pays whose settings are given and keep all: they are the device's to read).
  const long long ctas_at_once = (call.top_k || call.top_p || call.min_p ? 4ll : 2ll) * sm_count;
  int ctas = 1;
  while (ctas < kMostCtas && 2ll * ctas * call.rows <= ctas_at_once && bytes > 16384ll * ctas) ctas *= 2;
  return launch_threads<T, 256>(call, ctas, stream);
}

}  // namespace

cudaError_t launch_sample(const SampleCall& call, int sm_count, cudaStream_t stream) {
  return call.wide ? launch_type<float>(call, sm_count, stream) : launch_type<__nv_bfloat16>(call, sm_count, stream);
}

}  // namespace gv
