// Tokens from logits (declared in include/gevva_moe.h): temperature, top-k, top-p and min-p, from one given random number a row.
//
// With y = x, or cap * tanh(x / cap), a token's share is w = exp((y - y_max) / T).  Tokens are ranked by x, ties by index; kept are the ranks below
// top_k, those whose better ranks have less than top_p of what top_k leaves, and those with w >= min_p.  The token is the first of the
// vocabulary at which the sum of kept shares passes u times the sum of all kept ones.
//
// Floor: a row is read once.  A cluster of up to 16 CTAs holds a row in shared memory (two CTAs an SM: one row's reads run under another's work), and
// every further pass goes over shared memory:
//   1. the largest value, and for groups of threads of every size the smallest of their largest values: with at least k groups, at least k
//      values are not below that, and with about k groups only some k ln k are.
//   2. where a border by top_p, or by a large top_k, has to be found: all shares' sum, and how many values lie in each 32nd of an octave of
//      share.  From these counts the border is known to a few of them.
//   3. what may be kept goes to the first CTA's list, which sorts it, cuts it and walks over it; where more may be kept than a list holds, what lies
//      about the border goes there, with the sum of the shares above it.
//   4. then the kept shares are summed by CTAs, warps and steps in the order of the vocabulary, and the step that holds the token is walked over.
// The counts only say where to look: the border itself is taken from sums of shares in 64 bits, and where it does not lie in the list (values too
// many, too equal or too far apart for the counts) it is looked for by halving the range, a pass over shared memory a step.
// All sums are taken in an order that sizes alone give: the same inputs give the same token.
#include "gv_common.cuh"
#include "gv_shares.h"
#include "gv_step.h"

namespace gv {
namespace {

constexpr int kMostCtas = 16;
constexpr int kLevels = 10;     // groups of 2^level threads
constexpr int kSums = 3;
constexpr int kBins = 1024;     // of a 32nd of an octave of share; the last one has all that is smaller
constexpr int kTableCopies = 16;  // of the table of 2^(j/32), one for each lane of half a warp: no two lanes of a read meet in a bank

struct SampleParams {
  SampleCall call;
  int ctas;         // of a row's cluster
  int cta_vectors;  // 16-byte vectors of a row that a CTA holds
};

// Where the counts say that a border lies: bins first .. last hold it, and what is in front of them measures `above`.
struct BinWindow {
  int first, last;
  int count;     // in the window
  int whole;     // 1: the window has all from the largest value on (first is 0)
};

template <int kThreads>
struct SampleShared {
  static constexpr int kCap = 4 * kThreads;
  static constexpr int kWarps = kThreads / 32;
  double table[kExp2Entries * kTableCopies];
  unsigned long long mine[kCap];   // candidates of this CTA
  unsigned long long list[kCap];   // the cluster's, in its first CTA
  uint4 first[kMostCtas][4];       // largest key, its index, levels, settings
  double slots[2][kMostCtas][kSums];
  double warp_sums[kWarps][kSums];
  uint4 window;                    // a BinWindow, from the first CTA
  unsigned long long border;       // from the first CTA
  int bins[kBins];
  uint32_t warp_key[kWarps], warp_index[kWarps], warp_levels[kWarps][5];
  int mine_count, list_count, base, found;
  int edges[4];
};

__device__ __forceinline__ void cluster_store_double(uint32_t address, double v) {
  asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(address), "l"(__double_as_longlong(v)) : "memory");
}
__device__ __forceinline__ void cluster_store_u64(uint32_t address, unsigned long long v) {
  asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(address), "l"(v) : "memory");
}
__device__ __forceinline__ int cluster_load(uint32_t address) {
  int v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(address) : "memory");
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

template <typename T>
struct Vector;
template <>
struct Vector<float> {
  static constexpr int kValues = 4;
  static __device__ __forceinline__ void unpack(const uint4& v, float (&x)[4]) {
    x[0] = __uint_as_float(v.x);
    x[1] = __uint_as_float(v.y);
    x[2] = __uint_as_float(v.z);
    x[3] = __uint_as_float(v.w);
  }
};
template <>
struct Vector<__nv_bfloat16> {
  static constexpr int kValues = 8;
  static __device__ __forceinline__ void unpack(const uint4& v, float (&x)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};

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
    while (whole < count) whole *= 2;
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

// How shares are worked out: from 32 bits' whole part where temperature and values are of ordinary size, of capped values, or of any.
enum ShareForm : int { kPlain, kCapped, kAny };

__device__ __noinline__ double softened(float x, double cap) {
  // tanh(z) = 1 - 2 / (1 + exp(2 z)), of |z|
  const double z = fabs(static_cast<double>(x)) / cap;
  const double y = cap * (1.0 - 2.0 / (1.0 + exp(2.0 * z)));
  return x < 0.0f ? -y : y;
}

// The share of any value that may be taken, and its bin.
struct BinnedShare {
  double share;
  int bin;
};
__device__ __noinline__ BinnedShare other_share(float x, ShareForm form, double scale, double top, double cap, const double* table) {
  double distance = form == kCapped ? softened(x, cap) - top : static_cast<double>(x) - top;
  if (form == kAny) {
    if (isinf(x)) distance = 0.0;  // (the largest value is infinite then, and so is this one)
    else if (isinf(top)) return {0.0, kBins - 1};
  }
  const double at = -distance * scale;
  return {share_of(distance, scale, table, kTableCopies), at < kBins - 1 ? static_cast<int>(at + 0.5) : kBins - 1};
}

template <typename T, int kThreads>
struct Row {
  static constexpr int kE = Vector<T>::kValues;
  using Shared = SampleShared<kThreads>;
  static constexpr int kWarps = Shared::kWarps, kCap = Shared::kCap;

  Shared& sh;
  const uint4* slice;  // this CTA's part of the row
  int vectors;         // of it
  int begin_index;     // vocabulary index of its first value
  int ctas, rank;
  int lane, warp;
  int parity = 0;

  // shares
  ShareForm form;
  double scale, top, cap;  // of y
  float scale32, top32, cut;  // smaller values have no share (kPlain)
  // what top_k and top_p keep: order above border_key, or equal to it and index up to border_index
  bool bounded = false;
  uint32_t border_key = kNothing + 1, border_index = 0xffffffffu;

  __device__ __forceinline__ const double* table() const { return sh.table + (lane & (kTableCopies - 1)); }
  __device__ __forceinline__ uint32_t plain_whole(float x) const { return share_whole(x - top32, scale32); }
  __device__ __forceinline__ double plain_share(float x, uint32_t whole) const {
    return share_with(static_cast<double>(x) - top, scale, whole, table(), kTableCopies);
  }
  __device__ __forceinline__ BinnedShare other(float x) const { return other_share(x, form, scale, top, cap, table()); }
  __device__ __forceinline__ double share(float x) const {
    if (form == kPlain) return x >= cut ? plain_share(x, plain_whole(x)) : 0.0;
    return other(x).share;
  }
  static __device__ __forceinline__ int plain_bin(uint32_t whole) { return min(max(static_cast<int>(kShareWhole - whole), 0), kBins - 1); }
  __device__ __forceinline__ int bin_of(float x) const {
    if (form == kPlain) return x >= cut ? plain_bin(plain_whole(x)) : kBins - 1;
    return other(x).bin;
  }
  __device__ __forceinline__ bool inside(float x, uint32_t index) const {
    const float border = value_of(border_key);
    return x > border || (x == border && index <= border_index);
  }

  // A warp has vectors that follow one another, in steps of 32.
  __device__ __forceinline__ int warp_vectors() const { return (vectors + kWarps * 32 - 1) / (kWarps * 32) * 32; }

  template <class F>
  __device__ __forceinline__ void one_vector(int v, F&& f) const {
    float x[kE];
    Vector<T>::unpack(slice[v], x);
#pragma unroll
    for (int i = 0; i < kE; ++i) f(x[i], begin_index + v * kE + i);
  }
  template <class F>
  __device__ __forceinline__ void each_value(F&& f) const {
    const int each = warp_vectors(), end = min(vectors, (warp + 1) * each);
#pragma unroll 1
    for (int v = warp * each + lane; v < end; v += 32) one_vector(v, f);
  }

  __device__ __forceinline__ void cluster_barrier() {
    __syncwarp();
    if (ctas > 1) cluster_sync_all();
    else __syncthreads();
  }

  // Sums over the cluster, in every thread the same; sh.slots[which][rank] has the CTAs' own, sh.warp_sums the warps' of this one.
  template <int kCount>
  __device__ __forceinline__ int cluster_sums(double (&v)[kCount]) {
#pragma unroll
    for (int i = 0; i < kCount; ++i) v[i] = warp_sum(v[i]);
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < kCount; ++i) sh.warp_sums[warp][i] = v[i];
    }
    __syncthreads();
    const int which = parity;
    parity ^= 1;
    if (warp == 0 && lane < ctas) {
      const uint32_t peer = cluster_map_shared(smem_u32(&sh.slots[which][rank][0]), lane);
#pragma unroll
      for (int i = 0; i < kCount; ++i) {
        double sum = 0.0;
        for (int w = 0; w < kWarps; ++w) sum += sh.warp_sums[w][i];
        cluster_store_double(peer + 8 * i, sum);
      }
    }
    cluster_barrier();
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      v[i] = 0.0;
      for (int r = 0; r < ctas; ++r) v[i] += sh.slots[which][r][i];
    }
    return which;
  }

  // What lies from `low` to `high` in order and is inside goes to the first CTA's list; returns how many there are in all (more
  // than kCap: the list is not whole).  above(x, index) is called for what is inside and higher.
  template <class Above>
  __device__ __forceinline__ int gather(uint32_t low, uint32_t high, Above&& above) {
    const float from = value_of(low), upto = value_of(high);
    if (threadIdx.x == 0) sh.mine_count = 0;
    __syncthreads();
    const bool all = !bounded;
    each_value([&](float x, int index) {
      if (x >= from && (all || inside(x, index))) {
        if (x <= upto) {
          const int at = atomicAdd(&sh.mine_count, 1);
          if (at < kCap) sh.mine[at] = static_cast<unsigned long long>(~order_of(x)) << 32 | static_cast<uint32_t>(index);
        } else {
          above(x);
        }
      }
    });
    __syncthreads();
    const int count = sh.mine_count;
    const int which = parity;
    parity ^= 1;
    if (warp == 0) {
      if (lane < ctas) cluster_store_double(cluster_map_shared(smem_u32(&sh.slots[which][rank][0]), lane), static_cast<double>(count));
      if (lane == 0) sh.base = count > 0 && count <= kCap ? cluster_add(cluster_map_shared(smem_u32(&sh.list_count), 0), count) : kCap;
    }
    __syncthreads();
    if (count <= kCap) {
      const uint32_t list = cluster_map_shared(smem_u32(sh.list), 0);
      const int base = sh.base;
      for (int i = threadIdx.x; i < count; i += kThreads)
        if (base + i < kCap) cluster_store_u64(list + 8 * (base + i), sh.mine[i]);
    }
    cluster_barrier();
    double sum = 0.0;
    for (int r = 0; r < ctas; ++r) sum += sh.slots[which][r][0];
    if (threadIdx.x == 0) sh.list_count = 0;  // (for the next gathering, which a barrier comes before)
    return static_cast<int>(sum);
  }

  // Sums up to each of a thread's four entries of the list, over the whole CTA; returns the sum of all.
  __device__ __forceinline__ double list_upto(const double (&w)[4], double (&upto)[4], double& in_front) {
    const double inclusive = warp_upto(w[0] + w[1] + w[2] + w[3]);
    if (lane == 31) sh.warp_sums[warp][0] = inclusive;
    __syncthreads();
    double before = 0.0, all = 0.0;
    for (int v = 0; v < kWarps; ++v) {
      if (v == warp) before = all;
      all += sh.warp_sums[v][0];
    }
    const double previous = __shfl_up_sync(0xffffffffu, inclusive, 1);
    in_front = before + (lane > 0 ? previous : 0.0);
    double sum = in_front;
#pragma unroll
    for (int j = 0; j < 4; ++j) upto[j] = sum += w[j];
    __syncthreads();
    return all;
  }
  static __device__ __forceinline__ float ranked_value(unsigned long long entry) { return value_of(~static_cast<uint32_t>(entry >> 32)); }

  // In the list, sorted by rank: the first at which `above` and the measure of the entries up to it come to `target`; count: none does.
  __device__ __forceinline__ int list_border(int count, bool shares, double above, double target) {
    double w[4], upto[4], in_front;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = 4 * threadIdx.x + j;
      w[j] = i >= count ? 0.0 : shares ? share(ranked_value(sh.list[i])) : 1.0;
    }
    if (threadIdx.x == 0) sh.found = count;
    list_upto(w, upto, in_front);
#pragma unroll
    for (int j = 3; j >= 0; --j) {
      const int i = 4 * threadIdx.x + j;
      if (i < count && above + upto[j] >= target) atomicMin(&sh.found, i);
    }
    __syncthreads();
    return sh.found;
  }

  // The border out of the first CTA's list of `count`, in all CTAs; false: it is not there.  (`surely`: the last entry where rounding leaves none.)
  __device__ __forceinline__ bool border_from_list(int count, bool shares, double above, double target, bool surely) {
    if (rank == 0) {
      sort_list<kThreads>(sh.list, count);
      int at = above < target || surely ? list_border(count, shares, above, target) : count;
      if (surely && count > 0) at = min(at, count - 1);
      const unsigned long long entry = at < count ? sh.list[at] : 0;
      if (warp == 0 && lane < ctas) cluster_store_u64(cluster_map_shared(smem_u32(&sh.border), lane), entry);
    }
    cluster_barrier();
    const unsigned long long entry = sh.border;
    if (entry == 0) return false;  // (no value that may be taken has the complement of zero for its order)
    border_key = ~static_cast<uint32_t>(entry >> 32);
    border_index = static_cast<uint32_t>(entry);
    bounded = true;
    return true;
  }

  // ---- by counts of values in 32nds of an octave of share

  // The smallest order with a bin of at most `bin` (the largest value's is 0); searched by 32 lanes at a time.
  __device__ __forceinline__ uint32_t order_with(int bin, uint32_t largest) const {
    uint32_t low = kNothing + 1, high = largest;
    while (low < high) {
      const uint32_t step = (high - low) / 32 + 1, at = min(low + step * lane, high);
      const uint32_t yes = __ballot_sync(0xffffffffu, bin_of(value_of(at)) <= bin);  // ascending: none, then all
      if (yes & 1) return low;
      const int first = yes ? __ffs(yes) - 1 : 32;
      const uint32_t next = min(low + step * first, high);
      low = min(low + step * (first - 1) + 1, next);
      high = next;
    }
    return low;
  }

  // Counts what is inside by bins and, with `shares`, sums its shares; `sum` is of the cluster.
  __device__ __forceinline__ void count_bins(bool shares, double& sum) {
    for (int i = threadIdx.x; i < kBins; i += kThreads) sh.bins[i] = 0;
    __syncthreads();
    double v[1] = {0.0};
    if (form == kPlain && !bounded) {
      const float from = cut;
      if (shares) {
        each_value([&](float x, int) {
          const uint32_t whole = plain_whole(x);
          const double w = plain_share(x, whole);
          if (x >= from) {
            v[0] += w;
            atomicAdd(&sh.bins[plain_bin(whole)], 1);
          }
        });
      } else {
        each_value([&](float x, int) {
          if (x >= from) atomicAdd(&sh.bins[plain_bin(plain_whole(x))], 1);
        });
      }
    } else {
      each_value([&](float x, int index) {
        if (inside(x, index)) {
          const BinnedShare it = form == kPlain ? BinnedShare{share(x), bin_of(x)} : other(x);
          v[0] += it.share;
          atomicAdd(&sh.bins[it.bin], 1);
        }
      });
    }
    cluster_sums(v);
    sum = v[0];
  }

  // Where the counts say that the first `target` (shares, or values) end.  Counts times the shares of their bins' middles are off by up to 1.1 %:
  // so far to both sides, or, where that is more than the list holds, a tenth of it.  No border among the bins: count is zero.
  __device__ __forceinline__ BinWindow window_of_bins(bool shares, double target) {
    if (rank == 0) {
      constexpr int kEach = kBins / kThreads;
      int count[kEach];
      double mass[kEach], counted = 0.0, massed = 0.0;
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int bin = threadIdx.x * kEach + i;
        const uint32_t at = smem_u32(&sh.bins[bin]);
        count[i] = 0;
        for (int r = 0; r < ctas; ++r) count[i] += cluster_load(cluster_map_shared(at, r));
        // (what the last bin has lies at any distance: it is no place for a border)
        mass[i] = bin == kBins - 1 ? 0.0 : count[i] * scaled_by(table()[((0u - bin) & (kExp2Entries - 1)) * kTableCopies], 0u - bin);
        if (bin == kBins - 1) count[i] = 0;
        counted += count[i];
        massed += mass[i];
      }
      const double counts = warp_upto(counted), masses = warp_upto(massed);
      if (lane == 31) {
        sh.warp_sums[warp][0] = counts;
        sh.warp_sums[warp][1] = masses;
      }
      if (threadIdx.x < 4) sh.edges[threadIdx.x] = kBins;
      __syncthreads();
      double count_upto = counts - counted, mass_upto = masses - massed;
      for (int w = 0; w < warp; ++w) {
        count_upto += sh.warp_sums[w][0];
        mass_upto += sh.warp_sums[w][1];
      }
      const double most = target * (1.0 + 0.011), least = target * (1.0 - 0.011), more = target * (1.0 + 0.0011), less = target * (1.0 - 0.0011);
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        const int bin = threadIdx.x * kEach + i;
        count_upto += count[i];
        mass_upto += mass[i];
        sh.bins[bin] = static_cast<int>(count_upto);
        const double upto = shares ? mass_upto : count_upto;
        if (count[i] > 0) {
          if (upto >= (shares ? least : target)) atomicMin(&sh.edges[0], bin);
          if (upto >= (shares ? most : target)) atomicMin(&sh.edges[1], bin);
          if (upto >= (shares ? less : target)) atomicMin(&sh.edges[2], bin);
          if (upto >= (shares ? more : target)) atomicMin(&sh.edges[3], bin);
        }
      }
      __syncthreads();
      if (warp == 0) {
        BinWindow window{};
        for (int wide = 0; wide < 4 && window.count == 0; wide += 2) {
          const int first = sh.edges[wide];
          if (first == kBins) break;
          const int last = min(sh.edges[wide + 1], kBins - 2);
          const int in_front = first > 0 ? sh.bins[first - 1] : 0, upto = sh.bins[last];
          // (all of it only where it surely reaches the target)
          if (upto <= kCap && sh.edges[wide + 1] < kBins - 1 && (wide == 0 || !shares)) window = BinWindow{0, last, upto, 1};
          else if (upto - in_front <= kCap) window = BinWindow{first, last, upto - in_front, 0};
        }
        if (lane < ctas)
          cluster_store_uint4(cluster_map_shared(smem_u32(&sh.window), lane), make_uint4(window.first, window.last, window.count, window.whole));
      }
    }
    cluster_barrier();
    const uint4 w = sh.window;
    return BinWindow{static_cast<int>(w.x), static_cast<int>(w.y), static_cast<int>(w.z), static_cast<int>(w.w)};
  }

  // ---- by halving

  // The value, and among its ties the index, at which the measure (shares, or how many) of what is inside and ranks up to there comes to
  // `target`.  Sets the border; none where all that is inside does not come to it.
  __device__ __forceinline__ void find_border(bool shares, double target, uint32_t low, uint32_t high) {
    double above = 0.0, count = 2.0 * kCap;  // what is higher than `high` measures; how many lie from `low` to `high` (at first: many)
    for (int step = 0; low < high && count > kCap; ++step) {  // (every other step halves the range of orders: it ends in 64)
      const float middle = 0.5f * value_of(low) + 0.5f * value_of(high);
      uint32_t mid = step & 1 ? low + (high - low) / 2 : order_of(middle);
      mid = max(low, min(mid, order_below(high)));
      if (mid == 0x7fffffffu) mid = high > 0x80000000u ? 0x80000000u : 0x7ffffffeu;
      const float from = value_of(mid), bottom = value_of(low), upto = value_of(high);
      double v[3] = {0.0, 0.0, 0.0};  // how many, how many above the middle, what those measure
      each_value([&](float x, int index) {
        if (x >= bottom && x <= upto && inside(x, index)) {
          v[0] += 1.0;
          if (x > from) {
            v[1] += 1.0;
            if (shares) v[2] += share(x);
          }
        }
      });
      cluster_sums(v);
      const double measure = shares ? v[2] : v[1];
      if (above + measure >= target) {
        low = order_above(mid);
        count = v[1];
      } else {
        high = mid;
        above += measure;
        count = v[0] - v[1];
        if (count == 0.0) return;  // (there are not as many: all stay)
      }
    }
    if (low < high || count <= kCap) {
      const int gathered = gather(low, high, [](float) {});
      if (gathered <= kCap) {
        border_from_list(gathered, shares, above, target, true);
        return;
      }
    }
    // More ties than the list holds: so many of them, in the order of the vocabulary.
    const float value = value_of(low);
    double v[1] = {0.0};
    each_value([&](float x, int index) { v[0] += x == value && inside(x, index) ? 1.0 : 0.0; });
    cluster_sums(v);
    double ties = target - above;
    if (shares) ties /= share(value);
    ties = fmin(fmax(ceil(ties), 1.0), v[0]);
    const auto one = [&](float x, int i) { return x == value && inside(x, i) ? 1.0 : 0.0; };
    locate(
        0.0, one, one, [&](double) { return ties - 0.5; },
        [&](float, int i, double, double) {
          for (int r = 0; r < ctas; ++r) cluster_store_u64(cluster_map_shared(smem_u32(&sh.border), r), static_cast<unsigned long long>(static_cast<uint32_t>(i)));
        });
    cluster_barrier();
    border_key = low;
    border_index = static_cast<uint32_t>(sh.border);
    bounded = true;
  }

  // The first value of the vocabulary at which the sum of weights passes target_of(sum of all weights): found(value, index, weight, sum of all)
  // in one thread.  A lane's weights are `begun` and what rest(value, index) gives of each value.
  template <class Rest, class W, class Target, class Found>
  __device__ __forceinline__ void locate(double begun, Rest&& rest, W&& weight, Target&& target_of, Found&& found) {
    double v[1] = {begun};
    each_value([&](float x, int index) { v[0] += rest(x, index); });
    const int which = cluster_sums(v);
    const double all = v[0], target = target_of(all);
    // the CTA: the last with any weight where rounding leaves the target above all sums
    int cta = -1, last = 0;
    double front = 0.0, last_front = 0.0, sum = 0.0;
    for (int r = 0; r < ctas; ++r) {
      const double own = sh.slots[which][r][0];
      if (own > 0.0) {
        last = r;
        last_front = sum;
      }
      if (cta < 0 && sum + own > target) {
        cta = r;
        front = sum;
      }
      sum += own;
    }
    if (cta < 0) {
      cta = last;
      front = last_front;
    }
    if (rank != cta || !(all > 0.0)) return;
    // its warp, in the same way
    int in_warp = -1;
    double warp_front = 0.0;
    sum = front;
    last = 0;
    last_front = front;
    for (int w = 0; w < kWarps; ++w) {
      const double own = sh.warp_sums[w][0];
      if (own > 0.0) {
        last = w;
        last_front = sum;
      }
      if (in_warp < 0 && sum + own > target) {
        in_warp = w;
        warp_front = sum;
      }
      sum += own;
    }
    if (in_warp < 0) {
      in_warp = last;
      warp_front = last_front;
    }
    // its steps are summed by as many warps at a time, and the step that holds the target is walked through by one
    const int each = warp_vectors(), begin = in_warp * each, end = min(vectors, begin + each), steps = (end - begin + 31) / 32;
    double reached = warp_front;
    int last_step = 0;
    double last_reached = warp_front;
    for (int base = 0; base < steps; base += kWarps) {
      const int at = begin + (base + warp) * 32 + lane;
      double own = 0.0;
      if (at < end) one_vector(at, [&](float x, int index) { own += weight(x, index); });
      own = warp_sum(own);
      if (lane == 0) sh.warp_sums[warp][1] = own;
      __syncthreads();
      int hit = -1;
      double hit_front = 0.0;
      for (int w = 0; w < kWarps && base + w < steps; ++w) {
        const double one = sh.warp_sums[w][1];
        if (one > 0.0) {
          last_step = base + w;
          last_reached = reached;
        }
        if (hit < 0 && reached + one > target) {
          hit = base + w;
          hit_front = reached;
        }
        reached += one;
      }
      __syncthreads();
      if (hit >= 0 || base + kWarps >= steps) {
        const int step = hit >= 0 ? hit : last_step;
        const double step_front = hit >= 0 ? hit_front : last_reached;
        if (warp == 0) {
          const int v_at = begin + step * 32 + lane;
          double mine = 0.0;
          if (v_at < end) one_vector(v_at, [&](float x, int index) { mine += weight(x, index); });
          const double upto = warp_upto(mine), previous = __shfl_up_sync(0xffffffffu, upto, 1);
          const double lane_front = step_front + (lane > 0 ? previous : 0.0);
          const uint32_t passing = __ballot_sync(0xffffffffu, mine > 0.0 && step_front + upto > target);
          const uint32_t some = __ballot_sync(0xffffffffu, mine > 0.0);
          const int chosen = passing ? __ffs(passing) - 1 : 31 - __clz(some);
          if (lane == chosen) {
            double running = lane_front;
            float value = 0.0f;
            int index = -1;
            double taken = 0.0;
            bool done = false;
            one_vector(v_at, [&](float x, int i) {
              const double w = weight(x, i);
              if (!done && w > 0.0) {
                value = x;
                index = i;
                taken = w;
              }
              running += w;
              if (w > 0.0 && running > target) done = true;
            });
            found(value, index, taken, all);
          }
        }
        break;
      }
    }
  }
};

template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) sample_kernel(const SampleParams params) {
  using R = Row<T, kThreads>;
  constexpr int kE = R::kE, kWarps = R::kWarps, kCap = R::kCap;
  static __shared__ SampleShared<kThreads> sh;
  extern __shared__ uint4 held[];
  const SampleCall& p = params.call;
  const int ctas = params.ctas, row = blockIdx.x / ctas, rank = blockIdx.x - row * ctas;  // (a cluster is CTAs that follow one another)
  const int thread = threadIdx.x, lane = thread & 31, warp = thread >> 5;
  for (int i = thread; i < kExp2Entries * kTableCopies; i += kThreads) sh.table[i] = g_exp2_table[i / kTableCopies];
  if (thread == 0) sh.list_count = 0;
  if (ctas > 1) cluster_arrive();  // (a CTA writes to the others when all have begun)
  grid_launch_dependents();
  grid_dependency_wait();

  // The row from the 16-byte boundary at or in front of its first value: what a vector has of other rows, or of the bytes in front of
  // and behind the tensor (of the same 16, and so of the same allocation), counts as nothing.
  const T* const data = static_cast<const T*>(p.logits) + row * p.row_stride;
  const int lead = static_cast<int>((reinterpret_cast<uintptr_t>(data) & 15) / sizeof(T));
  const uint4* const source = reinterpret_cast<const uint4*>(data - lead);
  const int whole = (lead + p.vocabulary + kE - 1) / kE;  // vectors of the row
  const int first_vector = min(whole, rank * params.cta_vectors);
  R me{sh, held, min(whole - first_vector, params.cta_vectors), first_vector * kE - lead, ctas, rank, lane, warp};

  // settings of the row, read while its values are on their way
  const int each = me.warp_vectors(), end = min(me.vectors, (warp + 1) * each);
  for (int v = warp * each + lane; v < end; v += 32)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(held + v)), "l"(source + first_vector + v) : "memory");
  asm volatile("cp.async.commit_group;" ::: "memory");
  float temperature = p.temperature ? p.temperature[row] : 1.0f;
  int top_k = p.top_k ? p.top_k[row] : 0;
  float top_p = p.top_p ? p.top_p[row] : 1.0f, floor = p.min_p ? p.min_p[row] : 0.0f;
  const double u = fmin(fmax(static_cast<double>(p.uniforms[row]), 0.0), 1.0 - 0x1p-24);  // (not a number: zero)
  asm volatile("cp.async.wait_all;" ::: "memory");

  // ---- the largest value, the lowest index that has it, and the levels
  float highest = -INFINITY;
  for (int v = warp * each + lane; v < end; v += 32) {
    const int at = me.begin_index + v * kE;
    if (at < 0 || at + kE > p.vocabulary) {
      T values[kE];
      memcpy(values, held + v, 16);
#pragma unroll
      for (int i = 0; i < kE; ++i)
        if (at + i < 0 || at + i >= p.vocabulary) values[i] = static_cast<T>(-INFINITY);
      memcpy(held + v, values, 16);
    }
    me.one_vector(v, [&](float x, int) { highest = fmaxf(highest, x); });  // (of a number and none, the number)
  }
  const uint32_t key = order_of(highest);
  {
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
  if (warp != 0 && ctas > 1) cluster_wait();
  if (warp == 0) {
    const bool mine = lane < kWarps;
    uint32_t out[16];
    uint32_t group = mine ? sh.warp_key[lane] : 0;
    const uint32_t most = __reduce_max_sync(0xffffffffu, group);
    out[0] = most;
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
    if (ctas > 1) cluster_wait();
    if (lane < ctas) {
      const uint32_t peer = cluster_map_shared(smem_u32(&sh.first[rank][0]), lane);
#pragma unroll
      for (int i = 0; i < 4; ++i) cluster_store_uint4(peer + 16 * i, make_uint4(out[4 * i], out[4 * i + 1], out[4 * i + 2], out[4 * i + 3]));
    }
  }
  me.cluster_barrier();

  // The first CTA's settings are those of all: what CTAs meet at barriers by has to be the same in each, whatever another stream writes.
  const uint4 settings = sh.first[0][3];
  temperature = __uint_as_float(settings.x);
  top_k = static_cast<int>(settings.y);
  top_p = __uint_as_float(settings.z);
  floor = __uint_as_float(settings.w);
  const bool sampled = temperature > 0.0f;
  const double min_p = floor > 0.0f ? fmin(static_cast<double>(floor), 1.0) : 0.0;
  const bool by_count = sampled && top_k > 0 && top_k < p.vocabulary, by_sum = sampled && top_p < 1.0f, by_floor = sampled && min_p > 0.0;

  uint32_t largest = kNothing, lower = kNothing + 1;  // at least top_k values are not below `lower`
  {
    const uint32_t* entry = reinterpret_cast<const uint32_t*>(&sh.first[lane < ctas ? lane : 0][0]);
    largest = __reduce_max_sync(0xffffffffu, entry[0]);
    if (by_count) {
      int level = -1;
      for (int l = 0; l < kLevels && (1 << l) <= kThreads; ++l)
        if ((ctas * kThreads >> l) >= top_k) level = l;
      if (level >= 0) lower = max(lower, __reduce_min_sync(0xffffffffu, entry[2 + level]));
    }
  }
  const auto answer = [&](int token, float probability) {
    p.tokens[row] = token;
    if (p.probabilities) p.probabilities[row] = probability;
  };
  if (largest <= kNothing) {  // nothing to take
    if (rank == 0 && thread == 0) answer(-1, 0.0f);
    return;
  }
  const float most = value_of(largest);
  if (!sampled) {  // the best: the lowest index that has it, of the first CTA that has one
    uint32_t index = 0xffffffffu;
    me.each_value([&](float x, int i) {
      if (x == most) index = min(index, static_cast<uint32_t>(i));
    });
    index = __reduce_min_sync(0xffffffffu, index);
    if (lane == 0) sh.warp_index[warp] = index;
    __syncthreads();
    if (thread < kWarps) index = sh.warp_index[thread];
    if (warp == 0) index = __reduce_min_sync(0xffffffffu, index);
    bool before = false;
    for (int r = 0; r < rank; ++r) before |= sh.first[r][0].x == largest;
    if (!before && thread == 0 && index != 0xffffffffu) answer(static_cast<int>(index), 1.0f);
    return;
  }
  const double degrees = static_cast<double>(temperature);
  me.cap = p.softcap;
  me.scale = 1.4426950408889634074 * kExp2Entries / degrees;
  me.top = p.softcap > 0.0f ? softened(most, me.cap) : static_cast<double>(most);
  me.scale32 = static_cast<float>(me.scale);
  me.top32 = most;
  me.cut = fmaxf(__double2float_rd(static_cast<double>(most) - kShareOctaves * 0.69314718055994530942 * degrees), -3.402823466e38f);
  // (sizes at which 32 bits hold the whole part of every share that there is)
  const bool ordinary = fabsf(most) < 1e30f && me.cut > -1e30f && temperature > 1e-30f && temperature < 1e30f;
  me.form = p.softcap > 0.0f ? kCapped : ordinary ? kPlain : kAny;

  // The list has all that may be kept, inside the border: sorted by rank it is cut, sorted by index it is walked over.
  const auto finish = [&](int count, bool summed, double whole_sum) {
    sort_list<kThreads>(sh.list, count);
    const int ranks = by_count ? min(count, top_k) : count;
    double w[4], upto[4], in_front;
    unsigned long long entries[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = 4 * thread + j;
      entries[j] = i < ranks ? sh.list[i] : ~0ull;
      w[j] = i < ranks ? me.share(R::ranked_value(entries[j])) : 0.0;
    }
    const double sum = me.list_upto(w, upto, in_front);
    const double target = static_cast<double>(top_p) * (summed ? whole_sum : sum);
    int kept = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = 4 * thread + j;
      const bool stays = i < ranks && (i == 0 || !by_sum || (j == 0 ? in_front : upto[j - 1]) < target) && !(by_floor && w[j] < min_p);
      kept += __syncthreads_count(stays);
      // by index now, with the order behind it
      sh.list[i] = stays ? entries[j] << 32 | entries[j] >> 32 : ~0ull;
    }
    __syncthreads();
    sort_list<kThreads>(sh.list, count);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = 4 * thread + j;
      entries[j] = i < kept ? sh.list[i] : ~0ull;
      w[j] = i < kept ? me.share(value_of(~static_cast<uint32_t>(entries[j]))) : 0.0;
    }
    if (thread == 0) sh.found = kept - 1;
    const double all = me.list_upto(w, upto, in_front);
#pragma unroll
    for (int j = 3; j >= 0; --j)
      if (4 * thread + j < kept && upto[j] > u * all) atomicMin(&sh.found, 4 * thread + j);
    __syncthreads();
    const int found = sh.found;
    if (found >> 2 == thread) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if ((found & 3) == j) answer(static_cast<int>(entries[j] >> 32), static_cast<float>(w[j] / all));
    }
  };
  // Where the list may have all that may be kept: from which order on.  Up to kCap / 8 groups give some kCap / 8 * ln(kCap / 8) candidates,
  // which a list holds; of more groups it would not.
  uint32_t from = 0;
  if (p.vocabulary <= kCap && (by_count || by_sum)) {
    from = kNothing + 1;
  } else if (by_count) {
    if (top_k <= kCap / 8) from = lower;
  } else if (by_floor && !by_sum) {
    // Nothing further below the largest than this has a share of min_p; capped values: above where the cap's inverse is.
    double y = me.top + degrees * log(min_p);
    if (me.form == kCapped) {
      const double z = y / me.cap - 1e-12;
      y = z > -1.0 ? me.cap * 0.5 * log((1.0 + z) / fmax(1.0 - z, 1e-30)) : -INFINITY;
    }
    y -= 1e-6 * (fabs(y) + fabs(static_cast<double>(most)));
    const float bound = y > static_cast<double>(most) ? most : __double2float_rd(y);
    from = bound == bound ? max(order_of(bound), kNothing + 1) : kNothing + 1;
  }
  int listed = -1;  // entries of a list that has all
  bool summed = false;
  double whole_sum = 0.0;
  if (from != 0) {
    const int count = me.gather(from, largest, [](float) {});
    if (count <= kCap) listed = count;
  }
  double above_mine = 0.0;  // this lane's part of the sum above the border's window
  uint32_t window_high = 0;
  bool begun = false;
#pragma unroll 1
  for (int rule = 0; rule < 2 && listed < 0; ++rule) {  // top_k, then top_p
    if (rule == 0 ? !by_count : !by_sum) continue;
    const bool shares = rule == 1;
    double sum = 0.0, target = top_k;
    bool done = false;
    if (me.form != kAny) {
      me.count_bins(shares, sum);
      if (shares) target = static_cast<double>(top_p) * sum;
      const BinWindow window = me.window_of_bins(shares, target);
      if (window.count > 0) {
        const uint32_t low = max(me.order_with(window.last, largest), me.border_key);
        const uint32_t high = window.first > 0 ? order_below(me.order_with(window.first - 1, largest)) : largest;
        double v[1] = {0.0};
        const int count = me.gather(low, high, [&](float x) { v[0] += shares ? me.share(x) : 1.0; });
        if (window.whole && count <= kCap) {
          listed = count;
          summed = shares;
          whole_sum = sum;
          break;
        }
        above_mine = v[0];
        me.cluster_sums(v);
        done = count > 0 && count <= kCap && me.border_from_list(count, shares, v[0], target, false);
        if (done && shares) {
          begun = !by_floor;
          window_high = high;
        }
      }
    } else if (shares) {
      double v[1] = {0.0};
      me.each_value([&](float x, int i) { v[0] += me.inside(x, i) ? me.share(x) : 0.0; });
      me.cluster_sums(v);
      target = static_cast<double>(top_p) * v[0];
    }
    if (!done) me.find_border(shares, target, me.border_key, largest);
  }
  if (listed >= 0) {
    if (rank == 0) finish(listed, summed, whole_sum);
    return;
  }
  // The kept shares in the order of the vocabulary.
  const auto kept_share = [&](float x, int i) {
    if (!me.inside(x, i)) return 0.0;
    const double w = me.share(x);
    return by_floor && w < min_p ? 0.0 : w;
  };
  const auto target_of = [&](double all) { return u * all; };
  const auto found = [&](float, int i, double w, double all) { answer(i, static_cast<float>(w / all)); };
  if (begun) {  // what is above the window has been summed
    const float upto = value_of(window_high), from = value_of(me.border_key);
    me.locate(above_mine, [&](float x, int i) { return x >= from && x <= upto && me.inside(x, i) ? me.share(x) : 0.0; }, kept_share, target_of, found);
  } else if (me.form == kPlain && !me.bounded && !by_floor) {
    const float from = me.cut;
    me.locate(
        0.0,
        [&](float x, int) {
          const double w = me.plain_share(x, me.plain_whole(x));
          return x >= from ? w : 0.0;
        },
        kept_share, target_of, found);
  } else {
    me.locate(0.0, kept_share, kept_share, target_of, found);
  }
}

template <typename T, int kThreads>
cudaError_t launch_threads(const SampleCall& call, int ctas, cudaStream_t stream) {
  constexpr int kE = Vector<T>::kValues;
  SampleParams p{call, ctas, 0};
  p.cta_vectors = (call.vocabulary + 2 * (kE - 1) + kE * ctas - 1) / (kE * ctas);  // (with the lead at its largest)
  return launch_chained_clusters(sample_kernel<T, kThreads>, ctas, dim3(static_cast<unsigned>(call.rows) * ctas), dim3(kThreads),
                                 16 * static_cast<size_t>(p.cta_vectors), stream, p);
}

template <typename T>
cudaError_t launch_type(const SampleCall& call, int sm_count, cudaStream_t stream) {
  const long long bytes = static_cast<long long>(call.vocabulary) * sizeof(T);
  if (bytes <= 4096) return launch_threads<T, 128>(call, 1, stream);
  // As many CTAs as a row needs for 64 KB each, two of which an SM holds with their lists; more where rows are few, down to 8 KB each.
  int ctas = 1;
  while (ctas < kMostCtas && (bytes > 65536ll * ctas || (bytes > 16384ll * ctas && 2ll * ctas * call.rows <= 2 * sm_count))) ctas *= 2;
  return launch_threads<T, 512>(call, ctas, stream);
}

}  // namespace

cudaError_t launch_sample(const SampleCall& call, int sm_count, cudaStream_t stream) {
  return call.wide ? launch_type<float>(call, sm_count, stream) : launch_type<__nv_bfloat16>(call, sm_count, stream);
}

}  // namespace gv
