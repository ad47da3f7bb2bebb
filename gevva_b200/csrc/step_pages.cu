// Page tables and slots of a step, from the lengths of its requests (declared in include/gevva_moe.h).
//
// Two running sums over the requests, of their tokens and of their pages, say where each one's rows and pages begin; everything else follows
// for each row and each page by itself.  A cluster does it in one launch: every CTA works out both sums for itself (up to 16384
// requests in shared memory), takes its part of the rows and pages, and writes what a call may have been given as inputs too (lengths, the number
// of pages handed out) behind a barrier of the cluster, when all have read them.  Latency bounds plans and small trims: launch, two dependent
// reads, the sums, the search of a row's request, two dependent reads, a write.  Trims of large batches are bound by the cluster's eight SMs, through
// which all their table entries go.  In a graph: 64 requests 3.4 us, four prompts of 4608 tokens 5.8, 1000
// requests with drafts 7.4; trimmed, 64 requests 4.1, 1000 of which a third end 9.3 (15.8 with a search for each page instead of one for a
// warp's pages).
#include "gv_common.cuh"
#include "gv_step.h"

namespace gv {
namespace {

constexpr int kPagesThreads = 1024;
constexpr int kPagesCtas = 8;

struct PagesParams {
  PagesCall call;
  int page_shift;
};

__device__ __forceinline__ int pages_for(int tokens, int page_shift) {
  return static_cast<int>((static_cast<long long>(tokens) + (1 << page_shift) - 1) >> page_shift);
}

// The last entry of begins[0 .. count] (ascending, begins[0] = 0, begins[count] > at) that is not above `at`.
__device__ __forceinline__ int find_request(const int* begins, int count, int at) {
  int low = 0, high = count;
  while (high - low > 1) {
    const int mid = (low + high) >> 1;
    if (begins[mid] <= at) low = mid;
    else high = mid;
  }
  return low;
}

template <bool kTrim>
__global__ void __launch_bounds__(kPagesThreads, 1) step_pages_kernel(const PagesParams params) {
  extern __shared__ int shared[];
  __shared__ long long warp_rows[32], warp_pages[32];
  __shared__ int shared_taken;
  const PagesCall& p = params.call;
  const int n = p.sequences, shift = params.page_shift;
  int* const row_begins = shared;                        // [n + 1] (trim: not used)
  int* const page_begins = shared + (kTrim ? 0 : n + 1);  // [n + 1]
  int* const tokens = page_begins + n + 1;               // [n] that it has before (plan) or after (trim); the pages behind theirs move
  const int threads = blockDim.x, thread = threadIdx.x, lane = thread & 31, warp = thread >> 5;
  const int rank = static_cast<int>(cluster_cta_rank()), ctas = gridDim.x;  // (one cluster)
  grid_launch_dependents();
  grid_dependency_wait();

  if (thread == 0) shared_taken = *p.taken;  // (one read for the CTA: what another stream writes meanwhile makes wrong results, and nothing worse)
  // A thread takes `each` requests that follow one another.
  const int each = (n + threads - 1) / threads, first = min(n, thread * each), last = min(n, first + each);
  long long rows = 0, pages = 0;
  bool lost = false;  // a request whose numbers cannot be
  const long long room = static_cast<long long>(p.table_width) << shift;
  for (int s = first; s < last; ++s) {
    const int length = p.lengths[s], count = p.counts[s];
    const long long after = kTrim ? min(length, max(count, 0)) : static_cast<long long>(length) + count;
    if (length < 0 || length > room || after < 0 || after > room || (!kTrim && count < 0)) {
      lost = true;
      break;
    }
    const int now = pages_for(length, shift), then = pages_for(static_cast<int>(after), shift);
    tokens[s] = kTrim ? static_cast<int>(after) : length;
    page_begins[s] = kTrim ? now - then : then - now;
    pages += page_begins[s];
    if (!kTrim) {
      row_begins[s] = count;
      rows += count;
    }
  }
  // both sums over the threads in front
  long long rows_upto = rows, pages_upto = pages;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const long long r = __shfl_up_sync(0xffffffffu, rows_upto, d), q = __shfl_up_sync(0xffffffffu, pages_upto, d);
    if (lane >= d) {
      rows_upto += r;
      pages_upto += q;
    }
  }
  if (lane == 31) {
    warp_rows[warp] = rows_upto;
    warp_pages[warp] = pages_upto;
  }
  const bool any_lost = __syncthreads_or(lost);
  const int taken = shared_taken;
  int bad = any_lost ? static_cast<int>(kBadPage) : taken < 0 || taken > p.pool_pages ? static_cast<int>(kNoPages) : 0;
  long long all_rows = 0, all_pages = 0;
  for (int w = 0; w < threads / 32; ++w) {
    if (w == warp) {
      rows_upto += all_rows;
      pages_upto += all_pages;
    }
    all_rows += warp_rows[w];
    all_pages += warp_pages[w];
  }
  if (!bad && !kTrim && all_rows > p.tokens) bad = kTooLarge;
  if (!bad && (kTrim ? all_pages > taken : all_pages > p.pool_pages - taken)) bad = kNoPages;
  if (bad) {  // (all CTAs find the same) nothing is taken or given back, and no row is a token
    if (rank == 0 && thread == 0 && p.status) atomicExch(p.status, bad);
    all_rows = all_pages = 0;
  }
  if (!bad) {
    long long row = rows_upto - rows, page = pages_upto - pages;
    for (int s = first; s < last; ++s) {
      const int moved = page_begins[s];
      page_begins[s] = static_cast<int>(page);
      page += moved;
      if (!kTrim) {
        const int count = row_begins[s];
        row_begins[s] = static_cast<int>(row);
        row += count;
      }
    }
    if (thread == 0) {
      page_begins[n] = static_cast<int>(all_pages);
      if (!kTrim) row_begins[n] = static_cast<int>(all_rows);
    }
  }
  __syncthreads();

  const int whole = threads * ctas, me = rank * threads + thread;
  const int base = kTrim ? taken - static_cast<int>(all_pages) : taken;  // of the pages that move, in the pool's list
  if (!bad && all_pages <= whole) {  // a thread for each page
    if (me < all_pages) {
      const int s = find_request(page_begins, n, me);
      int* const entry = p.table + static_cast<size_t>(s) * p.table_stride + pages_for(tokens[s], shift) + (me - page_begins[s]);
      if (kTrim) p.pool[base + me] = *entry;
      else *entry = p.pool[base + me];
    }
  } else if (!bad) {
    // Pages by themselves, whoever's they are: one long request among many takes no longer than its share.  A warp takes pages that follow
    // one another, looks up whose the first is and goes on from there; four of a lane are on their way together.
    const long long each_warp = (all_pages + (whole >> 5) - 1) / (whole >> 5);
    const int from = static_cast<int>(min(all_pages, (me >> 5) * each_warp)), upto = static_cast<int>(min(all_pages, from + each_warp));
    int s = from < upto ? find_request(page_begins, n, from) : 0;
    for (long long first = from; first < upto; first += 4 * 32) {
      const int g = static_cast<int>(min(first + lane, static_cast<long long>(upto)));
      int* out[4];
      int page[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (32 * k >= upto - g) break;
        const int at = g + 32 * k;
        while (page_begins[s + 1] <= at) ++s;  // (page_begins[n] is behind all)
        int* const entry = p.table + static_cast<size_t>(s) * p.table_stride + pages_for(tokens[s], shift) + (at - page_begins[s]);
        out[k] = kTrim ? p.pool + base + at : entry;
        page[k] = kTrim ? *entry : p.pool[base + at];
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (32 * k < upto - g) *out[k] = page[k];
    }
  }
  if constexpr (!kTrim) {
    for (int t = me; t < p.tokens; t += whole) {
      int slot = -1, position = 0;
      if (t < all_rows) {
        const int s = find_request(row_begins, n, t);
        position = tokens[s] + t - row_begins[s];
        const int index = position >> shift, held = pages_for(tokens[s], shift);
        // (a new page comes straight from the list: its entry of the table may be on its way)
        const int page = index < held ? p.table[static_cast<size_t>(s) * p.table_stride + index] : p.pool[base + page_begins[s] + index - held];
        const long long at = (static_cast<long long>(page) << shift) + (position & ((1 << shift) - 1));
        if (at < 0 || at > 0x7fffffffll) {
          if (p.status) atomicExch(p.status, static_cast<int>(kBadPage));
        } else {
          slot = static_cast<int>(at);
        }
        if (p.shift) position = static_cast<int>(static_cast<unsigned>(position) + static_cast<unsigned>(p.shift[s]));
      }
      p.slots[t] = slot;
      p.positions[t] = position;
    }
  }
  cluster_sync_all();  // lengths and the number of pages have been read
  if (rank == 0) {
    for (int s = thread; s < n; s += threads) {
      if (!kTrim) p.offsets_out[s] = bad ? 0 : row_begins[s];
      p.lengths_out[s] = bad ? p.lengths[s] : kTrim ? tokens[s] : tokens[s] + row_begins[s + 1] - row_begins[s];
    }
    if (thread == 0) {
      if (!kTrim) p.offsets_out[n] = static_cast<int>(all_rows);
      *p.taken_out = kTrim ? taken - static_cast<int>(all_pages) : taken + static_cast<int>(all_pages);
    }
  }
}

}  // namespace

cudaError_t launch_step_pages(const PagesCall& call, cudaStream_t stream) {
  PagesParams p{call, 0};
  while ((1 << p.page_shift) < call.page_size) ++p.page_shift;
  const size_t bytes = sizeof(int) * ((call.trim ? 2 : 3) * static_cast<size_t>(call.sequences) + 2);
  // A thread for a request and for a row, up to a CTA's; then as many CTAs as a cluster may portably have.
  const int items = call.trim ? 32 * call.sequences : (call.sequences > call.tokens ? call.sequences : call.tokens);
  const int threads = items >= kPagesThreads ? kPagesThreads : (items + 31) / 32 * 32;
  int ctas = 1;
  while (ctas < kPagesCtas && ctas * kPagesThreads < items) ctas *= 2;
  static std::atomic<unsigned long long> allowed[2];
  const auto kernel = call.trim ? step_pages_kernel<true> : step_pages_kernel<false>;
  const cudaError_t e = allow_clusters(kernel, sizeof(int) * (3 * kMaxPlanSequences + 2), &allowed[call.trim]);
  if (e != cudaSuccess) return e;
  return launch_chained_clusters(kernel, ctas, dim3(ctas), dim3(threads), bytes, stream, p);
}

}  // namespace gv
