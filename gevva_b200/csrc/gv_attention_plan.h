// How attention work is counted and cut into pieces.  Plain integer arithmetic for host and device: the kernel walks it, and a
// host program plays it through (tests/attention_plan_probe.cpp).
//
// A sequence of `news` new tokens over `length` keys (the new ones included) has its token i at position length - news + i, which sees
// the keys up to that position, the last `window` of them only where a window is set.  Tokens are taken `step` at a time (a query
// tile) and keys 128 at a time (a key tile, counted from the sequence's first key).  An item is one query tile of one key head (and of
// one half of the value columns, for heads of 512); its work is its number of key tiles, at least one, so that rows that see nothing are
// written too.
#pragma once

#ifdef __CUDACC__
#define GV_HD __host__ __device__ __forceinline__
#else
#define GV_HD inline
#endif

namespace gv {

constexpr int kAttnKeys = 128;  // keys of a tile

struct AttnSequence {
  int news, past;    // past = length - news; below zero where there are fewer keys than new tokens
  int query_tiles;   // ceil(news / step)
};

GV_HD AttnSequence attn_sequence(int news, int length, int step) {
  AttnSequence s;
  s.news = news;
  s.past = length - news;
  s.query_tiles = (news + step - 1) / step;
  return s;
}

// One past the last key that any token of query tile q sees, and the first key that any of them does.
GV_HD int attn_key_end(const AttnSequence& s, int q, int step) {
  const int tokens = (q + 1) * step < s.news ? (q + 1) * step : s.news;
  return s.past + tokens > 0 ? s.past + tokens : 0;
}
GV_HD int attn_key_begin(const AttnSequence& s, int q, int step, int window) {
  const int first = s.past + q * step - window + 1;
  return window > 0 && first > 0 ? first : 0;
}
GV_HD int attn_first_tile(const AttnSequence& s, int q, int step, int window) { return attn_key_begin(s, q, step, window) / kAttnKeys; }
GV_HD int attn_tiles(const AttnSequence& s, int q, int step, int window) {
  const int tiles = (attn_key_end(s, q, step) + kAttnKeys - 1) / kAttnKeys - attn_first_tile(s, q, step, window);
  return tiles > 0 ? tiles : 1;
}

// Sum over i < n of floor((a * i + b) / m) for a, b >= 0 and m > 0, in as many rounds as Euclid's algorithm takes for (a, m).
GV_HD long long attn_floor_sum(long long n, long long m, long long a, long long b) {
  long long sum = 0;
  while (n > 0) {
    if (a >= m) {
      sum += n * (n - 1) / 2 * (a / m);
      a %= m;
    }
    if (b >= m) {
      sum += n * (b / m);
      b %= m;
    }
    const long long top = a * n + b;
    if (top < m) break;
    n = top / m;
    b = top % m;
    const long long t = m;
    m = a;
    a = t;
  }
  return sum;
}

// Key tiles of the first `count` query tiles of a sequence (for one head).
GV_HD long long attn_tiles_before(const AttnSequence& s, int count, int step, int window) {
  if (count <= 4) {
    long long sum = 0;
    for (int q = 0; q < count; ++q) sum += attn_tiles(s, q, step, window);
    return sum;
  }
  // query tiles in front of the first key see nothing and count one each
  int blind = s.past < 0 ? -s.past / step : 0;
  if (blind > s.query_tiles - 1) blind = s.query_tiles - 1;
  if (s.past + s.news <= 0) blind = s.query_tiles;
  if (count <= blind) return count;
  long long sum = blind;
  const int full = count < s.query_tiles - 1 ? count : s.query_tiles - 1;  // tiles of whole `step` tokens
  if (full > blind)
    sum += attn_floor_sum(full - blind, kAttnKeys, step,
                          static_cast<long long>(s.past) + static_cast<long long>(blind + 1) * step + kAttnKeys - 1);
  if (count == s.query_tiles) sum += (s.past + s.news + kAttnKeys - 1) / kAttnKeys;
  if (window > 0) {
    const int lead = window - 1 - s.past;
    int from = lead > 0 ? (lead + step - 1) / step : 0;
    if (from < blind) from = blind;
    if (count > from)
      sum -= attn_floor_sum(count - from, kAttnKeys, step,
                            static_cast<long long>(s.past) + static_cast<long long>(from) * step - window + 1);
  }
  return sum;
}

// The query tile that holds key tile `at` (0 <= at < attn_tiles_before(all)) of a head's work, counted from its first.
GV_HD int attn_find_query_tile(const AttnSequence& s, long long at, int step, int window) {
  int low = 0, high = s.query_tiles - 1;
  while (low < high) {
    const int mid = (low + high) / 2;
    if (attn_tiles_before(s, mid + 1, step, window) > at) high = mid;
    else low = mid + 1;
  }
  return low;
}

// Work, `heads` times the same, is dealt out to at most `parts` CTAs in runs of equal length: to as many for each head where that leaves
// no more than a sixteenth of them without, to fewer where a run would be shorter than `least` key tiles.
GV_HD int attn_parts(long long work, int parts, int heads, int least) {
  const int even = heads <= parts ? parts / heads * heads : parts;
  if (16 * even >= 15 * parts) parts = even;
  return work < static_cast<long long>(parts) * least ? static_cast<int>(work + least - 1) / least : parts;
}
// (Divisions in 32 bits where they do, up to 1023 parts of fewer than 2^22 key tiles: in 64 they are a hundred instructions.)
GV_HD long long attn_part_begin(long long work, int parts, int part) {
  if (work < (1ll << 22) && parts < 1024) return static_cast<unsigned>(work) * static_cast<unsigned>(part) / static_cast<unsigned>(parts);
  return work * part / parts;
}
GV_HD int attn_quotient(long long a, long long b) {
  if (a < (1ll << 32) && b < (1ll << 32)) return static_cast<int>(static_cast<unsigned>(a) / static_cast<unsigned>(b));
  return static_cast<int>(a / b);
}

// What a run has of one item: key tiles [skip, skip + take) of the `tiles` that query tile `tile` has.
struct AttnShare {
  int head, sequence, tile;
  int skip, take, tiles;
  int slot;    // of its sums among 2 * parts: 2 * part for a share that another run begins, the one behind for a share that this run's end
               // cuts off; -1: the whole item
  int behind;  // of a share that is cut off: in how many of the next runs the item goes on
};

// The shares of run `part`, key tiles [begin, end) of all work, in the order in which they are worked on: hand_out(share), false to end there.
// The run begins in `sequence`, `offset` key tiles behind that sequence's first in `head` (of `of_first`); load(sequence, &news,
// &length) tells a sequence's.  Behind the last of `sequences` comes the next head's first.
// Ends by itself, and names no slot or run that there is not, whatever load() tells: lengths that change while a call runs give wrong results
// and nothing worse.
template <class Load, class HandOut>
GV_HD bool attn_walk(long long work, int parts, int part, long long begin, long long end, int heads, int head, int sequence, long long offset,
                     long long of_first, int sequences, int step, int window, Load&& load, HandOut&& hand_out) {
  long long at = begin;
  bool ok = true;
  while (ok && at < end && head < heads) {
    int news, length;
    load(sequence, &news, &length);
    if (news > 0) {
      const AttnSequence q = attn_sequence(news, length, step);
      // A run inside one sequence that begins and ends inside items takes the last one first: runs of about an item's length, as
      // when a chunk has about as many query tiles as there are CTAs, then read the same keys at about the same time instead of
      // each one others (512 tokens behind 31488, heads of 512, 128 MB of keys and values: 690 -> 533 us).
      int tile = 0, last = -1;
      long long stop = end;
#ifdef __CUDACC__
#pragma unroll 1  // (a short reply's time is that of code fetched for the first time: this only once)
#endif
      for (int i = q.query_tiles > 1 && offset > 0 && offset + (end - at) <= of_first ? 1 : 0; i >= 0; --i) {
        const long long target = i > 0 ? offset + (end - at) - 1 : offset;
        const int found = attn_find_query_tile(q, target, step, window);
        const long long before = attn_tiles_before(q, found, step, window);
        if (i > 0) {
          last = found;
          stop = end - (target + 1 - before);
        } else {
          tile = found;
          offset -= before;
        }
      }
      if (last == tile) {
        last = -1;
        stop = end;
      }
      const int first = tile;
      const long long first_offset = offset, first_at = at;
      bool ahead = last >= 0;
      if (ahead) {
        tile = last;
        offset = 0;
        at = stop;
      }
      for (; ok && tile < q.query_tiles && (ahead || at < stop); ++tile) {
        const int tiles = attn_tiles(q, tile, step, window);
        const long long left = (ahead ? end : stop) - at;
        if (offset < 0 || offset >= tiles || left < 1) return ok;  // (the work is not what it was)
        AttnShare share;
        share.head = head;
        share.sequence = sequence;
        share.tile = tile;
        share.tiles = tiles;
        share.skip = static_cast<int>(offset);
        share.take = tiles - share.skip < left ? tiles - share.skip : static_cast<int>(left);
        share.slot = share.take == tiles ? -1 : 2 * part + (share.skip == 0 ? 1 : 0);
        share.behind = 0;
        if (share.skip == 0 && share.take < tiles) {
          int upto = part;
          while (upto + 1 < parts && attn_part_begin(work, parts, upto + 1) < at + tiles) ++upto;
          share.behind = upto - part;
        }
        at += share.take;
        offset = 0;
        ok = hand_out(share);
        if (ahead) {
          ahead = false;
          tile = first - 1;
          offset = first_offset;
          at = first_at;
        }
      }
      if (last >= 0) at = end;
    }
    offset = 0;
    if (++sequence >= sequences) {
      sequence = 0;
      ++head;
    }
  }
  return ok;
}

}  // namespace gv
