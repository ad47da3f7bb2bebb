// Without an argument: plays every CTA's run of attention work through on the host, by the code that the kernel walks it with (attn_walk, gv_attention_plan.h):
// reads cases "window step heads parts least sequences (news length)..." and prints "ok <cases>" where
//   - the shares hold every item's key tiles once (an item: head, sequence, query tile), none of them empty,
//   - sums go to slots that no other share has,
//   - an item that is whole goes to none; one that is cut is told of by the run it begins in and by no other, once a run, and the slots
//     that attention_join_kernel then reads (the second of that run, the first of the next `behind`) hold its key tiles in their order.
// With one: lengths that change while the work is walked.
#include <cstdio>
#include <map>
#include <tuple>
#include <vector>

#include "../gevva_b200/csrc/gv_attention_plan.h"

using namespace gv;

static bool fail(const char* what, long long a, long long b) {
  std::printf("%s: %lld %lld\n", what, a, b);
  return false;
}

using Item = std::tuple<int, int, int>;  // head, sequence, query tile
struct Sums {
  Item item;
  int skip, take;
};

// Lengths that change with every look at them: the walk ends, and its shares name key tiles, slots and runs that there are.
static bool change(int seed) {
  unsigned long long state = 0x9e3779b97f4a7c15ull * (seed + 1);
  const auto draw = [&](int low, int high) {
    state = state * 6364136223846793005ull + 1442695040888963407ull;
    return low + static_cast<int>((state >> 33) % (high - low + 1));
  };
  const int step = draw(1, 256), window = draw(0, 2) ? 0 : draw(1, 2000), heads = draw(1, 6), parts = draw(1, 160), sequences = draw(1, 90);
  const long long work = draw(1, 100000), part = draw(0, parts - 1);
  const long long begin = attn_part_begin(work, parts, part), end = attn_part_begin(work, parts, part + 1);
  AttnSequence now{};
  bool good = true;
  long long loads = 0;
  const int kind = draw(0, 3);  // all empty; all alike; any
  const auto load = [&](int, int* news, int* length) {
    *news = kind == 0 ? 0 : kind == 1 ? 1 : draw(0, 600);
    *length = kind == 1 ? 1 : draw(0, 40000);
    now = attn_sequence(*news, *length, step);
    if (++loads > 2ll * heads * sequences + 1000) good = fail("loads", loads, sequences);
  };
  const auto hand_out = [&](const AttnShare& share) {
    const int tiles = attn_tiles(now, share.tile, step, window);
    if (share.tile < 0 || share.tile >= now.query_tiles || share.tiles != tiles || share.skip < 0 || share.take < 1 || share.skip + share.take > tiles)
      return good = fail("share", share.skip, share.take);
    if (share.slot < -1 || share.slot >= 2 * parts || share.behind < 0 || part + share.behind >= parts) return good = fail("slot", share.slot, share.behind);
    return good;
  };
  attn_walk(work, parts, static_cast<int>(part), begin, end, heads, draw(0, heads), draw(0, sequences + 31), draw(-5, 3) * 1000000007ll, draw(0, 5000),
            sequences, step, window, load, hand_out);
  return good;
}

static bool play(int window, int step, int heads, int parts_most, int least, const std::vector<int>& news, const std::vector<int>& lengths) {
  const int sequences = static_cast<int>(news.size());
  std::vector<long long> of_sequence(sequences);
  long long of_head = 0;
  for (int s = 0; s < sequences; ++s) {
    const AttnSequence q = attn_sequence(news[s], lengths[s], step);
    for (int t = 0; t < q.query_tiles; ++t) of_sequence[s] += attn_tiles(q, t, step, window);
    of_head += of_sequence[s];
  }
  const long long work = of_head * heads;
  const int parts = attn_parts(work, parts_most, heads, least);
  std::map<Item, std::vector<std::pair<int, int>>> seen;  // [skip, skip + take) of an item
  std::map<Item, int> tiles_of;
  std::map<int, Sums> slots;
  std::map<Item, std::pair<int, int>> told;  // run, behind
  for (int part = 0; part < parts; ++part) {
    const long long begin = attn_part_begin(work, parts, part), end = attn_part_begin(work, parts, part + 1);
    // where the run begins, by counting
    const int head = static_cast<int>(begin / of_head);
    long long offset = begin - head * of_head;
    int s = 0;
    while (offset >= of_sequence[s]) offset -= of_sequence[s++];
    long long taken = 0;
    int records = 0;
    bool good = true;
    const auto load = [&](int sequence, int* n, int* length) {
      if (sequence < 0 || sequence >= sequences) good = fail("sequence", sequence, sequences);
      *n = news[sequence];
      *length = lengths[sequence];
    };
    const auto hand_out = [&](const AttnShare& share) {
      const Item item{share.head, share.sequence, share.tile};
      const AttnSequence q = attn_sequence(news[share.sequence], lengths[share.sequence], step);
      if (share.head < 0 || share.head >= heads || share.tile < 0 || share.tile >= q.query_tiles) return good = fail("item", share.head, share.tile);
      const int tiles = attn_tiles(q, share.tile, step, window);
      if (share.tiles != tiles || share.take < 1 || share.skip < 0 || share.skip + share.take > tiles) return good = fail("share", share.skip, share.take);
      tiles_of[item] = tiles;
      seen[item].push_back({share.skip, share.take});
      taken += share.take;
      if ((share.slot < 0) != (share.take == tiles)) return good = fail("slot of a whole item", share.slot, share.take);
      if (share.slot >= 0) {
        if (share.slot >= 2 * parts || !slots.insert({share.slot, Sums{item, share.skip, share.take}}).second) return good = fail("slot", share.slot, part);
      }
      if (share.behind != 0) {
        if (++records > 1 || !told.insert({item, {part, share.behind}}).second) return good = fail("told twice", part, share.behind);
      }
      return true;
    };
    if (!attn_walk(work, parts, part, begin, end, heads, head, s, offset, of_sequence[s], sequences, step, window, load, hand_out) || !good) return false;
    if (taken != end - begin) return fail("run", taken, end - begin);
  }
  // every item's key tiles once
  size_t items = 0;
  for (int h = 0; h < heads; ++h)
    for (int s = 0; s < sequences; ++s) items += (news[s] + step - 1) / step;
  if (seen.size() != items) return fail("items", static_cast<long long>(seen.size()), static_cast<long long>(items));
  for (auto& [item, shares] : seen) {
    std::vector<char> tile(tiles_of[item], 0);
    for (auto [skip, take] : shares)
      for (int x = skip; x < skip + take; ++x)
        if (tile[x]++) return fail("key tile twice", std::get<2>(item), x);
    for (size_t x = 0; x < tile.size(); ++x)
      if (!tile[x]) return fail("key tile of nobody", std::get<2>(item), static_cast<long long>(x));
    if ((shares.size() > 1) != (told.count(item) != 0)) return fail("cut and not told of", std::get<2>(item), static_cast<long long>(shares.size()));
  }
  // what the join reads
  size_t joined = 0;
  for (auto& [item, where] : told) {
    const auto [run, behind] = where;
    int next = 0;
    for (int i = 0; i <= behind; ++i) {
      const auto found = slots.find(2 * (run + i) + (i == 0 ? 1 : 0));
      if (found == slots.end() || found->second.item != item || found->second.skip != next) return fail("join", run, i);
      next += found->second.take;
      ++joined;
    }
    if (next != tiles_of[item]) return fail("join ends early", next, tiles_of[item]);
  }
  if (joined != slots.size()) return fail("slots that nobody joins", static_cast<long long>(joined), static_cast<long long>(slots.size()));
  return true;
}

int main(int argc, char**) {
  if (argc > 1) {  // any argument: lengths that change
    for (int seed = 0; seed < 200000; ++seed)
      if (!change(seed)) return 1;
    std::printf("ok\n");
    return 0;
  }
  int window, step, heads, parts, least, sequences, cases = 0;
  while (std::scanf("%d %d %d %d %d %d", &window, &step, &heads, &parts, &least, &sequences) == 6) {
    std::vector<int> news(sequences), lengths(sequences);
    for (int s = 0; s < sequences; ++s)
      if (std::scanf("%d %d", &news[s], &lengths[s]) != 2) return 2;
    if (!play(window, step, heads, parts, least, news, lengths)) {
      std::printf("case %d\n", cases);
      return 1;
    }
    ++cases;
  }
  std::printf("ok %d\n", cases);
  return 0;
}
