// Plays the distribution of attention work (gv_attention_plan.h) through on the host: reads cases "window step heads parts least sequences (news length)..."
// and walks every CTA's run as the kernel does; prints "ok" where the runs cover each item's key tiles once, in order, and the
// joins name the CTAs that hold an item's parts.
#include <cstdio>
#include <vector>

#include "../gevva_b200/csrc/gv_attention_plan.h"

using namespace gv;

static bool fail(const char* what, long long a, long long b) {
  std::printf("%s: %lld %lld\n", what, a, b);
  return false;
}

static bool play(int window, int step, int heads, int parts_most, int least, const std::vector<int>& news, const std::vector<int>& lengths) {
  std::vector<AttnSequence> all;
  long long work = 0;
  std::vector<long long> item_begin;  // of every item, in the order of the work
  std::vector<int> item_tiles;
  for (size_t s = 0; s < news.size(); ++s) {
    all.push_back(attn_sequence(news[s], lengths[s], step));
    const AttnSequence& q = all.back();
    // from the definition: tiles that hold a key which a token of the query tile sees
    long long before = 0;
    for (int t = 0; t < q.query_tiles; ++t) {
      int first = -1, last = -1;
      for (int i = t * step; i < (t + 1) * step && i < news[s]; ++i) {
        const int position = lengths[s] - news[s] + i;
        if (position < 0) continue;
        const int low = window > 0 && position - window + 1 > 0 ? position - window + 1 : 0;
        if (first < 0 || low / kAttnKeys < first) first = low / kAttnKeys;
        if (position / kAttnKeys > last) last = position / kAttnKeys;
      }
      const int want = last < 0 ? 1 : last - first + 1;
      if (attn_tiles(q, t, step, window) != want) return fail("tiles", attn_tiles(q, t, step, window), want);
      if (last >= 0 && attn_first_tile(q, t, step, window) != first) return fail("first", attn_first_tile(q, t, step, window), first);
      if (attn_tiles_before(q, t, step, window) != before) return fail("before", attn_tiles_before(q, t, step, window), before);
      for (int x : {0, want - 1})
        if (attn_find_query_tile(q, before + x, step, window) != t) return fail("find", before + x, t);
      before += want;
    }
    if (attn_tiles_before(q, q.query_tiles, step, window) != before) return fail("all", attn_tiles_before(q, q.query_tiles, step, window), before);
  }
  for (int h = 0; h < heads; ++h)
    for (const AttnSequence& q : all)
      for (int t = 0; t < q.query_tiles; ++t) {
        item_begin.push_back(work);
        item_tiles.push_back(attn_tiles(q, t, step, window));
        work += item_tiles.back();
      }
  const int parts = attn_parts(work, parts_most, heads, least);
  if (parts > parts_most || (work > 0 && parts < 1) || (work >= 2ll * parts_most * least && 16 * parts < 15 * parts_most)) return fail("parts", parts, work);
  if (work > 0 && attn_quotient(work - 1, work / heads) != heads - 1) return fail("quotient", work, heads);
  long long at = 0;
  for (int c = 0; c < parts; ++c) {
    const long long begin = attn_part_begin(work, parts, c), end = attn_part_begin(work, parts, c + 1);
    if (begin != at || end <= begin) return fail("run", begin, end);
    if (end - begin > (work + parts - 1) / parts) return fail("long run", end - begin, work);
    at = end;
  }
  if (at != work) return fail("end", at, work);
  // joins: an item cut by the end of the run that it begins in
  for (size_t i = 0; i < item_begin.size(); ++i) {
    int first = 0, last = 0;
    while (attn_part_begin(work, parts, first + 1) <= item_begin[i]) ++first;
    last = first;
    while (attn_part_begin(work, parts, last + 1) < item_begin[i] + item_tiles[i]) ++last;
    if (last >= parts) return fail("join", last, parts);
  }
  return true;
}

int main() {
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
