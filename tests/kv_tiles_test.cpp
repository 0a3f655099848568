// The tile attention kernel's cut of its work, replayed on the host: items in a
// line, equal spans, each CTA walking its own. Every unit is computed once, every
// part of a split item has a slot of its own, and the join finds exactly them.
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <vector>

#include "kv_attend_tiles.h"

using namespace pf;

#define CHECK(x) \
  do { \
    if (!(x)) { \
      std::printf("failed: %s, line %d, case %d\n", #x, __LINE__, round); \
      return 1; \
    } \
  } while (0)

int main(int argc, char** argv) {
  const int rounds = argc > 1 ? std::atoi(argv[1]) : 2000;
  std::mt19937 rng(7);
  auto pick = [&](int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(rng); };
  long split_items = 0;
  for (int round = 0; round < rounds; ++round) {
    const uint32_t ctas = pick(0, 3) ? pick(1, 160) : 148;
    std::vector<int64_t> units(pick(1, pick(0, 1) ? 6 : 600)), at;
    int64_t total = 0;
    for (auto& u : units) {
      u = pick(0, 3) ? pick(1, 40) : tile_units(pick(0, 300), pick(0, 90000));
      at.push_back(total);
      total += u;
    }
    const int64_t span = span_units(total, ctas);
    CHECK(span * ctas >= total);
    // Each CTA's walk.
    std::vector<int64_t> done(units.size());
    std::map<int64_t, std::pair<size_t, int64_t>> slots;  // slot -> item, CTA
    std::map<size_t, std::vector<int64_t>> parts;         // item -> slots in the order of CTAs
    for (int64_t c = 0; c < ctas; ++c) {
      int64_t begin = c * span, left = span;
      if (begin >= total) break;
      size_t item = 0;
      while (item + 1 < units.size() && at[item + 1] <= begin) ++item;
      int64_t unit = begin - at[item];
      bool first = true;
      while (left > 0 && item < units.size()) {
        const int64_t end = std::min(units[item], unit + left);
        CHECK(done[item] == unit);  // the CTAs before did those in front
        done[item] = end;
        left -= end - unit;
        if (!(unit == 0 && end == units[item])) {
          const int64_t slot = 2 * c + (first ? 0 : 1);
          CHECK(slot == part_slot(at[item], c, span) && slot < 2 * int64_t(ctas));
          CHECK(slots.emplace(slot, std::make_pair(item, c)).second);
          parts[item].push_back(slot);
        }
        first = false;
        unit = 0;
        ++item;
      }
    }
    for (size_t i = 0; i < units.size(); ++i) CHECK(done[i] == units[i]);
    // The join: the block of the CTA in whose span an item begins that the next CTA's span goes on with.
    size_t joined = 0;
    for (int64_t c = 0; c < ctas; ++c) {
      const int64_t next = (c + 1) * span;
      if (next >= total) continue;
      size_t item = 0;
      while (item + 1 < units.size() && at[item + 1] <= next) ++item;
      if (next == at[item] || at[item] / span != c) continue;
      const KvSplit s = item_split(at[item], units[item], span);
      std::vector<int64_t> found;
      for (int64_t p = s.first; p <= s.last; ++p) found.push_back(part_slot(at[item], p, span));
      CHECK(found == parts[item]);
      ++joined;
    }
    CHECK(joined == parts.size());
    split_items += joined;
  }
  std::printf("ok rounds=%d split=%ld\n", rounds, split_items);
  return 0;
}
