// The streaming attention kernel's cut of a sequence into parts, replayed on the
// host: the parts cover the tokens once, in order, and as many of them hold any as
// the join goes by, up to the longest table that is accepted.
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <random>

#include "kv_attend_stream.h"

using namespace pf;

#define CHECK(x) \
  do { \
    if (!(x)) { \
      std::printf("failed: %s, line %d, case %d: begin %d end %d parts %u of %d\n", #x, __LINE__, round, begin, end, p.parts, \
                  p.part_tokens); \
      return 1; \
    } \
  } while (0)

int main(int argc, char** argv) {
  const int rounds = argc > 1 ? std::atoi(argv[1]) : 2000;
  std::mt19937_64 rng(11);
  auto pick = [&](int64_t lo, int64_t hi) { return std::uniform_int_distribution<int64_t>(lo, hi)(rng); };
  long far = 0;
  for (int round = 0; round < rounds; ++round) {
    // The bound that the plan was made for, and parts as stream_plan makes them: multiples of the shortest.
    const int64_t top = int64_t(kKvMaxTokens);
    const int64_t longest = pick(0, 2) ? pick(top - 5000000, top) : pick(1, top);
    const int64_t units = (longest + kStreamMinPart - 1) / kStreamMinPart;
    const int64_t least = (units + kStreamMaxParts - 1) / kStreamMaxParts;
    const int64_t per = pick(0, 1) ? pick(least, std::min<int64_t>(units, 40 * least)) : pick(least, units);
    KvStreamPlan p{};
    p.part_tokens = int32_t(std::min<int64_t>(per * kStreamMinPart, 1 << 30));
    p.parts = uint32_t((longest + p.part_tokens - 1) / p.part_tokens);
    // A sequence: as long as the bound, shorter, behind a window's begin, or longer than a bound that was too low.
    const int32_t end = int32_t(pick(0, 1) ? longest : pick(0, 1) ? pick(0, longest) : pick(0, top));
    const int32_t begin = pick(0, 1) ? 0 : int32_t(pick(0, end));
    const int32_t used = stream_parts(p, end - begin);
    CHECK(used >= 1 && used <= int32_t(p.parts));
    int32_t at = begin;
    for (uint32_t part = 0; part < p.parts; ++part) {
      const KvPart s = stream_part(p, begin, end, part);
      CHECK(s.lo == at && s.hi >= s.lo && s.hi <= end);
      CHECK((s.hi > s.lo) == (int32_t(part) < used) || begin == end);
      at = s.hi;
    }
    CHECK(at == end);
    far += int64_t(begin) + int64_t(p.parts) * stream_part_tokens(p, end - begin) > INT32_MAX;
  }
  if (far < rounds / 20) {  // cases whose last part, were it whole, would pass 2^31
    std::printf("only %ld cases near the end\n", far);
    return 1;
  }
  std::printf("ok rounds=%d far=%ld\n", rounds, far);
  return 0;
}
