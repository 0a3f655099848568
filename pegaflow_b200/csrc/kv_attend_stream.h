// How the streaming attention kernel's grid splits the work (host and device).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "kv_ops.h"

namespace pf {

constexpr uint32_t kStreamMaxRows = 16;  // queries times heads of a group that one CTA takes
constexpr uint32_t kStreamMaxParts = 32768;  // a grid's y axis ends at 65,535
constexpr uint32_t kStreamMaxCluster = 8;  // parts that a cluster's CTAs join among themselves
constexpr uint32_t kStreamMinPart = 128;  // tokens: a batch for each warp

struct KvStreamPlan {
  uint32_t row_tiles;   // 8-row tiles of a CTA: 1 or 2
  uint32_t parts;       // CTAs along the tokens
  int32_t part_tokens;  // tokens of a part, a multiple of kStreamMinPart
  int32_t page_shift;   // log2 of the block size, -1 if it is no power of two
  uint32_t clusters;    // a sequence's parts are a cluster, which joins them
};

// Tokens of each part when `range` tokens are to be covered, and how many parts
// that takes: the plan's, unless the bound that it was made for was too low.
__host__ __device__ inline int32_t stream_part_tokens(const KvStreamPlan& p, int32_t range) {
  const int32_t least = (range + int32_t(p.parts) - 1) / int32_t(p.parts);
  return p.part_tokens > least ? p.part_tokens : least;
}
__host__ __device__ inline int32_t stream_parts(const KvStreamPlan& p, int32_t range) {
  const int64_t per = stream_part_tokens(p, range);
  return range <= per ? 1 : int32_t((range + per - 1) / per);
}

// The tokens [lo, hi) of a part; empty ones end where the range does. In 64 bits:
// a part may be millions of tokens long and the range end close to 2^31.
struct KvPart {
  int32_t lo;
  int32_t hi;
};
__host__ __device__ inline KvPart stream_part(const KvStreamPlan& p, int32_t begin, int32_t end, uint32_t part) {
  const int64_t per = stream_part_tokens(p, end - begin), lo = begin + int64_t(part) * per, hi = lo + per;
  return KvPart{int32_t(lo < end ? lo : end), int32_t(hi < end ? hi : end)};
}

KvStreamPlan stream_plan(const KvAttendArgs& k, int num_sms);
uint64_t stream_workspace(const KvAttendArgs& k, const KvStreamPlan& p);
cudaError_t launch_attend_stream(const KvAttendArgs& k, const KvStreamPlan& p, cudaStream_t stream);

}  // namespace pf
