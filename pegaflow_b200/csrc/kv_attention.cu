// Attention of a chunk of new tokens over a paged cache (pf_kv_attention_run):
// which kernel takes a call.
#include <algorithm>

#include "kv_attend_stream.h"
#include "kv_attend_tiles.h"

namespace pf {

// Rows (queries times heads of a group) for each KV head: up to 16, which is what the
// streaming kernel's registers hold, it moves the cache's bytes, which bound the call.
// More go to the tile kernel, on the tensor cores. From 17 to about 120 rows over codes
// (250 over 16-bit values) bytes would still be the bound, and the tile kernel is far
// from it: four tokens of 32 sequences over e4m3, 16 rows, take 222 us here (2.5 TB/s),
// eight, 32 rows, 384 there (1.5 TB/s).
static bool streams(const KvAttendArgs& k) {
  const uint64_t n = std::max<uint64_t>(1, k.a.n_tokens);
  const uint64_t most = k.a.max_q ? std::min<uint64_t>(k.a.max_q, n) : n;
  return most * (k.a.q_heads / k.cache.heads) <= kStreamMaxRows;
}

uint64_t kv_attention_workspace(const KvAttendArgs& k, int num_sms) {
  return streams(k) ? stream_workspace(k, stream_plan(k, num_sms)) : tile_plan(k, num_sms).bytes;
}

cudaError_t launch_kv_attention(const KvAttendArgs& k, int num_sms, cudaStream_t stream) {
  return streams(k) ? launch_attend_stream(k, stream_plan(k, num_sms), stream)
                    : launch_attend_tiles(k, tile_plan(k, num_sms), stream);
}

}  // namespace pf
