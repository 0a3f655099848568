// Attention of a chunk of new tokens over a paged cache (pf_kv_attention_run):
// which kernel takes a call.
#include <algorithm>

#include "kv_attend_stream.h"
#include "kv_attend_tiles.h"

namespace pf {

// Few rows for each KV head: the cache's bytes bound the call, and the
// streaming kernel moves them. More: the products do, on the tensor cores.
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
