// Attention of a chunk of new tokens over a paged cache (pf_kv_attention_run).
//
// A warp takes one query row: its lanes hold 4 values of the head each, a
// key's score is a shuffle sum, and the softmax is kept as a running maximum
// and sum in fp32 (one pass over the keys).
#include <algorithm>

#include "kv_attend.cuh"
#include "kv_attend_stream.h"

namespace pf {
namespace {

constexpr int kThreads = 256;

template <uint32_t Q, uint32_t STORE>
__global__ void __launch_bounds__(kThreads) kv_attend_row_kernel(const __grid_constant__ KvAttendArgs k) {
  using T = typename KvElem<Q>::type;
  const uint32_t lane = threadIdx.x & 31, d = lane * 4;
  const uint64_t id = uint64_t(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  if (id >= k.a.n_tokens * k.a.q_heads) return;
  const uint32_t token = uint32_t(id / k.a.q_heads), qh = uint32_t(id % k.a.q_heads);
  const uint32_t seq = kv_find_seq(reinterpret_cast<const int32_t*>(k.a.q_start), k.a.n_seqs, token);
  if (seq == k.a.n_seqs) return;
  const KvSeq s = kv_sequence(k, seq);
  if (!s.n) return;
  const int32_t i = int32_t(token) - s.first;
  float m, l;
  float4 o;
  attend_row_exactly<Q, STORE>(k, seq, token, qh, qh / (k.a.q_heads / k.cache.heads), kv_row_begin(k, s, i),
                               kv_row_end(k, s, i), m, l, o);
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  if (d < k.cache.head_dim) {
    KvPack<T, 4> r;
    r.v[0] = kv_from_float<Q>(o.x * inv);
    r.v[1] = kv_from_float<Q>(o.y * inv);
    r.v[2] = kv_from_float<Q>(o.z * inv);
    r.v[3] = kv_from_float<Q>(o.w * inv);
    *reinterpret_cast<KvPack<T, 4>*>(reinterpret_cast<T*>(k.a.out.data) + int64_t(token) * k.a.out.token_stride +
                                     int64_t(qh) * k.a.out.head_stride + d) = r;
  }
  if (k.a.lse && lane == 0) reinterpret_cast<float*>(k.a.lse)[id] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
}

template <uint32_t Q>
void launch_row(const KvAttendArgs& k, cudaStream_t stream) {
  const uint64_t pairs = k.a.n_tokens * k.a.q_heads;
  const uint32_t grid = static_cast<uint32_t>((pairs + kThreads / 32 - 1) / (kThreads / 32));
  switch (k.cache.dtype) {
    case PF_DTYPE_E4M3: kv_attend_row_kernel<Q, PF_DTYPE_E4M3><<<grid, kThreads, 0, stream>>>(k); break;
    case PF_DTYPE_INT8: kv_attend_row_kernel<Q, PF_DTYPE_INT8><<<grid, kThreads, 0, stream>>>(k); break;
    default: kv_attend_row_kernel<Q, Q><<<grid, kThreads, 0, stream>>>(k); break;
  }
}

}  // namespace

// Few rows for each KV head: the cache's bytes bound the call, and the
// streaming kernel moves them; the row kernel takes the rest.
static bool streams(const KvAttendArgs& k) {
  const uint64_t n = std::max<uint64_t>(1, k.a.n_tokens);
  const uint64_t most = k.a.max_q ? std::min<uint64_t>(k.a.max_q, n) : n;
  return most * (k.a.q_heads / k.cache.heads) <= kStreamMaxRows;
}

uint64_t kv_attention_workspace(const KvAttendArgs& k, int num_sms) {
  return streams(k) ? stream_workspace(k, stream_plan(k, num_sms)) : 0;
}

cudaError_t launch_kv_attention(const KvAttendArgs& k, int num_sms, cudaStream_t stream) {
  if (streams(k)) return launch_attend_stream(k, stream_plan(k, num_sms), stream);
  if (k.a.dtype == PF_DTYPE_BF16) {
    launch_row<PF_DTYPE_BF16>(k, stream);
  } else {
    launch_row<PF_DTYPE_FP16>(k, stream);
  }
  return cudaGetLastError();
}

}  // namespace pf
