// Attention of a chunk of new tokens over a paged cache (pf_kv_attention_run).
//
// A warp takes one query row: its lanes hold 4 values of the head each, a
// key's score is a shuffle sum, and the softmax is kept as a running maximum
// and sum in fp32 (one pass over the keys).
#include "kv_device.cuh"

namespace pf {
namespace {

constexpr int kThreads = 256;

template <uint32_t STORE>
__device__ __forceinline__ float4 load4(const pf_kv_side& side, int64_t block, uint32_t offset, uint32_t head, uint32_t d) {
  using T = typename KvElem<STORE>::type;
  const T* p = reinterpret_cast<const T*>(side.data) + block * side.block_stride + int64_t(offset) * side.token_stride +
               int64_t(head) * side.head_stride + d;
  const KvPack<T, 4> v = *reinterpret_cast<const KvPack<T, 4>*>(p);
  float s = 1.0f;
  if constexpr (STORE == PF_DTYPE_E4M3 || STORE == PF_DTYPE_INT8) {
    s = reinterpret_cast<const float*>(side.scale)[block * side.scale_block_stride +
                                                   int64_t(offset) * side.scale_token_stride +
                                                   int64_t(head) * side.scale_head_stride];
  }
  return make_float4(kv_to_float<STORE>(v.v[0]) * s, kv_to_float<STORE>(v.v[1]) * s, kv_to_float<STORE>(v.v[2]) * s,
                     kv_to_float<STORE>(v.v[3]) * s);
}

template <uint32_t Q, uint32_t STORE>
__global__ void __launch_bounds__(kThreads) kv_attend_row_kernel(const KvAttendArgs args) {
  using T = typename KvElem<Q>::type;
  const pf_kv_attention& a = args.a;
  const pf_kv_cache& c = args.cache;
  const uint32_t lane = threadIdx.x & 31;
  const uint64_t pair = uint64_t(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
  if (pair >= a.n_tokens * a.q_heads) return;
  const uint32_t token = uint32_t(pair / a.q_heads), qh = uint32_t(pair % a.q_heads);
  const uint32_t head = qh / (a.q_heads / c.heads);
  const int32_t* q_start = reinterpret_cast<const int32_t*>(a.q_start);
  const uint32_t seq = kv_find_seq(q_start, a.n_seqs, token);
  if (seq == a.n_seqs) return;
  const int64_t n = int64_t(q_start[seq + 1]) - q_start[seq], i = int64_t(token) - q_start[seq];
  int64_t len = reinterpret_cast<const int32_t*>(a.kv_len)[seq];
  const int64_t pos = len - n + i;
  if (len > int64_t(a.max_blocks) * c.block_size) {
    kv_flag(reinterpret_cast<int32_t*>(a.status), PF_KV_BAD_LENGTH);
    len = int64_t(a.max_blocks) * c.block_size;
  }
  const int64_t hi = a.causal ? min(len, pos + 1) : len;
  const int64_t lo = a.window ? max(int64_t(0), pos - a.window + 1) : 0;
  const int32_t* table = reinterpret_cast<const int32_t*>(a.block_table) + int64_t(seq) * a.table_stride;
  const uint32_t d = lane * 4;
  const bool mine = d < c.head_dim;
  float4 q = make_float4(0, 0, 0, 0), o = make_float4(0, 0, 0, 0);
  const int64_t at = int64_t(token) * a.query.token_stride + int64_t(qh) * a.query.head_stride + d;
  if (mine) {
    const KvPack<T, 4> v = *reinterpret_cast<const KvPack<T, 4>*>(reinterpret_cast<const T*>(a.query.data) + at);
    q = make_float4(kv_to_float<Q>(v.v[0]), kv_to_float<Q>(v.v[1]), kv_to_float<Q>(v.v[2]), kv_to_float<Q>(v.v[3]));
  }
  float m = -INFINITY, l = 0.0f;
  for (int64_t j = lo; j < hi; ++j) {
    const int64_t block = table[j / c.block_size];
    if (uint64_t(block) >= c.num_blocks) {
      kv_flag(reinterpret_cast<int32_t*>(a.status), PF_KV_BAD_BLOCK);
      continue;
    }
    const uint32_t offset = uint32_t(j % c.block_size);
    float s = 0.0f;
    float4 v = make_float4(0, 0, 0, 0);
    if (mine) {
      const float4 k = load4<STORE>(c.key, block, offset, head, d);
      v = load4<STORE>(c.value, block, offset, head, d);
      s = q.x * k.x + q.y * k.y + q.z * k.z + q.w * k.w;
    }
    for (int w = 16; w; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
    s *= a.scale;
    const float top = fmaxf(m, s);
    const float base = top == -INFINITY ? 0.0f : top;
    const float keep = expf(m - base), p = expf(s - base);
    l = l * keep + p;
    o = make_float4(o.x * keep + p * v.x, o.y * keep + p * v.y, o.z * keep + p * v.z, o.w * keep + p * v.w);
    m = top;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  if (mine) {
    KvPack<T, 4> r;
    r.v[0] = kv_from_float<Q>(o.x * inv);
    r.v[1] = kv_from_float<Q>(o.y * inv);
    r.v[2] = kv_from_float<Q>(o.z * inv);
    r.v[3] = kv_from_float<Q>(o.w * inv);
    const int64_t to = int64_t(token) * a.out.token_stride + int64_t(qh) * a.out.head_stride + d;
    *reinterpret_cast<KvPack<T, 4>*>(reinterpret_cast<T*>(a.out.data) + to) = r;
  }
  if (a.lse && lane == 0) {
    reinterpret_cast<float*>(a.lse)[pair] = l == 0.0f ? -INFINITY : m + logf(l);
  }
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

uint64_t kv_attention_workspace(const KvAttendArgs&, int) { return 0; }

cudaError_t launch_kv_attention(const KvAttendArgs& k, int, cudaStream_t stream) {
  if (k.a.dtype == PF_DTYPE_BF16) {
    launch_row<PF_DTYPE_BF16>(k, stream);
  } else {
    launch_row<PF_DTYPE_FP16>(k, stream);
  }
  return cudaGetLastError();
}

}  // namespace pf
