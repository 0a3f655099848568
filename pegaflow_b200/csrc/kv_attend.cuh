// What the attention kernels share: a sequence's geometry, a row's exact form,
// the joining of parts.
#pragma once

#include "kv_device.cuh"

namespace pf {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// A part's running maximum is raised only when a score passes it by this (in
// powers of two): the exponentials stay below 2^8 times the lift, which fp16, bf16
// and the fp32 sums hold as well as 1, and the accumulators are rescaled rarely.
constexpr float kRaise = 8.0f;
// Where weights become fp16 they are taken this many powers of two up: with kRaise and V scales (below 4) they still end
// at 2^15, and small ones keep fp16's 11 bits down to 2^-21 (2^-19 with V scales) of the row's largest instead of 2^-14.
// A row whose strong tokens hold nothing is what many small weights add up to.
constexpr float kLift = 7.0f;
constexpr float kLiftScaled = 5.0f;

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Kernels launched with programmatic serialisation start while the one before
// them drains: they wait here before they read what it wrote.
__device__ __forceinline__ void wait_for_previous_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_kernel_start() { asm volatile("griddepcontrol.launch_dependents;"); }

// One sequence, with what the device holds about it made safe to index by.
struct KvSeq {
  int32_t first;  // its first query row
  int32_t n;      // its queries, 0 if its offsets are out of order or out of range
  int32_t len;    // its cached tokens, as many as its block table row names
  int32_t pos0;   // position of its first query (negative: it sees nothing)
};

__device__ __forceinline__ KvSeq kv_sequence(const KvAttendArgs& k, uint32_t seq) {
  const int32_t* q_start = reinterpret_cast<const int32_t*>(k.a.q_start);
  KvSeq s;
  s.first = q_start[seq];
  const int64_t n = int64_t(q_start[seq + 1]) - s.first;
  const bool ok = s.first >= 0 && n >= 0 && s.first + n <= int64_t(k.a.n_tokens);
  s.n = ok ? int32_t(n) : 0;
  const int32_t len = reinterpret_cast<const int32_t*>(k.a.kv_len)[seq];
  const int64_t cap = int64_t(k.a.max_blocks) * k.cache.block_size;
  s.len = len < 0 ? 0 : len > cap ? int32_t(cap) : len;
  const int64_t pos0 = int64_t(len) - n;
  s.pos0 = pos0 < -(1 << 30) ? -(1 << 30) : int32_t(pos0);
  if (!ok || len > cap) kv_flag(reinterpret_cast<int32_t*>(k.a.status), PF_KV_BAD_LENGTH);
  return s;
}

// The cached tokens [lo, hi) that query i of a sequence sees.
__device__ __forceinline__ int32_t kv_row_end(const KvAttendArgs& k, const KvSeq& s, int32_t i) {
  return k.a.causal ? max(0, min(s.len, s.pos0 + i + 1)) : s.len;
}
__device__ __forceinline__ int32_t kv_row_begin(const KvAttendArgs& k, const KvSeq& s, int32_t i) {
  if (!k.a.window) return 0;
  const int64_t lo = int64_t(s.pos0) + i + 1 - int64_t(k.a.window);
  return lo < 0 ? 0 : lo > s.len ? s.len : int32_t(lo);
}

// The block of a token, or -1 (flagged) if its entry names none.
__device__ __forceinline__ int32_t kv_block(const KvAttendArgs& k, uint32_t seq, uint32_t entry) {
  const int32_t b = reinterpret_cast<const int32_t*>(k.a.block_table)[int64_t(seq) * k.a.table_stride + entry];
  if (uint64_t(int64_t(b)) < k.cache.num_blocks) return b;
  kv_flag(reinterpret_cast<int32_t*>(k.a.status), PF_KV_BAD_BLOCK);
  return -1;
}

template <uint32_t STORE>
__device__ __forceinline__ float4 kv_load4(const pf_kv_side& side, int64_t block, uint32_t offset, uint32_t head,
                                           uint32_t d) {
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

// One row of the formula over the tokens [lo, hi), by one warp, four tokens at a
// time, masked tokens never touched: lane l gets the values 4 l .. 4 l + 3 of
// sum_j 2^(s_j - m) v_j, and m (in powers of two) and the sum of the weights.
// `alive` (null: none) counts up every 1,024 tokens, for those who wait meanwhile.
//
// Matrix products multiply masked values by a weight of zero, which an infinity
// or a NaN turns into NaN; the kernels send the rows that this may have hit
// through here. It is for such rows alone: it reads the keys once for each row.
template <uint32_t Q, uint32_t STORE>
__device__ __noinline__ void attend_row_exactly(const KvAttendArgs& k, uint32_t seq, int64_t token, uint32_t qh,
                                                uint32_t head, int32_t lo, int32_t hi, float& m, float& l, float4& o,
                                                int* alive) {
  using T = typename KvElem<Q>::type;
  const pf_kv_cache& c = k.cache;
  const uint32_t d = (threadIdx.x & 31) * 4;
  const bool mine = d < c.head_dim;
  float4 q = make_float4(0, 0, 0, 0);
  if (mine) {
    const KvPack<T, 4> v = *reinterpret_cast<const KvPack<T, 4>*>(
        reinterpret_cast<const T*>(k.a.query.data) + token * k.a.query.token_stride + int64_t(qh) * k.a.query.head_stride + d);
    q = make_float4(kv_to_float<Q>(v.v[0]), kv_to_float<Q>(v.v[1]), kv_to_float<Q>(v.v[2]), kv_to_float<Q>(v.v[3]));
  }
  m = -INFINITY;
  l = 0.0f;
  o = make_float4(0, 0, 0, 0);
  constexpr int kAtOnce = 4;
  for (int32_t j0 = lo, n = 0; j0 < hi; j0 += kAtOnce, ++n) {
    float s[kAtOnce];
    float4 v[kAtOnce];
    bool on[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int32_t j = j0 + u, block = j < hi ? kv_block(k, seq, uint32_t(j) / c.block_size) : -1;
      on[u] = block >= 0;
      s[u] = 0.0f;
      v[u] = make_float4(0, 0, 0, 0);
      if (on[u] && mine) {
        const uint32_t offset = uint32_t(j) % c.block_size;
        const float4 x = kv_load4<STORE>(c.key, block, offset, head, d);
        v[u] = kv_load4<STORE>(c.value, block, offset, head, d);
        s[u] = q.x * x.x + q.y * x.y + q.z * x.z + q.w * x.w;
      }
    }
    float top = m;
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      for (int w = 16; w; w >>= 1) s[u] += __shfl_xor_sync(0xffffffffu, s[u], w);
      s[u] = on[u] ? s[u] * (k.a.scale * kLog2e) : -INFINITY;
      top = fmaxf(top, s[u]);
    }
    const float base = top == -INFINITY ? 0.0f : top, keep = exp2f(m - base);
    l *= keep;
    o = make_float4(o.x * keep, o.y * keep, o.z * keep, o.w * keep);
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const float p = exp2f(s[u] - base);
      l += p;
      if (on[u]) o = make_float4(o.x + p * v[u].x, o.y + p * v[u].y, o.z + p * v[u].z, o.w + p * v[u].w);
    }
    m = top;
    if (alive && (n & 255) == 255 && (threadIdx.x & 31) == 0) atomicAdd(alive, 1);
  }
}

}  // namespace pf
