// Writing tokens into a paged cache and reading them back (pf_kv_write,
// pf_kv_read): one row of head_dim values at a time.
//
// Both move every byte once and compute a few operations a value, so HBM bounds
// them (a small call: the launch). A group of lanes owns the row of one token
// and head, K and V together: each lane holds consecutive values of both, so
// that two 16-byte loads are in flight, and the row's maximum is a shuffle
// within the group. Rows that are not aligned for that go element by element,
// lanes side by side.
#include <algorithm>

#include "kv_device.cuh"

namespace pf {
namespace {

constexpr int kThreads = 256;
constexpr int kWriteElems = 8;  // values of a row that one lane holds

template <uint32_t STORE>
constexpr float kQmax = STORE == PF_DTYPE_E4M3 ? 448.0f : 127.0f;

// Value k of a lane: consecutive values (vector rows), or every L-th.
template <bool VEC, int E>
__device__ __forceinline__ uint32_t element(uint32_t lane, uint32_t log_l, int k) {
  return VEC ? lane * E + k : (uint32_t(k) << log_l) + lane;
}

template <uint32_t IN, bool VEC>
__device__ __forceinline__ void load_row(const pf_kv_rows& rows, uint32_t token, uint32_t head, uint32_t dim,
                                         uint32_t lane, uint32_t log_l, float (&x)[kWriteElems]) {
  using T = typename KvElem<IN>::type;
  const T* p = reinterpret_cast<const T*>(rows.data) + int64_t(token) * rows.token_stride + int64_t(head) * rows.head_stride;
  if constexpr (VEC) {
    KvPack<T, kWriteElems> v{};
    if (lane * kWriteElems < dim) v = *reinterpret_cast<const KvPack<T, kWriteElems>*>(p + lane * kWriteElems);
#pragma unroll
    for (int k = 0; k < kWriteElems; ++k) x[k] = kv_to_float<IN>(v.v[k]);
  } else {
#pragma unroll
    for (int k = 0; k < kWriteElems; ++k) {
      const uint32_t d = element<VEC, kWriteElems>(lane, log_l, k);
      x[k] = d < dim ? kv_to_float<IN>(p[d]) : 0.0f;
    }
  }
}

// One row into its slot. 8-bit: scale = max(amax / qmax, 2^-126) unless it is
// given, code = rne(clamp(x * (1 / scale))). The maximum is taken over the
// magnitudes' bits as integers, which order like the values and put NaN on top,
// so that a NaN or an infinity reaches the scale and the whole row reads as NaN.
template <uint32_t STORE, bool VEC>
__device__ __forceinline__ void store_row(const pf_kv_side& side, int64_t block, uint32_t offset, uint32_t head,
                                          uint32_t dim, uint32_t lane, uint32_t log_l, bool on, bool given,
                                          const float (&x)[kWriteElems]) {
  using T = typename KvElem<STORE>::type;
  KvPack<T, kWriteElems> out;
  if constexpr (STORE == PF_DTYPE_E4M3 || STORE == PF_DTYPE_INT8) {
    float* sp = reinterpret_cast<float*>(side.scale) + block * side.scale_block_stride +
                int64_t(offset) * side.scale_token_stride + int64_t(head) * side.scale_head_stride;
    float s;
    if (given) {
      s = on ? *sp : 1.0f;
    } else {
      uint32_t top = 0;
#pragma unroll
      for (int k = 0; k < kWriteElems; ++k) top = max(top, __float_as_uint(x[k]) & 0x7fffffffu);
      for (uint32_t w = (1u << log_l) >> 1; w; w >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, w));
      s = __uint_as_float(top) / kQmax<STORE>;
      s = s < kKvSmallestScale ? kKvSmallestScale : s;
      if (on && lane == 0) *sp = s;
    }
    const float inv = 1.0f / s;
#pragma unroll
    for (int k = 0; k < kWriteElems; ++k) {
      const float y = x[k] * inv;
      // The comparisons leave a NaN as it is.
      const float c = y > kQmax<STORE> ? kQmax<STORE> : y < -kQmax<STORE> ? -kQmax<STORE> : y;
      out.v[k] = kv_from_float<STORE>(c);
    }
  } else {
#pragma unroll
    for (int k = 0; k < kWriteElems; ++k) out.v[k] = kv_from_float<STORE>(x[k]);
  }
  if (!on) return;
  T* p = reinterpret_cast<T*>(side.data) + block * side.block_stride + int64_t(offset) * side.token_stride +
         int64_t(head) * side.head_stride;
  if constexpr (VEC) {
    if (lane * kWriteElems < dim) *reinterpret_cast<KvPack<T, kWriteElems>*>(p + lane * kWriteElems) = out;
  } else {
#pragma unroll
    for (int k = 0; k < kWriteElems; ++k) {
      const uint32_t d = element<VEC, kWriteElems>(lane, log_l, k);
      if (d < dim) p[d] = out.v[k];
    }
  }
}

template <uint32_t IN, uint32_t STORE, bool VEC>
__global__ void __launch_bounds__(kThreads) kv_write_kernel(const KvWriteArgs a, const uint32_t log_l) {
  const uint32_t lane = threadIdx.x & ((1u << log_l) - 1);
  const uint32_t heads = a.cache.heads, dim = a.cache.head_dim;
  const uint64_t pair = uint64_t(blockIdx.x) * (kThreads >> log_l) + (threadIdx.x >> log_l);
  bool on = pair < a.n * heads;
  const uint32_t token = on ? uint32_t(pair) / heads : 0;
  const uint32_t head = on ? uint32_t(pair) - token * heads : 0;
  const int64_t slot = on ? a.slots[token] : -1;
  float k[kWriteElems], v[kWriteElems];
  load_row<IN, VEC>(a.key, token, head, dim, lane, log_l, k);
  load_row<IN, VEC>(a.value, token, head, dim, lane, log_l, v);
  on = on && slot >= 0;
  if (on && uint64_t(slot) >= a.cache.num_blocks * a.cache.block_size) {
    kv_flag(a.status, PF_KV_BAD_BLOCK);
    on = false;
  }
  const uint64_t block = on ? uint64_t(slot) / a.cache.block_size : 0;
  const uint32_t offset = on ? uint32_t(uint64_t(slot) - block * a.cache.block_size) : 0;
  store_row<STORE, VEC>(a.cache.key, int64_t(block), offset, head, dim, lane, log_l, on, a.given_scales, k);
  store_row<STORE, VEC>(a.cache.value, int64_t(block), offset, head, dim, lane, log_l, on, a.given_scales, v);
}

// Values of a row that one lane holds when reading: a 16-byte load's worth.
template <uint32_t STORE>
constexpr int kReadElems = STORE == PF_DTYPE_E4M3 || STORE == PF_DTYPE_INT8 ? 16 : 8;

template <uint32_t STORE, uint32_t OUT, bool VEC>
__device__ __forceinline__ void move_row(const pf_kv_side& side, const pf_kv_rows& rows, int64_t block, uint32_t offset,
                                         uint32_t head, uint32_t row, uint32_t dim, uint32_t lane, uint32_t log_l,
                                         bool there) {
  constexpr int E = kReadElems<STORE>;
  using T = typename KvElem<STORE>::type;
  using O = typename KvElem<OUT>::type;
  const T* p = reinterpret_cast<const T*>(side.data) + block * side.block_stride + int64_t(offset) * side.token_stride +
               int64_t(head) * side.head_stride;
  O* o = reinterpret_cast<O*>(rows.data) + int64_t(row) * rows.token_stride + int64_t(head) * rows.head_stride;
  float s = 1.0f;
  if constexpr (STORE == PF_DTYPE_E4M3 || STORE == PF_DTYPE_INT8) {
    if (there) {
      s = reinterpret_cast<const float*>(side.scale)[block * side.scale_block_stride +
                                                     int64_t(offset) * side.scale_token_stride +
                                                     int64_t(head) * side.scale_head_stride];
    }
  }
  if constexpr (VEC) {
    if (lane * E >= dim) return;
    KvPack<O, E> out{};
    if (there) {
      const KvPack<T, E> v = *reinterpret_cast<const KvPack<T, E>*>(p + lane * E);
#pragma unroll
      for (int k = 0; k < E; ++k) out.v[k] = kv_from_float<OUT>(kv_to_float<STORE>(v.v[k]) * s);
    }
    *reinterpret_cast<KvPack<O, E>*>(o + lane * E) = out;
  } else {
#pragma unroll
    for (int k = 0; k < E; ++k) {
      const uint32_t d = element<VEC, E>(lane, log_l, k);
      if (d < dim) o[d] = kv_from_float<OUT>(there ? kv_to_float<STORE>(p[d]) * s : 0.0f);
    }
  }
}

template <uint32_t STORE, uint32_t OUT, bool VEC>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const KvReadArgs a, const uint32_t log_l) {
  const uint32_t lane = threadIdx.x & ((1u << log_l) - 1);
  const uint32_t heads = a.cache.heads, page = a.cache.block_size;
  const uint64_t pair = uint64_t(blockIdx.x) * (kThreads >> log_l) + (threadIdx.x >> log_l);
  if (pair >= a.n_rows * heads) return;
  const uint32_t row = uint32_t(pair) / heads, head = uint32_t(pair) - row * heads;
  const uint32_t seq = kv_find_seq(a.starts, a.n_seqs, row);
  if (seq == a.n_seqs) return;
  const int64_t token = int64_t(row) - a.starts[seq];
  const uint64_t entry = uint64_t(token) / page;
  int64_t block = -1;
  if (entry < a.max_blocks) {
    block = a.block_table[int64_t(seq) * a.table_stride + int64_t(entry)];
    if (uint64_t(block) >= a.cache.num_blocks) kv_flag(a.status, PF_KV_BAD_BLOCK);
  } else {
    kv_flag(a.status, PF_KV_BAD_LENGTH);
  }
  const bool there = uint64_t(block) < a.cache.num_blocks;
  if (!there) block = 0;
  const uint32_t offset = uint32_t(uint64_t(token) - entry * page);
  move_row<STORE, OUT, VEC>(a.cache.key, a.key, block, offset, head, row, a.cache.head_dim, lane, log_l, there);
  move_row<STORE, OUT, VEC>(a.cache.value, a.value, block, offset, head, row, a.cache.head_dim, lane, log_l, there);
}

bool multiple(int64_t a, int64_t b, int64_t c, int64_t of) { return a % of == 0 && b % of == 0 && c % of == 0; }

// Whether E consecutive values of a row can be moved as one pack.
bool side_packs(const pf_kv_cache& c, const pf_kv_side& s, int e) {
  const uint64_t bytes = std::min<uint64_t>(16, uint64_t(e) * kv_dtype_bytes(c.dtype));
  return c.head_dim % e == 0 && s.data % bytes == 0 &&
         multiple(s.block_stride, s.token_stride, s.head_stride, int64_t(bytes / kv_dtype_bytes(c.dtype)));
}
bool rows_pack(const pf_kv_rows& r, uint32_t dtype, int e) {
  const uint64_t bytes = std::min<uint64_t>(16, uint64_t(e) * kv_dtype_bytes(dtype));
  return r.data % bytes == 0 && multiple(r.token_stride, r.head_stride, 0, int64_t(bytes / kv_dtype_bytes(dtype)));
}

// Lanes of a row's group: the power of two that covers dim / e, at most 32.
uint32_t group_log(uint32_t dim, int e) {
  uint32_t l = 0;
  while ((uint32_t(e) << l) < dim) ++l;
  return l;
}

uint32_t grid_for(uint64_t pairs, uint32_t log_l) {
  const uint64_t per = kThreads >> log_l;
  return static_cast<uint32_t>((pairs + per - 1) / per);
}

template <uint32_t IN, uint32_t STORE>
void write_as(const KvWriteArgs& a, cudaStream_t stream) {
  const uint32_t log_l = group_log(a.cache.head_dim, kWriteElems);
  const uint32_t grid = grid_for(a.n * a.cache.heads, log_l);
  const bool vec = side_packs(a.cache, a.cache.key, kWriteElems) && side_packs(a.cache, a.cache.value, kWriteElems) &&
                   rows_pack(a.key, IN, kWriteElems) && rows_pack(a.value, IN, kWriteElems);
  if (vec) {
    kv_write_kernel<IN, STORE, true><<<grid, kThreads, 0, stream>>>(a, log_l);
  } else {
    kv_write_kernel<IN, STORE, false><<<grid, kThreads, 0, stream>>>(a, log_l);
  }
}

template <uint32_t IN>
void write_from(const KvWriteArgs& a, cudaStream_t stream) {
  switch (a.cache.dtype) {
    case PF_DTYPE_BF16: return write_as<IN, PF_DTYPE_BF16>(a, stream);
    case PF_DTYPE_FP16: return write_as<IN, PF_DTYPE_FP16>(a, stream);
    case PF_DTYPE_E4M3: return write_as<IN, PF_DTYPE_E4M3>(a, stream);
    default: return write_as<IN, PF_DTYPE_INT8>(a, stream);
  }
}

template <uint32_t STORE, uint32_t OUT>
void read_as(const KvReadArgs& a, cudaStream_t stream) {
  constexpr int E = kReadElems<STORE>;
  const uint32_t log_l = group_log(a.cache.head_dim, E);
  const uint32_t grid = grid_for(a.n_rows * a.cache.heads, log_l);
  const bool vec = side_packs(a.cache, a.cache.key, E) && side_packs(a.cache, a.cache.value, E) &&
                   rows_pack(a.key, OUT, E) && rows_pack(a.value, OUT, E);
  if (vec) {
    kv_read_kernel<STORE, OUT, true><<<grid, kThreads, 0, stream>>>(a, log_l);
  } else {
    kv_read_kernel<STORE, OUT, false><<<grid, kThreads, 0, stream>>>(a, log_l);
  }
}

template <uint32_t STORE>
void read_from(const KvReadArgs& a, cudaStream_t stream) {
  switch (a.dtype) {
    case PF_DTYPE_BF16: return read_as<STORE, PF_DTYPE_BF16>(a, stream);
    case PF_DTYPE_FP16: return read_as<STORE, PF_DTYPE_FP16>(a, stream);
    default: return read_as<STORE, PF_DTYPE_FP32>(a, stream);
  }
}

}  // namespace

cudaError_t launch_kv_write(const KvWriteArgs& a, cudaStream_t stream) {
  switch (a.dtype) {
    case PF_DTYPE_BF16: write_from<PF_DTYPE_BF16>(a, stream); break;
    case PF_DTYPE_FP16: write_from<PF_DTYPE_FP16>(a, stream); break;
    default: write_from<PF_DTYPE_FP32>(a, stream); break;
  }
  return cudaGetLastError();
}

cudaError_t launch_kv_read(const KvReadArgs& a, cudaStream_t stream) {
  switch (a.cache.dtype) {
    case PF_DTYPE_BF16: read_from<PF_DTYPE_BF16>(a, stream); break;
    case PF_DTYPE_FP16: read_from<PF_DTYPE_FP16>(a, stream); break;
    case PF_DTYPE_E4M3: read_from<PF_DTYPE_E4M3>(a, stream); break;
    default: read_from<PF_DTYPE_INT8>(a, stream); break;
  }
  return cudaGetLastError();
}

}  // namespace pf
