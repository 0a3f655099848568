// Writing tokens into a paged cache and reading them back (pf_kv_write,
// pf_kv_read).
//
// Both move every byte once, so HBM bounds them (a small call: the launch), as long
// as the instructions for a value stay few: at HBM's rate an SM has about 15 issue
// slots for 16 bytes of bf16. So values are handled in pairs, both sides' maxima
// travel through one chain of shuffles, indexes are divided by multiplying, and a
// thread has K and V in flight together. Rows that are not aligned for 16-byte
// pieces go element by element in kernels of their own. Measured for 8 heads of 128
// between bf16 and e4m3, calls over changing inputs: 8,192 tokens written in 16.4 us
// (3.1 TB/s: issue slots 68 % busy, the rest is latency, with one row read ahead),
// 10,240 read in 13.2 to 16.4 us (4.8 to 3.9 TB/s). Over the same inputs again and
// again, which L2 then holds, 14.3 and 12.3.
#include <algorithm>

#include "kv_device.cuh"

namespace pf {
namespace {

constexpr int kThreads = 256;

// i / n for i below 2^20 or so: the quotient in fp32, off by less than half of 1 / n.
__device__ __forceinline__ uint32_t divide(uint32_t i, float inverse) { return uint32_t((float(i) + 0.5f) * inverse); }

template <uint32_t STORE>
constexpr float kQmax = STORE == PF_DTYPE_E4M3 ? 448.0f : 127.0f;

// The scale of a row whose largest magnitude is `top`: NaN if it holds a NaN or
// an infinity, whatever its codes then are.
template <uint32_t STORE>
__device__ __forceinline__ float row_scale(float top) {
  const float s = top / kQmax<STORE>;
  return s < kKvSmallestScale ? kKvSmallestScale : s == INFINITY ? NAN : s;
}

// 1 / a given scale. Of none (0), or one so small that it would be infinite, the largest there is: values saturate,
// and zeros stay zeros, which an infinity would make NaN.
__device__ __forceinline__ float inverse(float s) {
  const float inv = 1.0f / s;
  return fabsf(inv) == INFINITY ? copysignf(3.402823466e38f, inv) : inv;
}

// Values of a row that a thread moves when reading: 16 bytes of a 16-bit result, so
// that a warp's stores fill whole sectors (with 16 codes and two stores 32 bytes
// apart, 10,240 tokens of 8 x 128 took 15.1 us instead of 12.1).
constexpr int kReadElems = 8;
constexpr uint32_t kReadMaxTokens = 64;  // of a block

// Strides in bytes that fit 32 bits, so that a step of an address is one
// multiplication (32 x 32 + 64 bits).
struct Strides {
  uint32_t a, b, c;
};
template <typename T>
__device__ __forceinline__ T* address(uint64_t base, const Strides& s, uint32_t a, uint32_t b, uint32_t c) {
  return reinterpret_cast<T*>(base + uint64_t(a) * s.a + uint64_t(b) * s.b + uint64_t(c) * s.c);
}
struct RowStrides {
  Strides key, value, key_scale, value_scale;  // block, token, head
  Strides key_rows, value_rows;                // token, head, -
};

struct WritePlan {
  uint32_t log_l;        // lanes of a row: a power of two
  uint32_t tokens;       // whose rows a block takes together
  uint32_t turns;        // that it needs for them, each a row for each group of lanes
  uint32_t all_turns;
  RowStrides strides;
  float heads_inverse;
  int32_t page_shift;
};

struct ReadPlan {
  uint32_t tokens;       // of a block
  uint32_t pieces;       // of kReadElems values, of a token's rows of one side
  uint32_t row_pieces;   // of one row
  RowStrides strides;
  float pieces_inverse;
  float row_inverse;
  int32_t page_shift;
};

// ------------------------------------------------------------- unaligned rows

// One row into its slot by the lanes of a group, every L-th value each. 8-bit:
// scale = max(amax / qmax, 2^-126) unless it is given, code = rne(clamp(x * (1 /
// scale))). The maximum is taken over the magnitudes' bits as integers, which order
// like the values and put NaN on top, so that a NaN or an infinity reaches the
// scale and the whole row reads as NaN.
template <uint32_t IN, uint32_t STORE>
__device__ __forceinline__ void write_elements(const pf_kv_rows& rows, const pf_kv_side& side, uint32_t token, int64_t block,
                                               int64_t offset, uint32_t head, uint32_t dim, uint32_t lane, uint32_t log_l,
                                               bool on, bool given) {
  using I = typename KvElem<IN>::type;
  using T = typename KvElem<STORE>::type;
  const I* from = reinterpret_cast<const I*>(rows.data) + int64_t(token) * rows.token_stride + int64_t(head) * rows.head_stride;
  T* to = reinterpret_cast<T*>(side.data) + block * side.block_stride + offset * side.token_stride + int64_t(head) * side.head_stride;
  float x[8], inv = 1.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t d = (uint32_t(i) << log_l) + lane;
    x[i] = on && d < dim ? kv_to_float<IN>(from[d]) : 0.0f;
  }
  if constexpr (STORE == PF_DTYPE_E4M3 || STORE == PF_DTYPE_INT8) {
    float* sp = reinterpret_cast<float*>(side.scale) + block * side.scale_block_stride + offset * side.scale_token_stride +
                int64_t(head) * side.scale_head_stride;
    if (given) {
      inv = inverse(on ? *sp : 1.0f);
    } else {
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
      for (uint32_t w = (1u << log_l) >> 1; w; w >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, w));
      const float s = row_scale<STORE>(__uint_as_float(top));
      if (on && lane == 0) *sp = s;
      inv = 1.0f / s;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t d = (uint32_t(i) << log_l) + lane;
    float y = x[i] * inv;
    if constexpr (STORE == PF_DTYPE_E4M3 || STORE == PF_DTYPE_INT8) {
      // The comparisons leave a NaN as it is.
      y = y > kQmax<STORE> ? kQmax<STORE> : y < -kQmax<STORE> ? -kQmax<STORE> : y;
    }
    if (on && d < dim) to[d] = kv_from_float<STORE>(y);
  }
}

template <uint32_t IN, uint32_t STORE>
__global__ void __launch_bounds__(kThreads) kv_write_elements_kernel(const __grid_constant__ KvWriteArgs a, const uint32_t log_l) {
  const uint32_t lane = threadIdx.x & ((1u << log_l) - 1);
  const uint32_t heads = a.cache.heads, dim = a.cache.head_dim;
  const uint64_t pair = uint64_t(blockIdx.x) * (kThreads >> log_l) + (threadIdx.x >> log_l);
  bool on = pair < a.n * heads;
  const uint32_t token = on ? uint32_t(pair) / heads : 0;
  const uint32_t head = on ? uint32_t(pair) - token * heads : 0;
  const int64_t slot = on ? a.slots[token] : -1;
  on = on && slot >= 0;
  if (on && uint64_t(slot) >= a.cache.num_blocks * a.cache.block_size) {
    kv_flag(a.status, PF_KV_BAD_BLOCK);
    on = false;
  }
  const int64_t block = on ? slot / int64_t(a.cache.block_size) : 0;
  const int64_t offset = on ? slot - block * a.cache.block_size : 0;
  write_elements<IN, STORE>(a.key, a.cache.key, token, block, offset, head, dim, lane, log_l, on, a.given_scales);
  write_elements<IN, STORE>(a.value, a.cache.value, token, block, offset, head, dim, lane, log_l, on, a.given_scales);
}

template <uint32_t STORE, uint32_t OUT>
__device__ __forceinline__ void read_elements(const pf_kv_side& side, const pf_kv_rows& rows, int64_t block, int64_t offset,
                                              uint32_t head, uint32_t row, uint32_t dim, uint32_t lane, bool there) {
  using T = typename KvElem<STORE>::type;
  using O = typename KvElem<OUT>::type;
  const T* p = reinterpret_cast<const T*>(side.data) + block * side.block_stride + offset * side.token_stride + int64_t(head) * side.head_stride;
  O* o = reinterpret_cast<O*>(rows.data) + int64_t(row) * rows.token_stride + int64_t(head) * rows.head_stride;
  float s = 1.0f;
  if constexpr (STORE == PF_DTYPE_E4M3 || STORE == PF_DTYPE_INT8) {
    if (there) {
      s = reinterpret_cast<const float*>(side.scale)[block * side.scale_block_stride + offset * side.scale_token_stride +
                                                     int64_t(head) * side.scale_head_stride];
    }
  }
  for (uint32_t d = lane; d < dim; d += 32) o[d] = kv_from_float<OUT>(there ? kv_to_float<STORE>(p[d]) * s : 0.0f);
}

// A warp for a token's row of each side.
template <uint32_t STORE, uint32_t OUT>
__global__ void __launch_bounds__(kThreads) kv_read_elements_kernel(const __grid_constant__ KvReadArgs a) {
  const uint32_t lane = threadIdx.x & 31;
  const uint32_t heads = a.cache.heads, page = a.cache.block_size;
  const uint64_t pair = uint64_t(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
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
  const int64_t offset = token - int64_t(entry * page);
  read_elements<STORE, OUT>(a.cache.key, a.key, block, offset, head, row, a.cache.head_dim, lane, there);
  read_elements<STORE, OUT>(a.cache.value, a.value, block, offset, head, row, a.cache.head_dim, lane, there);
}

// ------------------------------------------------------- aligned rows: writing

template <uint32_t IN>
using EightRaw = KvPack<uint32_t, IN == PF_DTYPE_FP32 ? 8 : 4>;

template <uint32_t IN>
__device__ __forceinline__ void to_pairs(float2 (&x)[4], const EightRaw<IN>& r) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (IN == PF_DTYPE_FP32) {
      x[i] = make_float2(__uint_as_float(r.v[2 * i]), __uint_as_float(r.v[2 * i + 1]));
    } else if constexpr (IN == PF_DTYPE_BF16) {
      x[i] = make_float2(__uint_as_float(r.v[i] << 16), __uint_as_float(r.v[i] & 0xffff0000u));
    } else {
      x[i] = __half22float2(*reinterpret_cast<const __half2*>(&r.v[i]));
    }
  }
}

// The largest magnitudes of a lane's K and V, as bits that order like the values,
// NaN on top: 16-bit types both in one word, K low.
template <uint32_t IN>
struct Tops {
  uint32_t k, v;
  __device__ __forceinline__ Tops(const EightRaw<IN>& a, const EightRaw<IN>& b) {
    if constexpr (IN == PF_DTYPE_FP32) {
      k = v = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) k = max(k, a.v[i] & 0x7fffffffu), v = max(v, b.v[i] & 0x7fffffffu);
    } else {
      uint32_t x = a.v[0] & 0x7fff7fffu, y = b.v[0] & 0x7fff7fffu;
#pragma unroll
      for (int i = 1; i < 4; ++i) x = __vmaxu2(x, a.v[i] & 0x7fff7fffu), y = __vmaxu2(y, b.v[i] & 0x7fff7fffu);
      k = __vmaxu2(__byte_perm(x, y, 0x5410), __byte_perm(x, y, 0x7632));
      v = 0;
    }
  }
  __device__ __forceinline__ void over_group(uint32_t log_l) {
    for (uint32_t w = (1u << log_l) >> 1; w; w >>= 1) {
      if constexpr (IN == PF_DTYPE_FP32) {
        k = max(k, __shfl_xor_sync(0xffffffffu, k, w)), v = max(v, __shfl_xor_sync(0xffffffffu, v, w));
      } else {
        k = __vmaxu2(k, __shfl_xor_sync(0xffffffffu, k, w));
      }
    }
  }
  __device__ __forceinline__ float of(bool value) const {
    if constexpr (IN == PF_DTYPE_FP32) return __uint_as_float(value ? v : k);
    const uint32_t bits = value ? k >> 16 : k & 0xffffu;
    if constexpr (IN == PF_DTYPE_BF16) return __uint_as_float(bits << 16);
    return __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
  }
};

// Eight codes of x * inv. `given`: the values may lie beyond the codes (the
// conversion to e4m3 saturates by itself).
template <uint32_t STORE>
__device__ __forceinline__ uint2 eight_codes(const float2 (&x)[4], float inv, bool given) {
  uint32_t r[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float y[4] = {x[2 * i].x * inv, x[2 * i].y * inv, x[2 * i + 1].x * inv, x[2 * i + 1].y * inv};
    if constexpr (STORE == PF_DTYPE_E4M3) {
      uint16_t lo, hi;
      asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(y[1]), "f"(y[0]));
      asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(y[3]), "f"(y[2]));
      r[i] = uint32_t(lo) | uint32_t(hi) << 16;
    } else {
      uint32_t b[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (given) y[j] = y[j] == y[j] ? fminf(fmaxf(y[j], -127.0f), 127.0f) : 0.0f;
        // Within +-127.5 the sum's low byte is the rounded value (ties to even, as any fp32 sum).
        b[j] = __float_as_uint(y[j] + 12582912.0f);
      }
      r[i] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    }
  }
  return make_uint2(r[0], r[1]);
}

// Blocks that an SM holds: 256 threads of 40 registers, of 64 where a lane's eight values are fp32.
template <uint32_t IN>
constexpr uint32_t kWriteBlocks = IN == PF_DTYPE_FP32 ? 4 : 6;
template <uint32_t IN, uint32_t STORE>
__global__ void __launch_bounds__(kThreads, kWriteBlocks<IN>) kv_write_rows_kernel(const __grid_constant__ KvWriteArgs a, const WritePlan plan) {
  using T = typename KvElem<IN>::type;
  using S = typename KvElem<STORE>::type;
  constexpr bool kQuant = STORE == PF_DTYPE_E4M3 || STORE == PF_DTYPE_INT8;
  const uint32_t lane = threadIdx.x & ((1u << plan.log_l) - 1), d = lane * 8;
  const uint32_t heads = a.cache.heads;
  const bool inside = d < a.cache.head_dim;
  // A turn's row: read while the turn before is worked on.
  struct Row {
    EightRaw<IN> k, v;
    int64_t slot;
    uint32_t head;
  };
  auto read = [&](uint32_t turn) {
    Row r{};
    r.slot = -1;
    if (turn >= plan.all_turns) return r;
    const uint32_t set = plan.turns == 1 ? turn : turn / plan.turns;
    const uint32_t row = (turn - set * plan.turns) * (kThreads >> plan.log_l) + (threadIdx.x >> plan.log_l);
    const uint32_t in = divide(row, plan.heads_inverse);
    const uint64_t token = uint64_t(set) * plan.tokens + in;
    if (in >= plan.tokens || token >= a.n) return r;
    r.head = row - in * heads;
    r.slot = a.slots[token];
    if (inside) {
      r.k = *address<const EightRaw<IN>>(a.key.data, plan.strides.key_rows, uint32_t(token), r.head, d);
      r.v = *address<const EightRaw<IN>>(a.value.data, plan.strides.value_rows, uint32_t(token), r.head, d);
    }
    return r;
  };
  // All lanes of a warp go on together: their groups' shuffles are warp-wide.
  Row next = read(blockIdx.x);
  for (uint32_t turn = blockIdx.x; turn < plan.all_turns; turn += gridDim.x) {
    const EightRaw<IN> k = next.k, v = next.v;
    const int64_t slot = next.slot;
    const uint32_t head = next.head;
    next = read(turn + gridDim.x);
    bool on = slot >= 0;
    if (on && uint64_t(slot) >= a.cache.num_blocks * a.cache.block_size) {
      kv_flag(a.status, PF_KV_BAD_BLOCK);
      on = false;
    }
    // A slot of the cache: its block fits 31 bits.
    const uint32_t block = !on ? 0 : uint32_t(plan.page_shift >= 0 ? slot >> plan.page_shift : slot / int64_t(a.cache.block_size));
    const uint32_t offset = on ? uint32_t(slot) - block * a.cache.block_size : 0;
    float2 x[4], y[4];
    to_pairs<IN>(x, k);
    to_pairs<IN>(y, v);
    S* kp = address<S>(a.cache.key.data, plan.strides.key, block, offset, head) + d;
    S* vp = address<S>(a.cache.value.data, plan.strides.value, block, offset, head) + d;
    if constexpr (kQuant) {
      // Even lanes make K's scale, odd ones V's (a group of one lane both, one after the other).
      float ki, vi;
      float* ksp = address<float>(a.cache.key.scale, plan.strides.key_scale, block, offset, head);
      float* vsp = address<float>(a.cache.value.scale, plan.strides.value_scale, block, offset, head);
      if (a.given_scales) {
        ki = inverse(on ? *ksp : 1.0f), vi = inverse(on ? *vsp : 1.0f);
      } else {
        Tops<IN> tops(k, v);
        tops.over_group(plan.log_l);
        if (plan.log_l) {
          const bool odd = threadIdx.x & 1;
          const float s = row_scale<STORE>(tops.of(odd)), inv = 1.0f / s;
          const float other = __shfl_xor_sync(0xffffffffu, inv, 1);
          ki = odd ? other : inv, vi = odd ? inv : other;
          if (on && lane < 2) *(odd ? vsp : ksp) = s;
        } else {
          const float ks = row_scale<STORE>(tops.of(false)), vs = row_scale<STORE>(tops.of(true));
          ki = 1.0f / ks, vi = 1.0f / vs;
          if (on) *ksp = ks, *vsp = vs;
        }
      }
      const uint2 kc = eight_codes<STORE>(x, ki, a.given_scales), vc = eight_codes<STORE>(y, vi, a.given_scales);
      if (on && inside) {
        *reinterpret_cast<uint2*>(kp) = kc;
        *reinterpret_cast<uint2*>(vp) = vc;
      }
    } else if (on && inside) {
      KvPack<S, 8> kc, vc;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        kc.v[2 * i] = kv_from_float<STORE>(x[i].x), kc.v[2 * i + 1] = kv_from_float<STORE>(x[i].y);
        vc.v[2 * i] = kv_from_float<STORE>(y[i].x), vc.v[2 * i + 1] = kv_from_float<STORE>(y[i].y);
      }
      *reinterpret_cast<KvPack<S, 8>*>(kp) = kc;
      *reinterpret_cast<KvPack<S, 8>*>(vp) = vc;
    }
  }
}

// ------------------------------------------------------- aligned rows: reading

// A thread's piece: 8 codes, or 8 values of 16 bits.
template <uint32_t STORE>
using PieceRaw = KvPack<uint32_t, STORE == PF_DTYPE_E4M3 || STORE == PF_DTYPE_INT8 ? 2 : 4>;
template <uint32_t STORE, uint32_t OUT>
__device__ __forceinline__ void store_piece(typename KvElem<OUT>::type* to, const PieceRaw<STORE>& raw, float s) {
  constexpr int E = kReadElems;
  const auto& w = raw.v;
  float2 x[E / 2];
#pragma unroll
  for (int i = 0; i < int(sizeof(w) / 4); ++i) {
    if constexpr (STORE == PF_DTYPE_E4M3) {
      uint32_t lo, hi;
      asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(lo) : "h"(uint16_t(w[i])));
      asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(hi) : "h"(uint16_t(w[i] >> 16)));
      x[2 * i] = __half22float2(*reinterpret_cast<const __half2*>(&lo));
      x[2 * i + 1] = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    } else if constexpr (STORE == PF_DTYPE_INT8) {
      // 2^23 + (code + 128) as fp32 bits, then minus 2^23 + 128: exact.
      const uint32_t u = w[i] ^ 0x80808080u;
      float y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) y[j] = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440 + j)) - 8388736.0f;
      x[2 * i] = make_float2(y[0], y[1]), x[2 * i + 1] = make_float2(y[2], y[3]);
    } else if constexpr (STORE == PF_DTYPE_BF16) {
      x[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    } else {
      x[i] = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    }
  }
  if constexpr (STORE == PF_DTYPE_E4M3 || STORE == PF_DTYPE_INT8) {
#pragma unroll
    for (int i = 0; i < E / 2; ++i) x[i].x *= s, x[i].y *= s;
  }
  constexpr int kPerStore = 16 / sizeof(typename KvElem<OUT>::type);  // values
#pragma unroll
  for (int i = 0; i < E; i += kPerStore) {
    uint4 r;
    if constexpr (OUT == PF_DTYPE_FP32) {
      r = make_uint4(__float_as_uint(x[i / 2].x), __float_as_uint(x[i / 2].y), __float_as_uint(x[i / 2 + 1].x), __float_as_uint(x[i / 2 + 1].y));
    } else {
      uint32_t p[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (OUT == PF_DTYPE_BF16) {
          asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(p[j]) : "f"(x[i / 2 + j].y), "f"(x[i / 2 + j].x));
        } else {
          asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(p[j]) : "f"(x[i / 2 + j].y), "f"(x[i / 2 + j].x));
        }
      }
      r = make_uint4(p[0], p[1], p[2], p[3]);
    }
    *reinterpret_cast<uint4*>(to + i) = r;
  }
}

// A block takes some rows of the result (tokens); their sequences and blocks are
// looked up once each, by one thread, then the threads go over the rows' pieces.
template <uint32_t STORE, uint32_t OUT>
__global__ void __launch_bounds__(kThreads) kv_read_rows_kernel(const __grid_constant__ KvReadArgs a, const ReadPlan plan) {
  constexpr int E = kReadElems;
  constexpr bool kQuant = STORE == PF_DTYPE_E4M3 || STORE == PF_DTYPE_INT8;
  using T = typename KvElem<STORE>::type;
  using O = typename KvElem<OUT>::type;
  __shared__ int2 place[kReadMaxTokens];  // {block, offset in it}; block -1: zeros, -2: not a sequence's row
  const uint32_t first = blockIdx.x * plan.tokens;
  const uint32_t tokens = uint32_t(min(uint64_t(plan.tokens), a.n_rows - first));
  if (threadIdx.x < tokens) {
    const uint32_t row = first + threadIdx.x, page = a.cache.block_size;
    const uint32_t seq = kv_find_seq(a.starts, a.n_seqs, row);
    int2 p = make_int2(-2, 0);
    if (seq < a.n_seqs) {
      const uint64_t token = uint64_t(int64_t(row) - a.starts[seq]);
      const uint64_t entry = plan.page_shift >= 0 ? token >> plan.page_shift : token / page;
      p = make_int2(-1, int32_t(token - entry * page));
      if (entry < a.max_blocks) {
        const int32_t b = a.block_table[int64_t(seq) * a.table_stride + int64_t(entry)];
        if (uint64_t(int64_t(b)) < a.cache.num_blocks) {
          p.x = b;
        } else {
          kv_flag(a.status, PF_KV_BAD_BLOCK);
        }
      } else {
        kv_flag(a.status, PF_KV_BAD_LENGTH);
      }
    }
    place[threadIdx.x] = p;
  }
  __syncthreads();
  const uint32_t pieces = tokens * plan.pieces;
#pragma unroll 2
  for (uint32_t i = threadIdx.x; i < pieces; i += kThreads) {
    const uint32_t in = divide(i, plan.pieces_inverse), at = i - in * plan.pieces;
    const uint32_t head = divide(at, plan.row_inverse), d = (at - head * plan.row_pieces) * E;
    const int2 p = place[in];
    if (p.x == -2) continue;
    const uint32_t b = uint32_t(max(p.x, 0)), offset = uint32_t(p.y);
    PieceRaw<STORE> k{}, v{};
    float ks = 0.0f, vs = 0.0f;
    if (p.x >= 0) {
      k = *reinterpret_cast<const PieceRaw<STORE>*>(address<const T>(a.cache.key.data, plan.strides.key, b, offset, head) + d);
      v = *reinterpret_cast<const PieceRaw<STORE>*>(address<const T>(a.cache.value.data, plan.strides.value, b, offset, head) + d);
      if constexpr (kQuant) {
        ks = *address<const float>(a.cache.key.scale, plan.strides.key_scale, b, offset, head);
        vs = *address<const float>(a.cache.value.scale, plan.strides.value_scale, b, offset, head);
      }
    }
    const uint32_t row = first + in;
    store_piece<STORE, OUT>(address<O>(a.key.data, plan.strides.key_rows, row, head, 0) + d, k, ks);
    store_piece<STORE, OUT>(address<O>(a.value.data, plan.strides.value_rows, row, head, 0) + d, v, vs);
  }
}

// ------------------------------------------------------------------ launching

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

// The strides in bytes, if they fit 32 bits.
bool fit(const int64_t (&s)[3], uint64_t bytes, Strides* out) {
  for (int64_t x : s) {
    if (x < 0 || uint64_t(x) * bytes > UINT32_MAX) return false;
  }
  *out = Strides{uint32_t(s[0] * bytes), uint32_t(s[1] * bytes), uint32_t(s[2] * bytes)};
  return true;
}
bool fit_all(const pf_kv_cache& c, const pf_kv_rows& key, const pf_kv_rows& value, uint32_t dtype, RowStrides* out) {
  const uint64_t n = kv_dtype_bytes(c.dtype), m = kv_dtype_bytes(dtype);
  return fit({c.key.block_stride, c.key.token_stride, c.key.head_stride}, n, &out->key) &&
         fit({c.value.block_stride, c.value.token_stride, c.value.head_stride}, n, &out->value) &&
         fit({c.key.scale_block_stride, c.key.scale_token_stride, c.key.scale_head_stride}, 4, &out->key_scale) &&
         fit({c.value.scale_block_stride, c.value.scale_token_stride, c.value.scale_head_stride}, 4, &out->value_scale) &&
         fit({key.token_stride, key.head_stride, 1}, m, &out->key_rows) &&
         fit({value.token_stride, value.head_stride, 1}, m, &out->value_rows);
}

// Lanes of a row's group: the power of two that covers dim / 8, at most 32.
uint32_t group_log(uint32_t dim) {
  uint32_t l = 0;
  while ((8u << l) < dim) ++l;
  return l;
}

template <uint32_t IN, uint32_t STORE>
void write_as(const KvWriteArgs& a, cudaStream_t stream) {
  const uint32_t log_l = group_log(a.cache.head_dim), heads = a.cache.heads, groups = kThreads >> log_l;
  RowStrides strides;
  if (side_packs(a.cache, a.cache.key, 8) && side_packs(a.cache, a.cache.value, 8) && rows_pack(a.key, IN, 8) &&
      rows_pack(a.value, IN, 8) && fit_all(a.cache, a.key, a.value, IN, &strides)) {
    const uint32_t tokens = std::max(1u, groups / heads), turns = (tokens * heads + groups - 1) / groups;
    const uint32_t all = static_cast<uint32_t>((a.n + tokens - 1) / tokens) * turns;
    const WritePlan plan{log_l, tokens, turns, all, strides, 1.0f / float(heads), page_shift(a.cache)};
    // As many blocks as an SM holds, so that all but a small call's rows are read a turn ahead.
    const uint32_t grid = std::min(all, a.num_sms * kWriteBlocks<IN>);
    kv_write_rows_kernel<IN, STORE><<<grid, kThreads, 0, stream>>>(a, plan);
  } else {
    kv_write_elements_kernel<IN, STORE><<<static_cast<uint32_t>((a.n * heads + groups - 1) / groups), kThreads, 0, stream>>>(a, log_l);
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
  constexpr int E = kReadElems;
  const uint32_t heads = a.cache.heads;
  RowStrides strides;
  if (side_packs(a.cache, a.cache.key, E) && side_packs(a.cache, a.cache.value, E) && rows_pack(a.key, OUT, E) &&
      rows_pack(a.value, OUT, E) && fit_all(a.cache, a.key, a.value, OUT, &strides)) {
    const uint32_t row = a.cache.head_dim / E, pieces = heads * row;
    // Two pieces for each thread, up to eight as long as an SM gets a dozen blocks: fewer blocks look rows up and wait
    // less (46,000 rows of 5 heads of 80: 23.2 us with two, 20.0 with eight; 2,048 rows of 12 of 64 with a write
    // before: 7.8 us with two, 10.7 with eight).
    const uint64_t each = a.n_rows * pieces / (uint64_t(kThreads) * 12 * a.num_sms);
    const uint32_t turns = static_cast<uint32_t>(std::min<uint64_t>(8, std::max<uint64_t>(2, each)));
    const uint32_t tokens = std::min(kReadMaxTokens, std::max(1u, turns * kThreads / pieces));
    const ReadPlan plan{tokens, pieces, row, strides, 1.0f / float(pieces), 1.0f / float(row), page_shift(a.cache)};
    kv_read_rows_kernel<STORE, OUT><<<static_cast<uint32_t>((a.n_rows + tokens - 1) / tokens), kThreads, 0, stream>>>(a, plan);
  } else {
    const uint64_t pairs = a.n_rows * heads;
    kv_read_elements_kernel<STORE, OUT><<<static_cast<uint32_t>((pairs + kThreads / 32 - 1) / (kThreads / 32)), kThreads, 0, stream>>>(a);
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
