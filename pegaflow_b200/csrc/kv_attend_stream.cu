// Attention of few query rows over long caches (decoding): the cache is streamed
// once, so HBM bounds it.
//
// For one sequence and one KV head, the rows (its queries times the heads of the
// group) are at most 8 or 16. A CTA takes a part of the tokens for them; its four
// warps take batches of 32 tokens in turn, each warp on its own: its running
// maximum, its sums, its accumulators, joined at the end of the part. Parts of a
// sequence are joined by their cluster, where they are one, or by a second kernel.
// Measured: 64 sequences of 1K to 16K tokens, 32 heads on 8 of 128 over e4m3, 1.2 GB,
// 252 us in calls without a pause (4.7 TB/s; 1,777 MHz under the power limit), 234 in
// twenty (1,965 MHz); one of 1,000 in bf16 8.2 us, which are latency.
//
// Each warp copies its rows (16-byte cp.async, from wherever the block table says)
// into a ring of its own in shared memory, two steps of 16 tokens ahead: with 8 to
// 16 warps on an SM 128 KB and more are on their way, what HBM's latency takes at
// full rate. (Loads into registers, one step ahead, reached 60 % of it.)
//
// The products are transposed, so that a warp's matrix instructions (m16n8k16)
// have 16 tokens or 16 values on the long side and 8 rows on the short one:
//   S^T = K Q^T (16 tokens x 8 rows),  O^T += V^T P^T (16 values x 8 rows).
// Their sums run over the head's values and over the tokens, whose order is free:
// a lane takes as its share of a row whatever 16 bytes it can read at once, and no
// fragment needs a transposing read: codes and values alike go from 16-byte reads
// into the instructions. A V^T fragment pairs two tokens' values: one byte
// permutation. P^T is S^T transposed: one movmatrix.
//
// 8-bit codes become fp16, which holds all of e4m3 and int8 exactly; the scales
// stay in fp32: K's multiplies the score, V's the weight. Weights times V's scales
// are rounded to fp16 for the second product, so they have a running maximum of their
// own, of the score plus the V scale's exponent, and an exponential of their own: a
// row's largest weight times scale is near 1 whatever the scales are, what the row
// does not see has no part in it, and the sum of the weights goes by the scores
// alone. A bf16
// query is brought into fp16's range by a power of two for each row: values down
// to 2^-28 of the row's largest stay exact, smaller ones are off by at most 2^-39
// of it.
#include <algorithm>

#include "kv_attend.cuh"
#include "kv_attend_stream.h"

namespace pf {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kBatch = 32;  // tokens whose addresses and scales a warp stages at once, one a lane
constexpr int kStep = 16;   // tokens of one matrix instruction
constexpr int kRing = 3;    // steps in a warp's ring

struct Staged {
  int64_t key;    // byte offset of the token's K row, -1 if it has none
  int64_t value;
  float key_scale;
  float value_scale;
};

template <bool BF16>
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
  if constexpr (BF16) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}

// 16 bytes into shared memory, zeros if they are not there.
__device__ __forceinline__ void copy16(void* to, const char* from, const char* valid, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(uint32_t(__cvta_generic_to_shared(to))),
               "l"(there ? from : valid), "r"(there ? 16 : 0)
               : "memory");
}

__device__ __forceinline__ void copy16(void* to, const char* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(uint32_t(__cvta_generic_to_shared(to))), "l"(from) : "memory");
}

// A value in the shared memory of another CTA of the cluster.
__device__ __forceinline__ float load_of(const float* p, uint32_t rank) {
  float v;
  asm volatile("{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %1, %2;\n ld.shared::cluster.f32 %0, [a];\n}"
               : "=f"(v)
               : "r"(uint32_t(__cvta_generic_to_shared(p))), "r"(rank)
               : "memory");
  return v;
}
__device__ __forceinline__ void cluster_meets() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (BF16) {
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  } else {
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  }
  return r;
}

template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t x) {
  if constexpr (BF16) return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&x));
}

// y times 2^by, in two steps: the power alone may lie outside fp32.
__device__ __forceinline__ float in_units(float y, float by) {
  const float half = exp2f(0.5f * by);
  return y * half * half;
}

// Two codes in the low (HIGH: high) 16 bits of x as two fp16 values.
template <uint32_t STORE, bool HIGH>
__device__ __forceinline__ uint32_t codes_to_half2(uint32_t x) {
  uint32_t r;
  if constexpr (STORE == PF_DTYPE_E4M3) {
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(uint16_t(HIGH ? x >> 16 : x)));
  } else {
    // 1024 + (code + 128) as fp16 bits, then minus 1152: all exact.
    const uint32_t biased = __byte_perm(x ^ 0x80808080u, 0x64646464u, HIGH ? 0x4342 : 0x4140);
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&biased), __floats2half2_rn(1152.0f, 1152.0f));
    r = *reinterpret_cast<const uint32_t*>(&v);
  }
  return r;
}

// Q, STORE: types. DP: head_dim rounded up to 64 or 128. NT: 8-row tiles.
template <uint32_t Q, uint32_t STORE, int DP, int NT>
struct Stream {
  static constexpr bool kQuant = STORE == PF_DTYPE_E4M3 || STORE == PF_DTYPE_INT8;
  static constexpr bool kBf16 = !kQuant && Q == PF_DTYPE_BF16;  // type of the products
  // The rounding of the weights is made good by a second product with what it left: HBM bounds the kernel, not the
  // products, and it takes no time (one sequence of 1,000 in bf16 8.2 us with and without, four of 32K 22.5; off by
  // 1.6e-3 in all, the result's own rounding, without by 2.1e-3). Not where a bf16 result over codes has weights in fp16:
  // they are eight times as fine as the result.
  static constexpr bool kExact = !kQuant || Q == PF_DTYPE_FP16;
  // Powers of two that weights (times V scales) are taken up when they become fp16, and that their sum goes with them.
  static constexpr float kUp = kBf16 ? 0.0f : kQuant ? kLiftScaled : kLift;
  static constexpr float kSumUp = kQuant ? 0.0f : kUp;
  static constexpr int kElt = kQuant ? 1 : 2;
  static constexpr int kRows = 8 * NT;
  static constexpr int kChunk = 16 / kElt;           // values of 16 bytes
  static constexpr int kKeyReads = DP * kElt / 64;   // 16-byte reads of a lane for one K row
  static constexpr int kValueBytes = DP / 8 * kElt;  // of a lane for one V row
  static constexpr int kValueRead = kValueBytes < 16 ? kValueBytes : 16;
  static constexpr int kValueReads = kValueBytes / kValueRead;
  static constexpr int kTiles = DP / 16;
  static constexpr int kRowBytes = DP * kElt;
  static constexpr int kPieces = kRowBytes / 16;
  // CTAs on an SM: as many as shared memory holds (DP 128 in 16 bits: two), registers permitting.
  static constexpr int kCtas = kRowBytes == 256 ? 2 : NT == 1 ? 4 : 2;

  // A step's rows. 16-byte pieces are swizzled by the row so that a quarter warp's reads meet all banks: K's are
  // of two neighbouring rows and four pieces, V's of four even (or odd) rows and two pieces.
  struct Step {
    unsigned char key[kStep][kRowBytes];
    unsigned char value[kStep][kRowBytes];
  };
  // A V scale as a power of two, which the values' maximum counts, and what is left of it: 1 to 2 (up to 4 from 2^127 on),
  // less below 2^-126, 0, an infinity or NaN.
  struct Scale {
    float exponent;
    float rest;
  };
  static __device__ __forceinline__ Scale split(float scale) {
    if constexpr (!kQuant) return Scale{0.0f, 1.0f};
    const int e = min(max(int(__float_as_uint(scale) >> 23 & 255) - 127, -126), 126);
    return Scale{float(e), scale * __uint_as_float(uint32_t(127 - e) << 23)};
  }
  static __device__ __forceinline__ int key_piece(int row, int piece) { return kPieces >= 8 ? piece ^ (row & 1) << 2 : piece; }
  static __device__ __forceinline__ int value_piece(int row, int piece) { return kPieces >= 8 ? piece ^ (row >> 1 & 3) << 1 : piece ^ (row >> 1 & 3); }
  struct Shared {
    union {
      Step ring[kWarps][kRing];
      float o[kWarps][sizeof(Step) * kRing / 4];  // [row][value] of a warp, when its ring is done with
    };
    Staged staged[kWarps][2][kBatch];
    float m[kWarps][kRows];
    float l[kWarps][kRows];
    float mv[kWarps][kRows];
    float part_m[kRows];  // the CTA's own, for the others of its cluster
    float part_l[kRows];
    float part_mv[kRows];
    int bad[kRows];
  };
  static_assert(sizeof(Step) * kRing >= kRows * DP * 4, "a warp's sums fit into its ring");
};

template <uint32_t Q, uint32_t STORE, int DP, int NT, bool CLUSTER>
__global__ void __launch_bounds__(kThreads, (Stream<Q, STORE, DP, NT>::kCtas))
    kv_attend_stream_kernel(const __grid_constant__ KvAttendArgs k, const KvStreamPlan plan) {
  using S = Stream<Q, STORE, DP, NT>;
  using T = typename KvElem<Q>::type;
  extern __shared__ __align__(16) unsigned char smem[];
  typename S::Shared& sh = *reinterpret_cast<typename S::Shared*>(smem);
  const pf_kv_cache& c = k.cache;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  // Along x, the axis that has room for any number: the heads of a sequence side by side, because in most layouts
  // their rows of a token are, and run at the same time they meet in HBM's open pages.
  const uint32_t part = blockIdx.y, seq = blockIdx.x / c.heads, head = blockIdx.x - seq * c.heads;
  const int32_t group = int32_t(k.a.q_heads / c.heads);
  let_next_kernel_start();
  auto page_of = [&](int32_t j) { return plan.page_shift >= 0 ? uint32_t(j) >> plan.page_shift : uint32_t(j) / c.block_size; };

  const KvSeq s = kv_sequence(k, seq);
  const int32_t rows = s.n * group;
  // One tile, unless a sequence has more queries than the bound that chose this kernel.
  for (int32_t row0 = 0; row0 < rows; row0 += S::kRows) {
    const int32_t row_last = min(rows, row0 + S::kRows) - 1;
    const int32_t begin = kv_row_begin(k, s, row0 / group);
    const int32_t end = kv_row_end(k, s, row_last / group);
    const KvPart span = stream_part(plan, begin, end, part);
    const int32_t lo = span.lo, hi = span.hi;
    if constexpr (!CLUSTER) {
      if (part && lo >= end) continue;
    }

    const char* key_base = reinterpret_cast<const char*>(c.key.data);
    const char* value_base = reinterpret_cast<const char*>(c.value.data);

    // A batch's addresses and scales are made two batches ahead: its blocks are read first, a batch later the
    // scales, and they go to shared memory when the batch before is begun. No read is waited for at once.
    int32_t block = -1;
    Staged fresh;
    auto stage_blocks = [&](int32_t batch) {
      const int32_t j = lo + batch * kBatch + lane;
      block = j < hi ? kv_block(k, seq, page_of(j)) : -1;
    };
    auto stage_addresses = [&](int32_t batch) {
      fresh = Staged{-1, -1, 0.0f, 0.0f};
      if (block >= 0) {
        const int64_t b = block;
        const int32_t j = lo + batch * kBatch + lane;
        const int64_t at = uint32_t(j) - page_of(j) * c.block_size;
        fresh.key = (b * c.key.block_stride + at * c.key.token_stride + int64_t(head) * c.key.head_stride) * S::kElt;
        fresh.value = (b * c.value.block_stride + at * c.value.token_stride + int64_t(head) * c.value.head_stride) * S::kElt;
        if constexpr (S::kQuant) {
          fresh.key_scale = reinterpret_cast<const float*>(c.key.scale)[b * c.key.scale_block_stride + at * c.key.scale_token_stride +
                                                                        int64_t(head) * c.key.scale_head_stride];
          fresh.value_scale = reinterpret_cast<const float*>(
              c.value.scale)[b * c.value.scale_block_stride + at * c.value.scale_token_stride +
                             int64_t(head) * c.value.scale_head_stride];
        }
      }
    };
    const int32_t batches = (hi - lo + kBatch - 1) / kBatch;
    // This warp's batches: warp, warp + 4, ...; step i is half of its batch i / 2.
    const int32_t mine = warp < batches ? (batches - warp + kWarps - 1) / kWarps : 0;
    typename S::Step* ring = sh.ring[warp];
    const char* key_from = key_base + lane % S::kPieces * 16;
    const char* value_from = value_base + lane % S::kPieces * 16;
    int32_t whole = 0;  // this warp's batches up to here have all their rows: most steps are copied without a look
    auto stage_store = [&](int32_t n) {
      sh.staged[warp][n & 1][lane] = fresh;
      if (n == whole && __all_sync(0xffffffffu, fresh.key >= 0)) ++whole;
    };
    auto copy_step = [&](int32_t i) {
      if (i < 2 * mine) {
        typename S::Step& to = ring[i % kRing];
        const Staged* rows = &sh.staged[warp][i >> 1 & 1][(i & 1) * kStep];
        constexpr int kRowsAtOnce = 32 / S::kPieces;
        const int piece = lane % S::kPieces;
        const bool there = piece * S::kChunk < int(c.head_dim);
        int64_t key_at[kStep / kRowsAtOnce], value_at[kStep / kRowsAtOnce];
#pragma unroll
        for (int x = 0; x < kStep / kRowsAtOnce; ++x) {
          key_at[x] = rows[x * kRowsAtOnce + lane / S::kPieces].key;
          value_at[x] = rows[x * kRowsAtOnce + lane / S::kPieces].value;
        }
        if (i >> 1 < whole && int(c.head_dim) == DP) {
#pragma unroll
          for (int x = 0; x < kStep / kRowsAtOnce; ++x) {
            const int row = x * kRowsAtOnce + lane / S::kPieces;
            copy16(to.key[row] + S::key_piece(row, piece) * 16, key_from + key_at[x]);
            copy16(to.value[row] + S::value_piece(row, piece) * 16, value_from + value_at[x]);
          }
        } else {
#pragma unroll
          for (int x = 0; x < kStep / kRowsAtOnce; ++x) {
            const int row = x * kRowsAtOnce + lane / S::kPieces;
            copy16(to.key[row] + S::key_piece(row, piece) * 16, key_base + key_at[x] + piece * 16, key_base, there && key_at[x] >= 0);
            copy16(to.value[row] + S::value_piece(row, piece) * 16, value_base + value_at[x] + piece * 16, value_base, there && value_at[x] >= 0);
          }
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };

    if (mine) {
      stage_blocks(warp);
      stage_addresses(warp);
      stage_blocks(warp + kWarps);
      stage_store(0);
      __syncwarp();
    }
    copy_step(0);
    copy_step(1);
    if (mine) {
      stage_addresses(warp + kWarps);
      stage_blocks(warp + 2 * kWarps);
    }
    // This lane's query rows: g of each tile (as an operand), 2 t and 2 t + 1 (as results).
    uint32_t q[NT][S::kTiles][2];
    float f[NT][2];
    int32_t row_lo[NT][2], row_hi[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int32_t r = row0 + n * 8 + g;
      const bool on = r < rows;
      const int32_t i = on ? r / group : 0;
      const T* p = reinterpret_cast<const T*>(k.a.query.data) + int64_t(s.first + i) * k.a.query.token_stride +
                   int64_t(int32_t(head) * group + (on ? r - i * group : 0)) * k.a.query.head_stride;
      uint32_t raw[S::kTiles * 2];
#pragma unroll
      for (int j = 0; j < S::kKeyReads; ++j) {
        const int d = (t + 4 * j) * S::kChunk;
#pragma unroll
        for (int h = 0; h < S::kChunk / 8; ++h) {
          const uint4 v = on && d < int(c.head_dim) ? *reinterpret_cast<const uint4*>(p + d + h * 8) : make_uint4(0, 0, 0, 0);
          const int at = j * (S::kChunk / 2) + h * 4;
          raw[at] = v.x, raw[at + 1] = v.y, raw[at + 2] = v.z, raw[at + 3] = v.w;
        }
      }
      float unit = 1.0f;
      if constexpr (S::kQuant && Q == PF_DTYPE_BF16) {
        // The row's largest exponent, over its four lanes.
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < S::kTiles * 2; ++j) top = max(top, max(raw[j] & 0x7fffu, (raw[j] >> 16) & 0x7fffu));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // 2^(14 - e) brings it to [2^14, 2^15); both powers are kept within fp32's normal range.
        const int e = min(max(int(top >> 7) - 127, -100), 127);
        const float bring = __uint_as_float(uint32_t(127 + 14 - e) << 23);
        unit = __uint_as_float(uint32_t(127 - 14 + e) << 23);
#pragma unroll
        for (int j = 0; j < S::kTiles * 2; ++j) {
          raw[j] = pack2<false>(__uint_as_float(raw[j] << 16) * bring, __uint_as_float(raw[j] & 0xffff0000u) * bring);
        }
      }
#pragma unroll
      for (int j = 0; j < S::kTiles; ++j) q[n][j][0] = raw[2 * j], q[n][j][1] = raw[2 * j + 1];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        // Row 2 t + e of the tile has its unit in lane (2 t + e) * 4.
        f[n][e] = k.a.scale * kLog2e * __shfl_sync(0xffffffffu, unit, (2 * t + e) * 4);
        const int32_t rr = row0 + n * 8 + 2 * t + e;
        row_lo[n][e] = rr < rows ? kv_row_begin(k, s, rr / group) : 0;
        row_hi[n][e] = rr < rows ? kv_row_end(k, s, rr / group) : INT32_MAX;  // a row that is none: nothing is kept of it
      }
    }
    // Tokens that every row of the tile sees.
    const int32_t all_lo = kv_row_begin(k, s, row_last / group), all_hi = kv_row_end(k, s, row0 / group);

    float o[NT][S::kTiles][4];
    float m[NT][2], l[NT][2];
    float mv[NT][2];  // what the values go by: the largest score with its V scale's exponent (16 bits: m itself)
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < S::kTiles; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.0f;
      m[n][0] = m[n][1] = mv[n][0] = mv[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.0f;
    }

#pragma unroll 1
    for (int32_t i = 0; i < 2 * mine; ++i) {
      const int32_t batch = warp + (i >> 1) * kWarps, j0 = lo + batch * kBatch + (i & 1) * kStep;
      if ((i & 1) == 0) {
        // The next batch's addresses: its buffer's last readers are behind the end of the batch before.
        stage_store((i >> 1) + 1);
        stage_addresses(batch + 2 * kWarps);
        stage_blocks(batch + 3 * kWarps);
      }
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      __syncwarp();  // this step's rows are there for all lanes, and all are done with the one before
      copy_step(i + 2);
      const typename S::Step& now = ring[i % kRing];
      const Staged s0 = sh.staged[warp][i >> 1 & 1][(i & 1) * kStep + g], s1 = sh.staged[warp][i >> 1 & 1][(i & 1) * kStep + g + 8];

      const typename S::Scale v0 = S::split(s0.value_scale), v1 = S::split(s1.value_scale);
      // S^T: c0, c1 are token g's scores for the rows 2 t and 2 t + 1, c2, c3 token g + 8's.
      float x[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        x[n][0] = x[n][1] = x[n][2] = x[n][3] = 0.0f;
      }
#pragma unroll
      for (int j = 0; j < S::kKeyReads; ++j) {
        const uint4 r0 = *reinterpret_cast<const uint4*>(now.key[g] + S::key_piece(g, t + 4 * j) * 16);
        const uint4 r1 = *reinterpret_cast<const uint4*>(now.key[g + 8] + S::key_piece(g + 8, t + 4 * j) * 16);
        const uint32_t w0[4] = {r0.x, r0.y, r0.z, r0.w}, w1[4] = {r1.x, r1.y, r1.z, r1.w};
#pragma unroll
        for (int u = 0; u < S::kChunk / 4; ++u) {
          const int tile = j * (S::kChunk / 4) + u;
          uint32_t a0, a1, a2, a3;
          if constexpr (S::kQuant) {
            a0 = codes_to_half2<STORE, false>(w0[u]), a2 = codes_to_half2<STORE, true>(w0[u]);
            a1 = codes_to_half2<STORE, false>(w1[u]), a3 = codes_to_half2<STORE, true>(w1[u]);
          } else {
            a0 = w0[2 * u], a2 = w0[2 * u + 1], a1 = w1[2 * u], a3 = w1[2 * u + 1];
          }
#pragma unroll
          for (int n = 0; n < NT; ++n) mma<S::kBf16>(x[n], a0, a1, a2, a3, q[n][tile][0], q[n][tile][1]);
        }
      }

      const bool masked = j0 < all_lo || j0 + kStep > all_hi || __any_sync(0xffffffffu, s0.key < 0 || s1.key < 0);
      bool raise = false;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float y = x[n][e] * f[n][e & 1];
          if constexpr (S::kQuant) y *= e < 2 ? s0.key_scale : s1.key_scale;
          x[n][e] = y;
        }
      }
      if (masked) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int32_t j = j0 + g + (e < 2 ? 0 : 8);
            const bool on = (e < 2 ? s0.key : s1.key) >= 0 && j >= row_lo[n][e & 1] && j < row_hi[n][e & 1];
            x[n][e] = on ? x[n][e] : -INFINITY;
          }
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          raise = raise || fmaxf(x[n][e], x[n][e + 2]) > m[n][e] + (kRaise + S::kSumUp);
          if constexpr (S::kQuant) raise = raise || fmaxf(x[n][e] + v0.exponent, x[n][e + 2] + v1.exponent) > mv[n][e] + (kRaise + S::kUp);
        }
      }
      if (__any_sync(0xffffffffu, raise)) {
        // What weights go by becomes the maximum less the lift; returns what that makes of earlier ones.
        auto raised = [](float& old, float top, float up) {
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
          top = fmaxf(top - up, old);
          const float keep = top == -INFINITY ? 0.0f : fast_exp2(old - top);
          old = top;
          return keep;
        };
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float keep[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            keep[e] = raised(m[n][e], fmaxf(x[n][e], x[n][e + 2]), S::kSumUp);
            l[n][e] *= keep[e];
            if constexpr (S::kQuant) keep[e] = raised(mv[n][e], fmaxf(x[n][e] + v0.exponent, x[n][e + 2] + v1.exponent), S::kUp);
          }
#pragma unroll
          for (int y = 0; y < S::kTiles; ++y) {
            o[n][y][0] *= keep[0], o[n][y][1] *= keep[1], o[n][y][2] *= keep[0], o[n][y][3] *= keep[1];
          }
        }
      }
      uint32_t p[NT][2], rest[NT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float base = m[n][e & 1] == -INFINITY ? 0.0f : m[n][e & 1];
          w[e] = fast_exp2(x[n][e] - base);
          l[n][e & 1] += w[e];
          if constexpr (S::kQuant) {
            const typename S::Scale& v = e < 2 ? v0 : v1;
            const float by = mv[n][e & 1] == -INFINITY ? 0.0f : mv[n][e & 1];
            w[e] = fast_exp2(x[n][e] + v.exponent - by) * v.rest;
          }
        }
        const uint32_t first = pack2<S::kBf16>(w[0], w[1]), second = pack2<S::kBf16>(w[2], w[3]);
        p[n][0] = transpose_8x8(first);
        p[n][1] = transpose_8x8(second);
        if constexpr (S::kExact) {
          const float2 a = unpack2<S::kBf16>(first), b = unpack2<S::kBf16>(second);
          rest[n][0] = transpose_8x8(pack2<S::kBf16>(w[0] - a.x, w[1] - a.y));
          rest[n][1] = transpose_8x8(pack2<S::kBf16>(w[2] - b.x, w[3] - b.y));
        }
      }
      // V^T: the tokens 2 t, 2 t + 1, 2 t + 8, 2 t + 9 of this lane's values.
#pragma unroll
      for (int j = 0; j < S::kValueReads; ++j) {
        uint32_t w[4][S::kValueRead / 4];
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const int row = 2 * t + (h & 1) + 8 * (h >> 1);
          if constexpr (S::kValueRead == 16) {
            const uint4 r = *reinterpret_cast<const uint4*>(now.value[row] + S::value_piece(row, g + 8 * j) * 16);
            w[h][0] = r.x, w[h][1] = r.y, w[h][2] = r.z, w[h][3] = r.w;
          } else {
            const uint2 r = *reinterpret_cast<const uint2*>(now.value[row] + S::value_piece(row, g >> 1) * 16 + (g & 1) * 8);
            w[h][0] = r.x, w[h][1] = r.y;
          }
        }
#pragma unroll
        for (int u = 0; u < S::kValueRead / 4; ++u) {
          if constexpr (S::kQuant) {
#pragma unroll
            for (int z = 0; z < 2; ++z) {
              const uint32_t sel = z ? 0x7362 : 0x5140;
              const uint32_t lo2 = __byte_perm(w[0][u], w[1][u], sel), hi2 = __byte_perm(w[2][u], w[3][u], sel);
              const uint32_t a0 = codes_to_half2<STORE, false>(lo2), a1 = codes_to_half2<STORE, true>(lo2);
              const uint32_t a2 = codes_to_half2<STORE, false>(hi2), a3 = codes_to_half2<STORE, true>(hi2);
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                mma<S::kBf16>(o[n][2 * u + z], a0, a1, a2, a3, p[n][0], p[n][1]);
                if constexpr (S::kExact) mma<S::kBf16>(o[n][2 * u + z], a0, a1, a2, a3, rest[n][0], rest[n][1]);
              }
            }
          } else {
            const uint32_t a0 = __byte_perm(w[0][u], w[1][u], 0x5410), a1 = __byte_perm(w[0][u], w[1][u], 0x7632);
            const uint32_t a2 = __byte_perm(w[2][u], w[3][u], 0x5410), a3 = __byte_perm(w[2][u], w[3][u], 0x7632);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              mma<S::kBf16>(o[n][4 * j + u], a0, a1, a2, a3, p[n][0], p[n][1]);
              if constexpr (S::kExact) mma<S::kBf16>(o[n][4 * j + u], a0, a1, a2, a3, rest[n][0], rest[n][1]);
            }
          }
        }
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncwarp();  // the ring is free for the sums

    // The warps' shares, then the part's: [row][value] in shared memory.
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float sum = l[n][e];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        if (g == 0) {
          sh.m[warp][n * 8 + 2 * t + e] = m[n][e];
          sh.mv[warp][n * 8 + 2 * t + e] = S::kQuant ? mv[n][e] : m[n][e];
          sh.l[warp][n * 8 + 2 * t + e] = sum;
        }
      }
#pragma unroll
      for (int i = 0; i < S::kTiles; ++i) {
        const int d = S::kQuant ? g * (DP / 8) + 2 * i : (i / 4 * 8 + g) * 8 + i % 4 * 2;
#pragma unroll
        for (int e = 0; e < 4; ++e) sh.o[warp][(n * 8 + 2 * t + (e & 1)) * DP + d + (e >> 1)] = o[n][i][e];
      }
    }
    if (threadIdx.x < S::kRows) sh.bad[threadIdx.x] = 0;
    __syncthreads();

    const int32_t used = stream_parts(plan, end - begin);
    // Rows of one tile see different tokens: an infinity behind one row's end may have met its weight of zero.
    const bool uneven = max(lo, all_lo) > lo || min(hi, all_hi) < hi;
    // Sums of weights are in units of 2^top, of weights times values in units of 2^top_v.
    auto finish = [&](int32_t r, uint32_t d, float top, float sum, float top_v, float value) {
      const int32_t i = r / group, qh = int32_t(head) * group + r - i * group;
      const int64_t token = int64_t(s.first) + i, id = token * k.a.q_heads + qh;
      if (CLUSTER || used == 1) {
        const float y = sum == 0.0f ? 0.0f : S::kQuant ? in_units(value / sum, top_v - top) : value / sum;
        if (d < c.head_dim) {
          reinterpret_cast<T*>(k.a.out.data)[token * k.a.out.token_stride + int64_t(qh) * k.a.out.head_stride + d] = kv_from_float<Q>(y);
        }
        if (d == 0 && k.a.lse) {
          reinterpret_cast<float*>(k.a.lse)[id] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * kLn2;
        }
      } else {
        float* ws = reinterpret_cast<float*>(k.a.workspace) + (id * plan.parts + part) * (DP + 4);
        ws[4 + d] = value;
        if (d == 0) ws[0] = top, ws[1] = sum, ws[2] = top_v;
      }
    };
    // What the CTA has of a row: for its cluster into the place of the first warp's share, or done with.
    auto leave = [&](int32_t row, uint32_t d, float top, float sum, float top_v, float value) {
      if constexpr (CLUSTER) {
        sh.o[0][row * DP + int32_t(d)] = value;
        if (d == 0) sh.part_m[row] = top, sh.part_l[row] = sum, sh.part_mv[row] = top_v;
      } else {
        finish(row0 + row, d, top, sum, top_v, value);
      }
    };
    for (int32_t e = threadIdx.x; e < S::kRows * DP; e += kThreads) {
      const int32_t row = e / DP;
      const uint32_t d = uint32_t(e % DP);
      if (row0 + row >= rows) break;
      float top = sh.m[0][row], top_v = sh.mv[0][row];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) top = fmaxf(top, sh.m[w][row]), top_v = fmaxf(top_v, sh.mv[w][row]);
      float sum = 0.0f, value = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float keep = top == -INFINITY ? 1.0f : exp2f(sh.m[w][row] - top);
        const float keep_v = !S::kQuant ? keep : top_v == -INFINITY ? 1.0f : exp2f(sh.mv[w][row] - top_v);
        sum += sh.l[w][row] * keep;
        value += sh.o[w][row * DP + int32_t(d)] * keep_v;
      }
      if (uneven && sum == sum && !isfinite(value)) {
        sh.bad[row] = 1;
      } else {
        leave(row, d, top, sum, top_v, value);
      }
    }
    if (uneven) {
      __syncthreads();
      for (int row = warp; row < S::kRows; row += kWarps) {
        if (!sh.bad[row]) continue;
        const int32_t r = row0 + row, i = r / group;
        float top, sum;
        float4 v;
        attend_row_exactly<Q, STORE>(k, seq, int64_t(s.first) + i, head * group + uint32_t(r - i * group), head,
                                     max(lo, kv_row_begin(k, s, i)), min(hi, kv_row_end(k, s, i)), top, sum, v, nullptr);
        if (lane * 4 < DP) {
          leave(row, lane * 4, top, sum, top, v.x);
          leave(row, lane * 4 + 1, top, sum, top, v.y);
          leave(row, lane * 4 + 2, top, sum, top, v.z);
          leave(row, lane * 4 + 3, top, sum, top, v.w);
        }
      }
    }
    if constexpr (CLUSTER) {
      // Joins the cluster's parts: weights 2^(m_part - max) over their sums, a share of the rows' values for each CTA.
      cluster_meets();
      for (int32_t e = int32_t(part) * kThreads + int32_t(threadIdx.x); e < S::kRows * DP; e += int32_t(plan.parts) * kThreads) {
        const int32_t row = e / DP;
        if (row0 + row >= rows) break;
        float m_of[kStreamMaxCluster], l_of[kStreamMaxCluster], v_of[kStreamMaxCluster], o_of[kStreamMaxCluster];
        float top = -INFINITY, top_v = -INFINITY;
#pragma unroll
        for (int p = 0; p < int(kStreamMaxCluster); ++p) {
          m_of[p] = p < used ? load_of(&sh.part_m[row], p) : -INFINITY;
          l_of[p] = p < used ? load_of(&sh.part_l[row], p) : 0.0f;
          v_of[p] = S::kQuant && p < used ? load_of(&sh.part_mv[row], p) : -INFINITY;
          o_of[p] = p < used ? load_of(&sh.o[0][e], p) : 0.0f;
        }
#pragma unroll
        for (int p = 0; p < int(kStreamMaxCluster); ++p) top = fmaxf(top, m_of[p]), top_v = fmaxf(top_v, v_of[p]);
        const float base = top == -INFINITY ? 0.0f : top, base_v = top_v == -INFINITY ? 0.0f : top_v;
        float sum = 0.0f, value = 0.0f;
#pragma unroll
        for (int p = 0; p < int(kStreamMaxCluster); ++p) {
          const float by = exp2f(m_of[p] - base);
          sum += l_of[p] * by;
          value += o_of[p] * (S::kQuant ? exp2f(v_of[p] - base_v) : by);
        }
        finish(row0 + row, uint32_t(e % DP), top, sum, top_v, value);
      }
      cluster_meets();  // shared memory is read by the others until here
    }
    __syncthreads();  // shared memory is used again by the next tile
  }
}

// Joins the parts of the rows that have several: weights 2^(m_part - max) over the
// parts' sums. A block takes a row, its warps parts in turn, so that as many loads
// are in flight as a row has parts; a lane has 4 values.
constexpr int kJoinWarps = 8;
template <uint32_t Q, int DP>
__global__ void __launch_bounds__(kJoinWarps * 32) kv_join_stream_kernel(const __grid_constant__ KvAttendArgs k, const KvStreamPlan plan) {
  using T = typename KvElem<Q>::type;
  __shared__ float4 values[kJoinWarps][32];
  __shared__ float sums[kJoinWarps], tops[kJoinWarps], tops_v[kJoinWarps];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint64_t id = blockIdx.x;
  const uint32_t token = uint32_t(id / k.a.q_heads), qh = uint32_t(id % k.a.q_heads);
  const uint32_t seq = kv_find_seq(reinterpret_cast<const int32_t*>(k.a.q_start), k.a.n_seqs, token);
  KvSeq s{0, 0, 0, 0};
  if (seq < k.a.n_seqs) s = kv_sequence(k, seq);
  const int32_t group = int32_t(k.a.q_heads / k.cache.heads), rows = s.n * group;
  const int32_t r = (int32_t(token) - s.first) * group + int32_t(qh) % group;
  const int32_t tile_rows = 8 * int32_t(plan.row_tiles);
  const int32_t row0 = r / tile_rows * tile_rows, row_last = min(rows, row0 + tile_rows) - 1;
  const int32_t used = stream_parts(plan, kv_row_end(k, s, row_last / group) - kv_row_begin(k, s, row0 / group));
  // Every block waits, those without work too: this kernel's end is what the next in the stream goes by.
  wait_for_previous_kernel();
  if (seq == k.a.n_seqs || r >= rows || used == 1) return;
  const float* ws = reinterpret_cast<const float*>(k.a.workspace) + id * plan.parts * (DP + 4);
  // The warp's own running maxima, then the block's.
  float top = -INFINITY, top_v = -INFINITY, sum = 0.0f;
  float4 o = make_float4(0, 0, 0, 0);
  const bool mine = lane * 4 < DP;
#pragma unroll 1
  for (int32_t p0 = warp; p0 < used; p0 += 4 * kJoinWarps) {
    float m[4], l[4], mv[4];
    float4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int32_t p = p0 + u * kJoinWarps;
      const float* w = ws + int64_t(p) * (DP + 4);
      m[u] = p < used ? w[0] : -INFINITY;
      l[u] = p < used ? w[1] : 0.0f;
      mv[u] = p < used ? w[2] : -INFINITY;
      v[u] = p < used && mine ? *reinterpret_cast<const float4*>(w + 4 + lane * 4) : make_float4(0, 0, 0, 0);
    }
    const float now = fmaxf(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])), top);
    const float now_v = fmaxf(fmaxf(fmaxf(mv[0], mv[1]), fmaxf(mv[2], mv[3])), top_v);
    const float base = now == -INFINITY ? 0.0f : now, base_v = now_v == -INFINITY ? 0.0f : now_v;
    const float keep = exp2f(top_v - base_v);
    sum *= exp2f(top - base);
    o.x *= keep, o.y *= keep, o.z *= keep, o.w *= keep;
    top = now, top_v = now_v;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float by = exp2f(mv[u] - base_v);
      sum += l[u] * exp2f(m[u] - base);
      o.x += v[u].x * by, o.y += v[u].y * by, o.z += v[u].z * by, o.w += v[u].w * by;
    }
  }
  values[warp][lane] = o;
  if (lane == 0) sums[warp] = sum, tops[warp] = top, tops_v[warp] = top_v;
  __syncthreads();
  if (warp) return;
  for (int w = 0; w < kJoinWarps; ++w) top = fmaxf(top, tops[w]), top_v = fmaxf(top_v, tops_v[w]);
  const float base = top == -INFINITY ? 0.0f : top, base_v = top_v == -INFINITY ? 0.0f : top_v;
  sum = 0.0f, o = make_float4(0, 0, 0, 0);
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w) {
    const float by = exp2f(tops_v[w] - base_v);
    const float4 v = values[w][lane];
    sum += sums[w] * exp2f(tops[w] - base);
    o.x += v.x * by, o.y += v.y * by, o.z += v.z * by, o.w += v.w * by;
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  if (lane * 4 < int(k.cache.head_dim)) {
    KvPack<T, 4> y;
    y.v[0] = kv_from_float<Q>(in_units(o.x * inv, base_v - base));
    y.v[1] = kv_from_float<Q>(in_units(o.y * inv, base_v - base));
    y.v[2] = kv_from_float<Q>(in_units(o.z * inv, base_v - base));
    y.v[3] = kv_from_float<Q>(in_units(o.w * inv, base_v - base));
    *reinterpret_cast<KvPack<T, 4>*>(reinterpret_cast<T*>(k.a.out.data) + int64_t(token) * k.a.out.token_stride +
                                     int64_t(qh) * k.a.out.head_stride + lane * 4) = y;
  }
  if (lane == 0 && k.a.lse) reinterpret_cast<float*>(k.a.lse)[id] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * kLn2;
}

uint32_t most_queries(const KvAttendArgs& k) {
  const uint64_t n = std::max<uint64_t>(1, k.a.n_tokens);
  return static_cast<uint32_t>(k.a.max_q ? std::min<uint64_t>(k.a.max_q, n) : n);
}

// Stream<>::kCtas for a call.
uint32_t ctas_per_sm(const KvAttendArgs& k, const KvStreamPlan& p) {
  const uint32_t row = (k.cache.head_dim <= 64 ? 64 : 128) * kv_dtype_bytes(k.cache.dtype);
  return row == 256 ? 2 : p.row_tiles == 1 ? 4 : 2;
}

template <uint32_t Q, uint32_t STORE, int DP, int NT, bool CLUSTER>
cudaError_t launch_as(const KvAttendArgs& k, const KvStreamPlan& p, cudaStream_t stream) {
  using S = Stream<Q, STORE, DP, NT>;
  const auto kernel = kv_attend_stream_kernel<Q, STORE, DP, NT, CLUSTER>;
  const int shm = int(sizeof(typename S::Shared));
  if (shm > 48 * 1024) {
    const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, shm);
    if (err != cudaSuccess) return err;
  }
  if constexpr (CLUSTER) {
    cudaLaunchAttribute cluster;
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = 1, cluster.val.clusterDim.y = p.parts, cluster.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(k.a.n_seqs * k.cache.heads, p.parts);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = shm;
    cfg.stream = stream;
    cfg.attrs = &cluster;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, k, p);
  }
  kernel<<<dim3(k.a.n_seqs * k.cache.heads, p.parts), kThreads, shm, stream>>>(k, p);
  if (p.parts == 1) return cudaGetLastError();
  cudaError_t err = cudaGetLastError();
  if (err != cudaSuccess) return err;
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<uint32_t>(k.a.n_tokens * k.a.q_heads));
  cfg.blockDim = dim3(kJoinWarps * 32);
  cfg.stream = stream;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kv_join_stream_kernel<Q, DP>, k, p);
}

template <uint32_t Q, uint32_t STORE>
cudaError_t launch_dims(const KvAttendArgs& k, const KvStreamPlan& p, cudaStream_t stream) {
  const bool c = p.clusters;
  if (k.cache.head_dim <= 64) {
    if (p.row_tiles == 1) return c ? launch_as<Q, STORE, 64, 1, true>(k, p, stream) : launch_as<Q, STORE, 64, 1, false>(k, p, stream);
    return c ? launch_as<Q, STORE, 64, 2, true>(k, p, stream) : launch_as<Q, STORE, 64, 2, false>(k, p, stream);
  }
  if (p.row_tiles == 1) return c ? launch_as<Q, STORE, 128, 1, true>(k, p, stream) : launch_as<Q, STORE, 128, 1, false>(k, p, stream);
  return c ? launch_as<Q, STORE, 128, 2, true>(k, p, stream) : launch_as<Q, STORE, 128, 2, false>(k, p, stream);
}

template <uint32_t Q>
cudaError_t launch_store(const KvAttendArgs& k, const KvStreamPlan& p, cudaStream_t stream) {
  switch (k.cache.dtype) {
    case PF_DTYPE_E4M3: return launch_dims<Q, PF_DTYPE_E4M3>(k, p, stream);
    case PF_DTYPE_INT8: return launch_dims<Q, PF_DTYPE_INT8>(k, p, stream);
    default: return launch_dims<Q, Q>(k, p, stream);
  }
}

}  // namespace

KvStreamPlan stream_plan(const KvAttendArgs& k, int num_sms) {
  KvStreamPlan p;
  p.page_shift = page_shift(k.cache);
  const uint32_t rows = most_queries(k) * (k.a.q_heads / k.cache.heads);
  p.row_tiles = rows <= 8 ? 1 : 2;
  uint64_t longest = uint64_t(k.a.max_blocks) * k.cache.block_size;
  if (k.a.max_kv) longest = std::min<uint64_t>(longest, k.a.max_kv);
  if (k.a.window) longest = std::min<uint64_t>(longest, uint64_t(k.a.window) + most_queries(k));
  longest = std::max<uint64_t>(longest, 1);
  // Parts of equal length: the CTAs run in rounds of as many as fit, each round as long as a part and its start and
  // end (queries, addresses, joining: about 384 tokens' time). Few sequences: one round, whose parts are as short as
  // that leaves them. Many: sequences are rarely equally long, so among splits that are within a tenth of the best
  // the finest is taken, which evens them out (64 sequences of 1K to 16K tokens, at 1,965 MHz: 286 us in one round, 221
  // in seven).
  const uint64_t items = std::max<uint64_t>(1, uint64_t(k.a.n_seqs) * k.cache.heads);
  const uint64_t slots = uint64_t(num_sms) * ctas_per_sm(k, p);
  const uint64_t units = (longest + kStreamMinPart - 1) / kStreamMinPart;  // shortest parts
  auto cost = [&](uint64_t per) {
    const uint64_t parts = (units + per - 1) / per;
    return (items * parts + slots - 1) / slots * (per + 3);
  };
  uint64_t best = UINT64_MAX;
  const uint64_t least = (units + kStreamMaxParts - 1) / kStreamMaxParts;
  for (uint64_t per = least; per <= units; per += (per + 15) / 16) best = std::min(best, cost(per));
  uint64_t per = least;
  while (per < units && cost(per) * 10 > best * 11) per += (per + 15) / 16;
  per = std::min(per, units);
  p.part_tokens = static_cast<int32_t>(std::min<uint64_t>(per * kStreamMinPart, 1u << 30));
  p.parts = static_cast<uint32_t>((longest + p.part_tokens - 1) / p.part_tokens);
  // Up to eight parts that all run at once are a cluster and joined by it, without a second launch (one sequence of
  // 1,000 tokens: 7.1 us instead of 7.7, eight of 4,000: 21.8 instead of 22.9). In several rounds a cluster waits for
  // room for all of its parts (16 sequences of 100 to 8,000 tokens: 70 us instead of 50).
  p.clusters = p.parts > 1 && p.parts <= kStreamMaxCluster && items * p.parts <= slots;
  return p;
}

uint64_t stream_workspace(const KvAttendArgs& k, const KvStreamPlan& p) {
  if (p.parts == 1 || p.clusters) return 0;
  const uint64_t dp = k.cache.head_dim <= 64 ? 64 : 128;
  return k.a.n_tokens * k.a.q_heads * p.parts * (dp + 4) * sizeof(float);
}

cudaError_t launch_attend_stream(const KvAttendArgs& k, const KvStreamPlan& p, cudaStream_t stream) {
  return k.a.dtype == PF_DTYPE_BF16 ? launch_store<PF_DTYPE_BF16>(k, p, stream) : launch_store<PF_DTYPE_FP16>(k, p, stream);
}

}  // namespace pf
