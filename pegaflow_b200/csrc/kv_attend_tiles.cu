// Attention of chunks of new tokens: the products are matrix products, and the
// tensor cores and the exponentials bound it.
//
// An item (kv_attend_tiles.h) is 256 query rows (queries times the heads of a
// group) of one sequence and KV head: two tiles of 128, so that the tensor cores
// work for one while the other's softmax runs. For each 128 keys and each tile
//   S = Q K^T            tcgen05.mma, Q and K in shared memory, S in TMEM
//   P = 2^(S f - m)      a thread for each row, P in TMEM over S
//   O += P V             tcgen05.mma, P in TMEM, V in shared memory, O in TMEM
// and at the end O / sum(P). 128 x 128 x 128 takes the tensor cores 512 clocks, so
// 256 x 128 keys take 2,048; their 32,768 exponentials take the special-function
// units (16 a clock) 2,048 too. m follows the row's maximum only when it rises by
// 2^8 (kRaise): then, rarely, O is rescaled in TMEM by the threads of that tile.
// Measured for 2,048 tokens, 32 heads on 8 of 128, in calls without a pause, whose
// clocks the power limit sets: after 10,240 in bf16 405 us (933 TFLOP/s at 1,750 MHz),
// after 32,768 over e4m3 1.46 ms (775 at 1,890 MHz). Twenty calls, at 1,965 MHz: 361 us
// and 1.41 ms. Times of variants below are of such short runs.
//
// P has the type of V: over bf16 its rounding to 8 bits is seen in the result (off by
// 2.3e-3, 1.7e-3 being the result's own rounding; a second product for what it leaves,
// as the streaming kernel has, would be half as much again of the tensor cores' work).
// In fp16 it is taken 2^7 up (kLift), so that small weights keep their bits longer.
//
// Warps 0-3 and 4-7: the softmax of the two halves. Three or five: load Q, K and
// V. The last: issues the products. mbarriers order them; every wait is bounded, and
// one that runs out ends the call with a status bit and no hang.
//
// A tile of 128 16-bit keys comes by TMA, a box of each block, where all 128 are
// seen and the block size allows it (8 to 128 tokens, or whole tiles); else a row
// at a time by 16-byte copies, with zeros for tokens that are not there: any
// block size works, and nothing behind a sequence's end is ever multiplied.
//
// 8-bit codes are copied into their stage as they are and become fp16, which holds
// all of e4m3 and int8 exactly, there. K's scales stay in fp32 and multiply the
// scores. V's, divided by a power of two that follows the largest, multiply V there
// where the result is bf16 (two roundings of 2^-11 beside its own of 2^-8), and the
// fp32 weights where it is fp16 (2.9e-4 off in all, 4.0e-4 the other way, 2.1e-4
// being its own rounding; 1.51 ms instead of 1.39 for 2,048 tokens after 32,768). Rows
// that see V scales 2^14 apart are made again where it shows.
// As in the streaming kernel a bf16 query is brought into fp16's range by a power
// of two for each row.
#include <cuda.h>

#include <algorithm>
#include <type_traits>

#include "kv_attend.cuh"
#include "kv_attend_tiles.h"

namespace pf {
namespace {

constexpr int kSoftmaxWarps = 8;
constexpr int kInfos = 4;
constexpr long long kWaitClocks = 2000000000ll;  // of the SM, for each wait: a second or a little more

// What the softmax needs to know of a tile of keys.
struct alignas(16) KeyInfo {
  float key_scale[kTileKeys];
  float value_scale[kTileKeys];  // divided by a power of two that keeps weights in fp16's range
  int64_t key_at[kTileKeys];  // byte offsets of the rows, -1 for a token that is not seen
  int64_t value_at[kTileKeys];
  uint32_t seen[kTileKeys / 32];
  uint32_t v_exp;             // that power's exponent field; it never falls within an item
  uint32_t boxed;             // came by TMA
  float top_scale;            // the largest of value_scale
  float low_scale;            // and the smallest, of tokens that are there
  uint32_t far;               // one of them is below kFarScale, and of more than zeros
};

// A V scale, or a weight times it, below this share of the unit is no normal fp16 number:
// it is off by up to 2^-25, and so a value of 448 codes by 2^-16.2.
constexpr float kFarScale = 1.0f / 16384;
// Rows that have such and whose largest value is below this (for each unit of their weights, or for each token where
// the weights are scaled) are made again: what is left is off by 2^-11 of that value at most.
constexpr float kSmallRow = 1.0f / 32;

struct Watch {
  int failed;  // a wait gave up
  int alive;   // counts up while rows are made again
};

struct KvBoxMaps {
  CUtensorMap key;
  CUtensorMap value;
};

template <uint32_t Q, uint32_t STORE, int DP>
struct Tiles {
  static constexpr bool kQuant = STORE == PF_DTYPE_E4M3 || STORE == PF_DTYPE_INT8;
  static constexpr bool kBf16 = !kQuant && Q == PF_DTYPE_BF16;
  // Where V's scales go: into V as it becomes fp16, by the loading warps, which have time for that; a result of fp16
  // is too fine for the rounding that this costs, and takes them with the weights.
  static constexpr bool kScaledValues = kQuant && Q == PF_DTYPE_BF16;
  static constexpr int kStages = 4;  // two tiles' K and V
  // 12 warps may have 168 registers, 13 to 16 have 128. 16 bits: 12 warps, copying takes few. 8 bits: expanding codes
  // takes more, and 14 warps are best (2,048 tokens after 32,768: 1.49 ms with four loading, 1.39 with five, 1.45 with
  // six or seven, which take issue slots from the softmax), but where the softmax has 128 scaled weights in hand:
  // 128 registers spill there (1.89 ms; with 168 1.51).
  static constexpr int kLoadWarps = kQuant && (kScaledValues || DP == 64) ? 5 : 3;
  static constexpr int kLoadThreads = kLoadWarps * 32;
  static constexpr int kMmaWarp = kSoftmaxWarps + kLoadWarps;
  static constexpr int kThreads = (kMmaWarp + 1) * 32;
  static constexpr int kTileBytes = 128 * DP * 2;  // 128 rows of Q, K or V: DP / 64 blocks of [128][128 bytes]
  struct Shared {
    unsigned char q[2][kTileBytes];
    unsigned char kv[kStages][kTileBytes];
    KeyInfo info[kInfos];
    float q_unit[2][kTileRows];  // by the item's parity
    int64_t q_at[kTileRows];
    uint32_t warp_max[2][kTileKeys / 32];  // of V's scales, by the tile's parity
    uint32_t warp_min[2][kTileKeys / 32];
    uint64_t q_full, q_empty;
    uint64_t kv_full[kStages], kv_empty[kStages];
    uint64_t info_full[kInfos], info_empty[kInfos];
    uint64_t s_full[2], p_full[2], o_full[2], o_free[2], done;
    uint32_t tmem;
    Watch watch;
    Watch stuck[2];  // waits for copies and products in flight that gave up as well
  };
  // TMEM columns (all 512 are allocated, so they begin at 0).
  static constexpr uint32_t kS = 0, kO = 256;
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void bar_init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool bar_try(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
      : "=r"(done)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return done;
}
// Whether the phase of `parity` completed, within kWaitClocks and before another
// wait of this CTA gave up. Rows made again token by token take their time: as
// long as they get on, the clock starts anew. Out of line: the kernel waits in
// some twenty places, and with this in each it is slower (391 us against 358 for
// 2,048 tokens after 10,240: the code that runs all the time no longer fits).
__device__ __noinline__ bool bar_wait_longer(uint64_t* bar, uint32_t parity, Watch* w) {
  volatile int* failed = &w->failed;
  volatile int* alive = &w->alive;
  if (*failed) return false;
  long long t0 = clock64();
  int last = *alive;
  for (;;) {
#pragma unroll 1
    for (int i = 0; i < 64; ++i) {
      if (bar_try(bar, parity)) return true;
    }
    if (*failed) return false;
    const int now = *alive;
    if (now != last) {
      last = now;
      t0 = clock64();
    } else if (clock64() - t0 > kWaitClocks) {
      *failed = 1;
      return false;
    }
  }
}

__device__ __forceinline__ bool bar_wait(uint64_t* bar, uint32_t parity, Watch* watch) {
  return bar_try(bar, parity) || bar_wait_longer(bar, parity, watch);
}

// The same for a warp, as one.
__device__ __forceinline__ bool bar_wait_warp(uint64_t* bar, uint32_t parity, Watch* watch) {
  return __all_sync(0xffffffffu, bar_wait(bar, parity, watch));
}
// Meets the other loading threads; whether all of them say yes. A warp arrives as
// one (.aligned), and its lanes may come from waits that they left at different
// times.
template <int THREADS>
__device__ __forceinline__ bool loaders_agree(bool ok) {
  uint32_t all;
  __syncwarp();
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n barrier.cta.red.and.pred.aligned q, 1, %2, p;\n selp.u32 %0, 1, 0, q;\n}"
      : "=r"(all)
      : "r"(uint32_t(ok)), "n"(THREADS)
      : "memory");
  return all;
}

__device__ __forceinline__ void bar_arrive_expecting(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
// A box of one block's rows for one head: 64 values wide (zeros past head_dim).
__device__ __forceinline__ void load_box(uint32_t to, const CUtensorMap* map, int d, int token, int head, int block, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(to),
      "l"(map), "r"(d), "r"(token), "r"(head), "r"(block), "r"(smem_u32(bar))
      : "memory");
}

__device__ __forceinline__ void fence_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tmem_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// One thread of a converged warp, always the same. Products are issued under it:
// their operands live in uniform registers, and only here does the compiler know
// that one thread's values are the warp's (issued by `lane == 0` each of them
// took 100 clocks).
__device__ __forceinline__ bool elected() {
  uint32_t yes;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(yes));
  return yes;
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// D[tmem] (+)= A[smem] B[smem]
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(uint32_t(add))
      : "memory");
}
// D[tmem] (+)= A[tmem] B[smem]
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(uint32_t(add))
      : "memory");
}

// Shared-memory operand in blocks of [rows][128 bytes], 16-byte pieces swizzled by
// the row's low three bits: groups of 8 rows are 1,024 bytes apart. `across` is
// the distance of the blocks where the instruction spans several (V: its N side).
__device__ __forceinline__ uint64_t operand(uint32_t address, uint32_t across) {
  return uint64_t((address & 0x3ffff) >> 4) | uint64_t(across >> 4) << 16 | uint64_t(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61;
}

// 128 rows x n columns, fp32 result; b_rows: B is stored with its N side contiguous.
__host__ __device__ constexpr uint32_t instruction(bool bf16, uint32_t n, bool b_rows) {
  return 1u << 4 | (bf16 ? 1u << 7 | 1u << 10 : 0u) | (b_rows ? 1u << 16 : 0u) | (n >> 3) << 17 | (128u >> 4) << 24;
}

#define PF_R4(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3])
#define PF_I4(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3])
__device__ __forceinline__ void tmem_load32(uint32_t (&r)[32], uint32_t at) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,"
      "%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : PF_R4(r, 0), PF_R4(r, 4), PF_R4(r, 8), PF_R4(r, 12), PF_R4(r, 16), PF_R4(r, 20), PF_R4(r, 24), PF_R4(r, 28)
      : "r"(at));
}
__device__ __forceinline__ void tmem_store32(uint32_t at, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::PF_I4(r, 0),
      PF_I4(r, 4), PF_I4(r, 8), PF_I4(r, 12), PF_I4(r, 16), PF_I4(r, 20), PF_I4(r, 24), PF_I4(r, 28), "r"(at)
      : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t at, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::PF_I4(r, 0),
      PF_I4(r, 4), PF_I4(r, 8), PF_I4(r, 12), "r"(at)
      : "memory");
}
// The registers are operands, so that nothing reads them before the wait.
#define PF_RW4(r, i) "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3])
__device__ __forceinline__ void tmem_wait_load(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : PF_RW4(r, 0), PF_RW4(r, 4), PF_RW4(r, 8), PF_RW4(r, 12), PF_RW4(r, 16), PF_RW4(r, 20), PF_RW4(r, 24), PF_RW4(r, 28)
               :
               : "memory");
}
__device__ __forceinline__ void tmem_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <bool BF16>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
  uint32_t r;
  if constexpr (BF16) {
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  } else {
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  }
  return r;
}

// Four codes as four fp16 values.
template <uint32_t STORE>
__device__ __forceinline__ uint2 codes_to_half4(uint32_t x) {
  uint2 r;
  if constexpr (STORE == PF_DTYPE_E4M3) {
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r.x) : "h"(uint16_t(x)));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r.y) : "h"(uint16_t(x >> 16)));
  } else {
    // 1024 + (code + 128) as fp16 bits, then minus 1152: all exact.
    x ^= 0x80808080u;
    const uint32_t lo = __byte_perm(x, 0x64646464u, 0x4140), hi = __byte_perm(x, 0x64646464u, 0x4342);
    const __half2 off = __floats2half2_rn(1152.0f, 1152.0f);
    const __half2 a = __hsub2(*reinterpret_cast<const __half2*>(&lo), off), b = __hsub2(*reinterpret_cast<const __half2*>(&hi), off);
    r.x = *reinterpret_cast<const uint32_t*>(&a), r.y = *reinterpret_cast<const uint32_t*>(&b);
  }
  return r;
}

// Four codes times a scale, in fp16.
__device__ __forceinline__ uint2 times_half4(uint2 x, __half2 by) {
  const __half2 a = __hmul2(*reinterpret_cast<const __half2*>(&x.x), by), b = __hmul2(*reinterpret_cast<const __half2*>(&x.y), by);
  return make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}

// One CTA's walk along its span: every role does it for itself.
struct Item {
  KvSeq s;
  uint32_t seq;
  int32_t head;
  int32_t row0;    // first row of the tile within the sequence's
  int32_t rows;    // rows of the tile
  int32_t first;   // tokens that its rows see
  int32_t end;
  int32_t begin;   // where its first tile of keys begins
  int32_t units;   // of the whole item
  int32_t unit0;   // this CTA's
  int32_t unit1;
  int32_t slot;    // where its part goes, -1: the item is whole
  int32_t group;
};

// Units of a row tile of a sequence.
__device__ __forceinline__ int32_t units_of(const KvAttendArgs& k, const KvSeq& s, int32_t group, int32_t tile) {
  const int32_t last = min(s.n * group, (tile + 1) * kTileRows) - 1;
  return tile_units(kv_row_begin(k, s, tile * kTileRows / group) & -kTileKeys, kv_row_end(k, s, last / group));
}

// Where the span of CTA `cta` begins; a warp finds it together.
__device__ __forceinline__ KvSpan find_span(const KvAttendArgs& k, const KvTilePlan& p, int64_t cta, int64_t* span) {
  const int lane = threadIdx.x & 31;
  const int32_t n_seqs = int32_t(k.a.n_seqs), heads = int32_t(k.cache.heads), group = int32_t(k.a.q_heads) / heads;
  const int64_t* costs = reinterpret_cast<const int64_t*>(reinterpret_cast<const char*>(k.a.workspace) + p.costs_at);
  const int64_t total = costs[n_seqs];
  *span = span_units(total, p.ctas);
  const int64_t at = cta * *span;
  if (at >= total) return KvSpan{n_seqs, 0, 0, 0};
  int32_t lo = 0, hi = n_seqs;  // the last sequence with costs[lo] <= at
  while (hi - lo > 1) {
    // 31 places between them at a time.
    const int32_t step = (hi - lo + 31) / 32, mid = lo + (lane + 1) * step;
    const uint32_t past = __ballot_sync(0xffffffffu, mid >= hi || costs[mid] > at);
    const int first = __ffs(past) - 1;  // lane 31's is at or past hi
    hi = min(hi, lo + (first + 1) * step);
    lo += first * step;
  }
  const KvSeq s = kv_sequence(k, uint32_t(lo));
  const int32_t tiles = (s.n * group + kTileRows - 1) / kTileRows;
  int64_t rest = at - costs[lo];
  for (int32_t base = 0; base < tiles; base += 32) {
    const int32_t t = base + lane;
    const int32_t units = t < tiles ? units_of(k, s, group, t) : 0;
    int64_t sum = int64_t(units) * heads;
    for (int w = 1; w < 32; w <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, sum, w);
      if (lane >= w) sum += x;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, sum > rest);
    if (past) {
      const int l = __ffs(past) - 1;
      const int32_t u = __shfl_sync(0xffffffffu, units, l);
      const int64_t in = rest - (__shfl_sync(0xffffffffu, sum, l) - int64_t(u) * heads);
      return KvSpan{lo, base + l, int32_t(in / u), int32_t(in % u)};
    }
    rest -= __shfl_sync(0xffffffffu, sum, 31);
  }
  return KvSpan{n_seqs, 0, 0, 0};
}

struct Walk {
  const KvAttendArgs& k;
  int32_t seq, tile, head, unit;
  int64_t left;
  int32_t cta;
  bool first;

  __device__ Walk(const KvAttendArgs& args, const KvTilePlan& p) : k(args), cta(int32_t(blockIdx.x)), first(true) {
    const KvSpan span = find_span(args, p, blockIdx.x, &left);
    seq = span.seq, tile = span.tile, head = span.head, unit = span.unit;
  }

  __device__ bool next(Item& it) {
    it.group = int32_t(k.a.q_heads / k.cache.heads);
    for (;;) {
      if (left <= 0 || seq >= int32_t(k.a.n_seqs)) return false;
      it.s = kv_sequence(k, uint32_t(seq));
      it.row0 = tile * kTileRows;
      it.rows = min(kTileRows, it.s.n * it.group - it.row0);
      if (it.rows > 0) break;
      ++seq, tile = 0, head = 0, unit = 0;
    }
    it.seq = uint32_t(seq);
    it.head = head;
    it.first = kv_row_begin(k, it.s, it.row0 / it.group);
    it.begin = it.first & -kTileKeys;
    it.end = kv_row_end(k, it.s, (it.row0 + it.rows - 1) / it.group);
    it.units = tile_units(it.begin, it.end);
    it.unit0 = unit;
    it.unit1 = int32_t(min(int64_t(it.units), unit + left));
    left -= it.unit1 - it.unit0;
    it.slot = it.unit0 == 0 && it.unit1 == it.units ? -1 : 2 * cta + (first ? 0 : 1);
    first = false;
    unit = 0;
    if (++head == int32_t(k.cache.heads)) {
      head = 0;
      ++tile;  // a sequence's end is seen by the next call
    }
    return true;
  }
};

// What the sequences in front of each cost, and all of them: one block, a warp for
// a sequence, its lanes over the row tiles.
__global__ void __launch_bounds__(1024) kv_tile_costs_kernel(const __grid_constant__ KvAttendArgs k, const KvTilePlan p) {
  let_next_kernel_start();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int32_t n_seqs = int32_t(k.a.n_seqs), heads = int32_t(k.cache.heads);
  const int32_t group = int32_t(k.a.q_heads) / heads;
  int64_t* costs = reinterpret_cast<int64_t*>(reinterpret_cast<char*>(k.a.workspace) + p.costs_at);
  __shared__ int64_t part[2][32];
  int64_t front = 0;
  for (int32_t base = 0; base < n_seqs; base += 32) {
    const int32_t seq = base + warp;
    int64_t cost = 0;
    if (seq < n_seqs) {
      const KvSeq s = kv_sequence(k, uint32_t(seq));
      const int32_t tiles = (s.n * group + kTileRows - 1) / kTileRows;
      for (int32_t t = lane; t < tiles; t += 32) cost += units_of(k, s, group, t);
      for (int w = 16; w; w >>= 1) cost += __shfl_xor_sync(0xffffffffu, cost, w);
      cost *= heads;
    }
    int64_t* sums = part[base >> 5 & 1];  // the other's readers may still be at it
    if (lane == 0) sums[warp] = cost;
    __syncthreads();
    int64_t sum = sums[lane];
    const int64_t mine = sum;
    for (int w = 1; w < 32; w <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, sum, w);
      if (lane >= w) sum += x;
    }
    if (warp == 0 && base + lane < n_seqs) costs[base + lane] = front + sum - mine;
    front += __shfl_sync(0xffffffffu, sum, 31);
  }
  if (threadIdx.x == 0) costs[n_seqs] = front;
}

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)), "l"(reinterpret_cast<const uint64_t&>(c)));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)));
  return d;
}

// The larger of three, NaN if one is.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Which of 32 tokens the row sees: lo <= place < hi, and they are there.
__device__ __forceinline__ uint32_t seen_bits(const KeyInfo& info, int piece, int32_t lo, int32_t hi) {
  const int32_t from = min(max(lo - piece * 32, 0), 32), to = min(max(hi - piece * 32, 0), 32);
  const uint32_t below_to = to == 32 ? 0xffffffffu : (1u << to) - 1, below_from = from == 32 ? 0xffffffffu : (1u << from) - 1;
  return info.seen[piece] & below_to & ~below_from;
}

// A scale in other units, y, that keeps a trace (and its sign) where it becomes too
// small for them: what a row sees of V scales is nothing only if all of them are zero.
__device__ __forceinline__ float still_there(float x, float y) {
  return x != 0.0f && fabsf(y) < kKvSmallestScale ? copysignf(kKvSmallestScale, x) : y;
}

// The largest V scale among the tokens that the row sees, or, if all of the tile
// are within 2^4, the smallest there is.
__device__ __noinline__ float largest_seen(const KeyInfo& info, int32_t lo, int32_t hi) {
  if (info.low_scale >= info.top_scale * (1.0f / 16)) {
    uint32_t any = 0;
    for (int piece = 0; piece < 4; ++piece) any |= seen_bits(info, piece, lo, hi);
    return any ? info.low_scale : 0.0f;
  }
  float top = 0.0f;
#pragma unroll 1
  for (int piece = 0; piece < 4; ++piece) {
    const uint32_t seen = seen_bits(info, piece, lo, hi);
#pragma unroll
    for (int x = 0; x < 32; ++x) top = fmaxf(top, seen >> x & 1 ? fabsf(info.value_scale[piece * 32 + x]) : 0.0f);
  }
  return top;
}

// Multiplies a row's fp32 values, or pairs of 16-bit ones, in TMEM: rarely done,
// so out of the way. Loads and stores of TMEM keep no order among themselves: the
// caller has waited for its own of both (tmem_wait_load, tmem_wait_store).
__device__ __noinline__ void rescale_sums(uint32_t at, int columns, float by) {
#pragma unroll 1
  for (int x = 0; x < columns; x += 32) {
    uint32_t s[32];
    tmem_load32(s, at + x);
    tmem_wait_load(s);
#pragma unroll
    for (int i = 0; i < 32; ++i) s[i] = __float_as_uint(__uint_as_float(s[i]) * by);
    tmem_store32(at + x, s);
  }
}
template <bool BF16>
__device__ __noinline__ void rescale_weights(uint32_t at, float by) {
  uint32_t p[16];
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
               : PF_R4(p, 0), PF_R4(p, 4), PF_R4(p, 8), PF_R4(p, 12)
               : "r"(at));
  asm volatile("tcgen05.wait::ld.sync.aligned;" : PF_RW4(p, 0), PF_RW4(p, 4), PF_RW4(p, 8), PF_RW4(p, 12) : : "memory");
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    float2 w;
    if constexpr (BF16) {
      w = make_float2(__uint_as_float(p[i] << 16), __uint_as_float(p[i] & 0xffff0000u));
    } else {
      w = __half22float2(*reinterpret_cast<const __half2*>(&p[i]));
    }
    p[i] = pack_pair<BF16>(w.x * by, w.y * by);
  }
  tmem_store16(at, p);
}

// 32 weights 2^y as 16-bit pairs (SCALED: times the V scales), and their sum in fp32.
template <bool SCALED, bool BF16>
__device__ __forceinline__ float2 weights32(uint32_t (&p)[16], const float2 (&y)[16], const float* scales) {
  float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
#pragma unroll
  for (int x = 0; x < 16; ++x) {
    float2 w = make_float2(fast_exp2(y[x].x), fast_exp2(y[x].y));
    sum[x & 1] = add2(sum[x & 1], w);
    if constexpr (SCALED) w = mul2(w, *reinterpret_cast<const float2*>(scales + 2 * x));
    p[x] = pack_pair<BF16>(w.x, w.y);
  }
  return add2(sum[0], sum[1]);
}

// What a row's softmax carries from tile to tile.
struct RowState {
  float m;  // what the weights go by: 2^(score - m). The maximum less the lift
  float l;  // their sum
};

// One tile's scores of a row into weights 2^(score f - m), 16-bit pairs over the
// scores in TMEM, 32 scores at a time. m stays as long as no score passes it by
// kRaise more than the lift. Where one does (or the row had none yet), m becomes the
// largest score so far less the lift, and the sum, O (o_columns of it) and the weights already made follow.
template <bool QUANT, bool SCALED, bool BF16, bool MASKED>
__device__ __forceinline__ void row_weights(RowState& row, const KeyInfo& info, uint32_t s_at, uint32_t o_at, int o_columns,
                                            int32_t lo, int32_t hi, float f) {
  constexpr float kUp = BF16 ? 0.0f : SCALED ? kLiftScaled : kLift;
  float2 all = make_float2(row.l, 0.0f);
  const float2 ff = make_float2(f, f);
  uint32_t s[32];
  tmem_load32(s, s_at);
#pragma unroll 1
  for (int piece = 0; piece < 4; ++piece) {
    float2 y[16];
    float4 ks[QUANT ? 8 : 1];
    if constexpr (QUANT) {
#pragma unroll
      for (int x = 0; x < 8; ++x) ks[x] = *reinterpret_cast<const float4*>(&info.key_scale[piece * 32 + 4 * x]);
    }
    const uint32_t seen = MASKED ? seen_bits(info, piece, lo, hi) : 0;
    const float base = row.m == -INFINITY ? 0.0f : row.m;
    const float2 minus = make_float2(-base, -base);
    tmem_wait_load(s);
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      y[x] = make_float2(__uint_as_float(s[2 * x]), __uint_as_float(s[2 * x + 1]));
      if constexpr (QUANT) y[x] = mul2(y[x], x % 2 ? make_float2(ks[x / 2].z, ks[x / 2].w) : make_float2(ks[x / 2].x, ks[x / 2].y));
      if constexpr (MASKED) {
        y[x].x = seen >> (2 * x) & 1 ? y[x].x : -INFINITY;
        y[x].y = seen >> (2 * x + 1) & 1 ? y[x].y : -INFINITY;
      }
      y[x] = fma2(y[x], ff, minus);
    }
    if (piece < 3) tmem_load32(s, s_at + (piece + 1) * 32);  // on its way meanwhile
    // The exponentials do not wait for the maximum: they are made again where it is passed.
    uint32_t p[16];
    const float* scales = info.value_scale + piece * 32;
    float2 sum = weights32<SCALED, BF16>(p, y, scales);
    float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int x = 0; x < 16; ++x) tops[x & 3] = max3_nan(tops[x & 3], y[x].x, y[x].y);
    const float top = max3_nan(max3_nan(tops[0], tops[1], tops[2]), tops[3], tops[3]);
    const bool raise = top > (row.m == -INFINITY ? -INFINITY : kRaise + kUp);  // a NaN raises nothing: it reaches the sum
    if (__any_sync(0xffffffffu, raise)) {
      // What is read back below was stored asynchronously (weights of pieces before, O by a rescaling), and the next
      // scores are still on their way into registers that a call may save: both are waited for first.
      tmem_wait_load(s);
      tmem_wait_store();
      float keep = 1.0f;
      if (raise) {
        const float by = top - kUp, m = base + by;
        keep = fast_exp2(row.m - m);  // 0 at first
        const float2 shift = make_float2(-by, -by);
#pragma unroll
        for (int x = 0; x < 16; ++x) y[x] = add2(y[x], shift);
        row.m = m;
        all = mul2(all, make_float2(keep, keep));
        sum = weights32<SCALED, BF16>(p, y, scales);
      }
      __syncwarp();
      rescale_sums(o_at, o_columns, keep);
      for (int before = 0; before < piece; ++before) rescale_weights<BF16>(s_at + before * 16, keep);
    }
    all = add2(all, sum);
    tmem_store16(s_at + piece * 16, p);
  }
  row.l = all.x + all.y;
}

template <uint32_t Q, uint32_t STORE, int DP>
__global__ void __launch_bounds__((Tiles<Q, STORE, DP>::kThreads), 1)
    kv_attend_tiles_kernel(const __grid_constant__ KvAttendArgs k, const __grid_constant__ KvTilePlan plan,
                           const __grid_constant__ KvBoxMaps maps) {
  using S = Tiles<Q, STORE, DP>;
  using T = typename KvElem<Q>::type;
  constexpr int kLoadThreads = S::kLoadThreads, kMmaWarp = S::kMmaWarp;
  extern __shared__ unsigned char raw_smem[];
  typename S::Shared& sh =
      *reinterpret_cast<typename S::Shared*>(raw_smem + ((1024 - (smem_u32(raw_smem) & 1023)) & 1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const pf_kv_cache& c = k.cache;
  Watch* watch = &sh.watch;

  if (threadIdx.x == 0) {
    bar_init(&sh.q_full, kLoadThreads);
    bar_init(&sh.q_empty, 1);
    for (int i = 0; i < S::kStages; ++i) bar_init(&sh.kv_full[i], kLoadThreads), bar_init(&sh.kv_empty[i], 1);
    for (int i = 0; i < kInfos; ++i) bar_init(&sh.info_full[i], kLoadThreads), bar_init(&sh.info_empty[i], kSoftmaxWarps * 32);
    for (int i = 0; i < 2; ++i) {
      bar_init(&sh.s_full[i], 1), bar_init(&sh.p_full[i], 128);
      bar_init(&sh.o_full[i], 1), bar_init(&sh.o_free[i], 128);
    }
    bar_init(&sh.done, 1);
    sh.watch = sh.stuck[0] = sh.stuck[1] = Watch{0, 0};
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sh.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tmem_before_sync();
  __syncthreads();
  tmem_after_sync();
  const uint32_t tmem = 0;
  if (sh.tmem != 0) sh.watch.failed = 1;  // cannot be: the waits would end the call
  wait_for_previous_kernel();  // the costs
  let_next_kernel_start();

  Walk walk(k, plan);
  Item it;

  if (warp >= kSoftmaxWarps && warp < kMmaWarp) {
    // ------------------------------------------------------------- loading
    const int tid = threadIdx.x - kSoftmaxWarps * 32;
    uint32_t tile_no = 0, stage_no = 0, item_no = 0;
    // A thread whose wait gave up goes on without copying to the next place where all loading threads meet.
    bool ok = true;
    // Copies rows of 16-bit values; their arrival counts for the stage's barrier by itself (the products' thread
    // orders them before its instructions' reads).
    auto copy_rows = [&](const int64_t* at, uint64_t data) -> bool {
      constexpr int kPieces = DP / 8;
      if (!bar_wait(&sh.kv_empty[stage_no % S::kStages], (stage_no / S::kStages & 1) ^ 1, watch)) return false;
      const int piece = tid % kPieces;
      const bool there = piece * 8 < int(c.head_dim);
      const uint32_t base = smem_u32(sh.kv[stage_no % S::kStages]) + (piece >> 3) * 16384;
      const char* from = reinterpret_cast<const char*>(data) + piece * 16;
      // Eight rows' offsets are read, then the eight copies are issued: the reads' latency is met once.
      constexpr int kRows = kLoadThreads / kPieces, kAhead = 8;
#pragma unroll 1
      for (int r0 = tid / kPieces; r0 < kTileKeys; r0 += kRows * kAhead) {
        int64_t off[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) off[i] = r0 + i * kRows < kTileKeys ? at[r0 + i * kRows] : -1;
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          const int r = r0 + i * kRows;
          const bool on = there && off[i] >= 0;
          if (r < kTileKeys) {
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(base + r * 128 + ((piece & 7) ^ (r & 7)) * 16),
                         "l"(on ? from + off[i] : reinterpret_cast<const char*>(data)), "r"(on ? 16 : 0)
                         : "memory");
          }
        }
      }
      asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&sh.kv_full[stage_no % S::kStages])) : "memory");
      ++stage_no;
      return true;
    };
    // Rows of codes: copied as they are into the stage's upper half, then read by all loading threads and, when all
    // have, written over it as fp16.
    constexpr int kCodePieces = DP / 16;  // 16-byte pieces of a row
    constexpr int kCodeRows = kLoadThreads / kCodePieces;
    constexpr int kCodeLoads = (kTileKeys + kCodeRows - 1) / kCodeRows;
    auto copy_codes = [&](uint32_t stage, const int64_t* at, uint64_t data) -> bool {
      const bool free = bar_wait(&sh.kv_empty[stage % S::kStages], (stage / S::kStages & 1) ^ 1, watch);
      if (free) {
        const int piece = tid % kCodePieces;
        const bool there = piece * 16 < int(c.head_dim);
        const uint32_t base = smem_u32(sh.kv[stage % S::kStages]) + S::kTileBytes / 2 + piece * 16;
        const char* from = reinterpret_cast<const char*>(data) + piece * 16;
        int64_t off[kCodeLoads];
#pragma unroll
        for (int i = 0; i < kCodeLoads; ++i) {
          const int r = tid / kCodePieces + i * kCodeRows;
          off[i] = r < kTileKeys ? at[r] : -1;
        }
#pragma unroll
        for (int i = 0; i < kCodeLoads; ++i) {
          const int r = tid / kCodePieces + i * kCodeRows;
          const bool on = there && off[i] >= 0;
          if (r < kTileKeys) {
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(base + r * DP),
                         "l"(on ? from + off[i] : reinterpret_cast<const char*>(data)), "r"(on ? 16 : 0)
                         : "memory");
          }
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      return free;
    };
    auto expand_codes = [&](uint32_t stage, const float* scales) -> bool {
      if (!loaders_agree<kLoadThreads>(ok)) return false;  // all copies are there
      unsigned char* base = sh.kv[stage % S::kStages];
      uint4 codes[kCodeLoads];
#pragma unroll
      for (int i = 0; i < kCodeLoads; ++i) {
        const int r = tid / kCodePieces + i * kCodeRows;
        if (r < kTileKeys) codes[i] = *reinterpret_cast<const uint4*>(base + S::kTileBytes / 2 + r * DP + tid % kCodePieces * 16);
      }
      loaders_agree<kLoadThreads>(true);  // and read
      const int piece = tid % kCodePieces * 2;  // of 16 bytes of fp16
      base += (piece >> 3) * 16384;
#pragma unroll
      for (int i = 0; i < kCodeLoads; ++i) {
        const int r = tid / kCodePieces + i * kCodeRows;
        if (r >= kTileKeys) break;
        uint2 x = codes_to_half4<STORE>(codes[i].x), y = codes_to_half4<STORE>(codes[i].y);
        uint2 z = codes_to_half4<STORE>(codes[i].z), w = codes_to_half4<STORE>(codes[i].w);
        if (scales) {
          const __half2 by = __float2half2_rn(scales[r]);  // below 2
          x = times_half4(x, by), y = times_half4(y, by), z = times_half4(z, by), w = times_half4(w, by);
        }
        // Eight threads write a row: those of its second block the other piece first, so that all banks are met.
        const uint4 lo = make_uint4(x.x, x.y, y.x, y.y), hi = make_uint4(z.x, z.y, w.x, w.y);
        const int swapped = piece >> 3;
        *reinterpret_cast<uint4*>(base + r * 128 + (((piece & 7) + swapped) ^ (r & 7)) * 16) = swapped ? hi : lo;
        *reinterpret_cast<uint4*>(base + r * 128 + (((piece & 7) + (swapped ^ 1)) ^ (r & 7)) * 16) = swapped ? lo : hi;
      }
      fence_async_shared();
      bar_arrive(&sh.kv_full[stage % S::kStages]);
      return true;
    };

    while (loaders_agree<kLoadThreads>(ok) && walk.next(it)) {
      auto page_of = [&](int32_t j) { return plan.page_shift >= 0 ? uint32_t(j) >> plan.page_shift : uint32_t(j) / c.block_size; };
      // Each thread's tokens of a tile: tid and, with three warps, tid + 96 for the first.
      auto token_of = [&](int32_t unit, int u) { return it.begin + unit * kTileKeys + tid + u * kLoadThreads; };
      int32_t block[2], ahead[2] = {-1, -1};
      auto look_up = [&](int32_t unit, int32_t (&to)[2]) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int32_t j = token_of(unit, u);
          const bool on = unit < it.unit1 && tid + u * kLoadThreads < kTileKeys && j >= it.first && j < it.end;
          to[u] = on ? kv_block(k, it.seq, page_of(j)) : -1;
        }
      };
      // A tile's scales, a tile ahead: `block` is its own by then.
      float ks[2] = {0.0f, 0.0f}, vs[2] = {0.0f, 0.0f};
      auto load_scales = [&](int32_t unit) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          ks[u] = vs[u] = 0.0f;
          if (block[u] >= 0) {
            const int32_t j = token_of(unit, u);
            const int64_t b = block[u], at = uint32_t(j) - page_of(j) * c.block_size;
            ks[u] = reinterpret_cast<const float*>(c.key.scale)[b * c.key.scale_block_stride + at * c.key.scale_token_stride + it.head * c.key.scale_head_stride];
            vs[u] = reinterpret_cast<const float*>(c.value.scale)[b * c.value.scale_block_stride + at * c.value.scale_token_stride + it.head * c.value.scale_head_stride];
          }
        }
      };
      look_up(it.unit0, block);
      if constexpr (S::kQuant) load_scales(it.unit0);

      // Q: the rows' places first, a thread for each; then 16-byte pieces, neighbouring threads on one row.
      ok = loaders_agree<kLoadThreads>(bar_wait(&sh.q_empty, (item_no & 1) ^ 1, watch));
      if (!ok) break;
      for (int r = tid; r < kTileRows; r += kLoadThreads) {
        const int32_t row = it.row0 + r, i = row / it.group;
        sh.q_at[r] = r < it.rows ? (int64_t(it.s.first + i) * k.a.query.token_stride +
                                    int64_t(it.head * it.group + row - i * it.group) * k.a.query.head_stride) * 2 : -1;
      }
      loaders_agree<kLoadThreads>(true);
      {
        constexpr int kPieces = DP / 8, kRows = kLoadThreads / kPieces, kAhead = 8;
        const int piece = tid % kPieces;
        const bool there = piece * 8 < int(c.head_dim);
        const char* from = reinterpret_cast<const char*>(k.a.query.data) + piece * 16;
        const int q_rows = it.rows <= 128 ? 128 : kTileRows;
        if (!S::kQuant && k.a.scale >= 0.0f) {
          // As they are: asynchronous copies, whose arrival counts for the barrier.
          for (int r0 = tid / kPieces; r0 < q_rows; r0 += kRows * kAhead) {
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
              const int r = r0 + i * kRows;
              if (r < q_rows) {
                const int64_t off = sh.q_at[r];
                const bool on = there && off >= 0;
                const uint32_t to = smem_u32(sh.q[r >> 7]) + (piece >> 3) * 16384 + (r & 127) * 128 + ((piece & 7) ^ (r & 7)) * 16;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(on ? from + off : from - piece * 16), "r"(on ? 16 : 0)
                             : "memory");
              }
            }
          }
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&sh.q_full)) : "memory");
          for (int r = tid; r < kTileRows; r += kLoadThreads) sh.q_unit[item_no & 1][r] = 1.0f;
        } else {
          const uint32_t flip = k.a.scale < 0.0f ? 0x80008000u : 0u;
          for (int r0 = tid / kPieces; r0 < q_rows; r0 += kRows * kAhead) {
            uint4 v[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
              const int r = r0 + i * kRows;
              const int64_t off = r < q_rows ? sh.q_at[r] : -1;
              v[i] = make_uint4(0, 0, 0, 0);
              if (there && off >= 0) v[i] = *reinterpret_cast<const uint4*>(from + off);
            }
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
              const int r = r0 + i * kRows;
              float bring = 1.0f;
              if constexpr (S::kQuant && Q == PF_DTYPE_BF16) {
                // The row's largest exponent, over its threads (all lanes come along, whatever their row).
                uint32_t top = 0;
                for (uint32_t x : {v[i].x, v[i].y, v[i].z, v[i].w}) top = max(top, max(x & 0x7fffu, x >> 16 & 0x7fffu));
#pragma unroll
                for (int w = kPieces >> 1; w; w >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, w));
                const int e = min(max(int(top >> 7) - 127, -100), 127);
                bring = __uint_as_float(uint32_t(127 + 14 - e) << 23);
                if (piece == 0 && r < q_rows) sh.q_unit[item_no & 1][r] = __uint_as_float(uint32_t(127 - 14 + e) << 23);
              } else {
                if (piece == 0 && r < q_rows) sh.q_unit[item_no & 1][r] = 1.0f;
              }
              auto convert = [&](uint32_t x) {
                x ^= flip;
                if constexpr (S::kQuant && Q == PF_DTYPE_BF16) {
                  x = pack_pair<false>(__uint_as_float(x << 16) * bring, __uint_as_float(x & 0xffff0000u) * bring);
                }
                return x;
              };
              if (r < q_rows) {
                *reinterpret_cast<uint4*>(sh.q[r >> 7] + (piece >> 3) * 16384 + (r & 127) * 128 + ((piece & 7) ^ (r & 7)) * 16) =
                    make_uint4(convert(v[i].x), convert(v[i].y), convert(v[i].z), convert(v[i].w));
              }
            }
          }
          fence_async_shared();
          bar_arrive(&sh.q_full);
        }
      }

      // What the softmax needs of a tile, and where its rows are.
      uint32_t v_exp = 1;
      auto offsets = [&](int32_t unit, KeyInfo& info) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int x = tid + u * kLoadThreads;
          if (x >= kTileKeys) break;  // whole warps
          const int32_t j = token_of(unit, u);
          const int64_t b = block[u], at = uint32_t(j) - page_of(j) * c.block_size;
          constexpr int kElt = S::kQuant ? 1 : 2;
          info.key_at[x] = b < 0 ? -1 : (b * c.key.block_stride + at * c.key.token_stride + it.head * c.key.head_stride) * kElt;
          info.value_at[x] = b < 0 ? -1 : (b * c.value.block_stride + at * c.value.token_stride + it.head * c.value.head_stride) * kElt;
          if constexpr (S::kQuant) {
            info.key_scale[x] = ks[u];
            const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(vs[u]) & 0x7fffffffu);
            const uint32_t low = __reduce_min_sync(0xffffffffu, b < 0 ? 0x7f800000u : __float_as_uint(vs[u]) & 0x7fffffffu);
            if (lane == 0) sh.warp_max[tile_no & 1][x >> 5] = top, sh.warp_min[tile_no & 1][x >> 5] = low;
          }
        }
      };
      auto prepare = [&](int32_t unit) -> bool {
        KeyInfo& info = sh.info[tile_no % kInfos];
        ok = ok && bar_wait(&sh.info_empty[tile_no % kInfos], (tile_no / kInfos & 1) ^ 1, watch);
        const uint32_t seen = __ballot_sync(0xffffffffu, block[0] >= 0);
        if (lane == 0 && tid < kTileKeys) info.seen[tid >> 5] = seen;
        if (tid < kTileKeys - kLoadThreads) {
          const uint32_t last = __ballot_sync(0xffffffffu, block[1] >= 0);
          if (lane == 0) info.seen[kLoadThreads / 32] = last;
        }
        if constexpr (S::kQuant) {
          offsets(unit, info);
          if (tid == 0) info.far = 0;
        }
        // Meeting here also keeps the slots apart: who writes a slot again (kInfos tiles on; warp_max: two) has
        // met those who read it last.
        ok = loaders_agree<kLoadThreads>(ok);
        if (!ok) return false;
        if constexpr (S::kQuant) {
          const uint32_t* w = sh.warp_max[tile_no & 1];
          v_exp = max(v_exp, min(max(max(w[0], w[1]), max(w[2], w[3])) >> 23, 253u));
          const float v_inv = __uint_as_float((254 - v_exp) << 23);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            if (tid + u * kLoadThreads < kTileKeys) {
              const float in_units = still_there(vs[u], vs[u] * v_inv);
              info.value_scale[tid + u * kLoadThreads] = in_units;
              // The smallest scale that a row is written with is that of zeros.
              if (fabsf(in_units) < kFarScale && fabsf(vs[u]) > kKvSmallestScale) info.far = 1;
            }
          }
          if (tid == 0) {
            info.v_exp = v_exp;
            const uint32_t* low = sh.warp_min[tile_no & 1];
            const float top_scale = __uint_as_float(max(max(w[0], w[1]), max(w[2], w[3])));
            const float low_scale = __uint_as_float(min(min(low[0], low[1]), min(low[2], low[3])));
            info.top_scale = still_there(top_scale, top_scale * v_inv);
            info.low_scale = still_there(low_scale, low_scale * v_inv);
          }
        }
        bar_arrive(&sh.info_full[tile_no % kInfos]);
        return true;
      };
      // A whole tile of one side by TMA: the thread that has a box's first token issues it.
      auto load_boxes = [&](int32_t unit, const CUtensorMap& map) -> bool {
        const uint32_t stage = stage_no++ % S::kStages;
        if (!bar_wait(&sh.kv_empty[stage], ((stage_no - 1) / S::kStages & 1) ^ 1, watch)) return false;
        uint32_t mine = 0;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int x = tid + u * kLoadThreads;
          if (x < kTileKeys && x % plan.box_rows == 0) mine += plan.box_rows * DP * 2;
        }
        if (mine) {
          bar_arrive_expecting(&sh.kv_full[stage], mine);
        } else {
          bar_arrive(&sh.kv_full[stage]);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int x = tid + u * kLoadThreads;
          if (x < kTileKeys && x % plan.box_rows == 0) {
            const int32_t j = token_of(unit, u);
#pragma unroll
            for (int d = 0; d < DP; d += 64) {
              load_box(smem_u32(sh.kv[stage]) + d / 64 * 16384 + x * 128, &map, d, int(uint32_t(j) - page_of(j) * c.block_size), it.head, block[u], &sh.kv_full[stage]);
            }
          }
        }
        return true;
      };
      if constexpr (S::kQuant) {
        // Two stages' copies are on their way while one is expanded: this tile's V and the next one's K.
        if (!prepare(it.unit0)) break;
        const KeyInfo* info = &sh.info[tile_no % kInfos];
        ok = copy_codes(stage_no, info->key_at, c.key.data);
        ok = copy_codes(stage_no + 1, info->value_at, c.value.data) && ok;
        look_up(it.unit0 + 1, block);
        bool broken = false;
        for (int32_t unit = it.unit0; unit < it.unit1; ++unit) {
          const float* scales = S::kScaledValues ? info->value_scale : nullptr;
          const bool more = unit + 1 < it.unit1;
          // What the next tile needs is read while this one's K is expanded.
          load_scales(unit + 1);
          look_up(unit + 2, ahead);
          asm volatile("cp.async.wait_group 1;" ::: "memory");
          broken = !expand_codes(stage_no, nullptr);
          if (broken) break;
          ++tile_no;
          if (more) {
            broken = !prepare(unit + 1);
            if (broken) break;
            info = &sh.info[tile_no % kInfos];
            ok = copy_codes(stage_no + 2, info->key_at, c.key.data);
            block[0] = ahead[0], block[1] = ahead[1];
            asm volatile("cp.async.wait_group 1;" ::: "memory");
          } else {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
          }
          broken = !expand_codes(stage_no + 1, scales);
          if (broken) break;
          if (more) ok = copy_codes(stage_no + 3, info->value_at, c.value.data);
          stage_no += 2;
        }
        if (broken) break;
      } else {
        for (int32_t unit = it.unit0; unit < it.unit1; ++unit, ++tile_no) {
          if (!prepare(unit)) break;
          KeyInfo& info = sh.info[tile_no % kInfos];
          const bool whole = (info.seen[0] & info.seen[1] & info.seen[2] & info.seen[3]) == 0xffffffffu;
          const bool boxed = whole && plan.box_rows;
          info.boxed = boxed;  // all threads write the same
          if (boxed) {
            ok = load_boxes(unit, maps.key) && load_boxes(unit, maps.value);
          } else {
            offsets(unit, info);
            if (!loaders_agree<kLoadThreads>(true)) break;  // the offsets are written
            ok = copy_rows(info.key_at, c.key.data) && copy_rows(info.value_at, c.value.data);
          }
          look_up(unit + 1, block);
        }
      }
      ++item_no;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (*reinterpret_cast<volatile int*>(&watch->failed)) {  // boxes that nobody waits for any more
      for (uint32_t n = stage_no > S::kStages ? stage_no - S::kStages : 0; n < stage_no; ++n) {
        bar_wait(&sh.kv_full[n % S::kStages], n / S::kStages & 1, &sh.stuck[1]);
      }
    }
  } else if (warp == kMmaWarp) {
    // ------------------------------------------------------------ products
    constexpr uint32_t kScores = instruction(S::kBf16, kTileKeys, false), kSums = instruction(S::kBf16, DP, true);
    uint32_t stage_no = 0, info_no = 0, item_no = 0, tile_no[2] = {0, 0}, o_no[2] = {0, 0};
    const uint32_t q_at = smem_u32(sh.q), kv_at = smem_u32(sh.kv);
    // A stage is there. What copies wrote (no box, no store with a fence of its own) is ordered before what the
    // products read.
    auto filled = [&](uint32_t stage, uint32_t info) {
      const bool ok = bar_wait_warp(&sh.kv_full[stage % S::kStages], stage / S::kStages & 1, watch);
      if constexpr (!S::kQuant) {
        if (!sh.info[info % kInfos].boxed) fence_async_shared();
      }
      return ok;
    };
    // The stage and the half are constants here: addresses and descriptors are then uniform from the start, and an
    // instruction is issued in its own time, not in that of six moves to uniform registers.
    auto scores = [&](auto half, auto stage) {
      constexpr int h = decltype(half)::value, st = decltype(stage)::value;
      const uint64_t a = operand(q_at + h * S::kTileBytes, 16), b = operand(kv_at + st * S::kTileBytes, 16);
      if (elected()) {
#pragma unroll
        for (int x = 0; x < DP / 16; ++x) {
          constexpr uint32_t kBlock = 16384 >> 4, kPiece = 32 >> 4;
          const uint32_t off = (x >> 2) * kBlock + (x & 3) * kPiece;
          mma_ss(S::kS + h * 128, a + off, b + off, kScores, x > 0);
        }
        mma_commit(&sh.s_full[h]);
      }
      __syncwarp();
    };
    auto sums = [&](auto half, auto stage, bool add) {
      constexpr int h = decltype(half)::value, st = decltype(stage)::value;
      const uint64_t b = operand(kv_at + st * S::kTileBytes, 16384);
      if (elected()) {
        mma_ts(S::kO + h * 128, S::kS + h * 128, b, kSums, add);
#pragma unroll
        for (int x = 1; x < kTileKeys / 16; ++x) mma_ts(S::kO + h * 128, S::kS + h * 128 + x * 8, b + x * (2048 >> 4), kSums, true);
      }
      __syncwarp();
    };
    auto commit = [&](uint64_t* bar) {
      if (elected()) mma_commit(bar);
      __syncwarp();
    };
    using Zero = std::integral_constant<int, 0>;
    using One = std::integral_constant<int, 1>;
    bool ok = true;
    int32_t units = 0;  // of the item
    int halves = 0;
    // Tile j of the item, in the stages 2 B and 2 B + 1.
    auto tile = [&](int32_t j, auto parity) {
      constexpr int B = decltype(parity)::value;
      using Key = std::integral_constant<int, 2 * B>;
      using Value = std::integral_constant<int, 2 * B + 1>;
      using NextKey = std::integral_constant<int, 2 - 2 * B>;
      const uint32_t v = stage_no + 1, next_key = stage_no + 2;
      if (j == 0) {
        if (!(ok = filled(stage_no, info_no))) return;
        tmem_after_sync();
        scores(Zero{}, Key{});
        if (halves == 2) scores(One{}, Key{});
        commit(&sh.kv_empty[Key::value]);
        if (units == 1) commit(&sh.q_empty);
      }
      if (!(ok = filled(v, info_no))) return;
      auto half = [&](auto which) -> bool {
        constexpr int h = decltype(which)::value;
        if (!bar_wait_warp(&sh.p_full[h], tile_no[h]++ & 1, watch)) return false;
        if (j == 0 && !bar_wait_warp(&sh.o_free[h], (o_no[h]++ & 1) ^ 1, watch)) return false;
        tmem_after_sync();
        sums(which, Value{}, j > 0);
        if (j + 1 < units) {
          if (h == 0 && !filled(next_key, info_no + 1)) return false;
          scores(which, NextKey{});
        } else {
          commit(&sh.o_full[h]);
        }
        return true;
      };
      if (!(ok = half(Zero{}))) return;
      if (halves == 2 && !(ok = half(One{}))) return;
      commit(&sh.kv_empty[Value::value]);
      if (j + 1 < units) commit(&sh.kv_empty[NextKey::value]);
      if (j + 2 == units) commit(&sh.q_empty);
      stage_no += 2;
      ++info_no;
    };
    while (ok && walk.next(it)) {
      halves = it.rows > 128 ? 2 : 1;
      units = it.unit1 - it.unit0;
      if (!(ok = bar_wait_warp(&sh.q_full, item_no & 1, watch))) break;
      if constexpr (!S::kQuant) fence_async_shared();
      for (int32_t j = 0; j < units && ok; ++j) {
        if (stage_no & 2) {
          tile(j, One{});
        } else {
          tile(j, Zero{});
        }
      }
      ++item_no;
    }
    // Whatever was issued is done before the memory that it uses is given back.
    commit(&sh.done);
    bar_wait(&sh.done, 0, &sh.stuck[0]);
  } else {
    // ------------------------------------------------------------- softmax
    const int h = warp >> 2, r = threadIdx.x;  // r: the row of the item
    const uint32_t lanes = uint32_t(warp & 3) << 21;  // lane 32 * (warp % 4) in the address' upper half
    const uint32_t s_at = tmem + S::kS + h * 128 + lanes, o_at = tmem + S::kO + h * 128 + lanes;
    uint32_t tile_no = 0, s_no = 0, o_no = 0, item_no = 0;
    const float factor = fmaxf(fabsf(k.a.scale) * kLog2e, 1e-30f);  // never 0, which would turn -inf into NaN
    bool ok = true;
    while (ok && walk.next(it)) {
      const bool active = h * 128 < it.rows;
      const bool mine = r < it.rows;
      const int32_t row = it.row0 + (mine ? r : 0), i = row / it.group;
      const int32_t row_lo = mine ? kv_row_begin(k, it.s, i) : 0, row_hi = mine ? kv_row_end(k, it.s, i) : INT32_MAX;
      RowState sm{-INFINITY, 0.0f};
      float f = factor;
      uint32_t v_exp = 1;
      float seen_scale = 0.0f;  // the largest V scale that the row sees, in units of 2^(v_exp - 127)
      bool far = false;         // a tile held scales far below the unit of its time
      for (int32_t unit = it.unit0; unit < it.unit1; ++unit, ++tile_no) {
        KeyInfo& info = sh.info[tile_no % kInfos];
        if (!(ok = bar_wait_warp(&sh.info_full[tile_no % kInfos], tile_no / kInfos & 1, watch))) break;
        if (!active) {
          bar_arrive(&sh.info_empty[tile_no % kInfos]);
          continue;
        }
        if (unit == it.unit0) f = fmaxf(factor * sh.q_unit[item_no & 1][r], 1.2e-38f);
        if (!(ok = bar_wait_warp(&sh.s_full[h], s_no & 1, watch))) break;
        ++s_no;
        tmem_after_sync();
        const int32_t j0 = it.begin + unit * kTileKeys;
        const bool whole = (info.seen[0] & info.seen[1] & info.seen[2] & info.seen[3]) == 0xffffffffu;
        const bool masked = !whole || __any_sync(0xffffffffu, row_lo > j0 || row_hi < j0 + kTileKeys);
        const int o_columns = unit > it.unit0 ? DP : 0;  // O holds nothing yet in front of an item's first tile
        if constexpr (S::kQuant) {
          const uint32_t e = info.v_exp;
          if (e > v_exp) {
            const float by = e - v_exp > 126 ? 0.0f : __uint_as_float((127 - (e - v_exp)) << 23);
            rescale_sums(o_at, o_columns, by);
            seen_scale = still_there(seen_scale, seen_scale * by);
            v_exp = e;
          }
          seen_scale = fmaxf(seen_scale, masked ? largest_seen(info, row_lo - j0, row_hi - j0) : info.top_scale);
          far = far || info.far;
        }
        if (masked) {
          row_weights<S::kQuant, S::kQuant && !S::kScaledValues, S::kBf16, true>(sm, info, s_at, o_at, o_columns, row_lo - j0, row_hi - j0, f);
        } else {
          row_weights<S::kQuant, S::kQuant && !S::kScaledValues, S::kBf16, false>(sm, info, s_at, o_at, o_columns, 0, 0, f);
        }
        tmem_wait_store();
        tmem_before_sync();
        bar_arrive(&sh.p_full[h]);
        bar_arrive(&sh.info_empty[tile_no % kInfos]);
      }
      ++item_no;
      if (!ok) break;
      if (!active) continue;
      if (!(ok = bar_wait_warp(&sh.o_full[h], o_no & 1, watch))) break;
      ++o_no;
      tmem_after_sync();
      const float m = sm.m, l = sm.l;
      // The result, or this CTA's part of it. An infinity or a NaN in a value that this row does not see may
      // have met its weight of zero: such rows are made again, token by token.
      const float v_unit = S::kQuant ? __uint_as_float(v_exp << 23) : 1.0f;
      const int64_t token = int64_t(it.s.first) + i;
      const int32_t qh = it.head * it.group + row - i * it.group;
      T* out = reinterpret_cast<T*>(k.a.out.data) + token * k.a.out.token_stride + int64_t(qh) * k.a.out.head_stride;
      float* part = reinterpret_cast<float*>(reinterpret_cast<char*>(k.a.workspace) + plan.parts_at) +
                    int64_t(max(it.slot, 0)) * kTileRows * (DP + 2) + r;
      const float times = it.slot >= 0 ? v_unit : l == 0.0f ? 0.0f : v_unit / l;
      // And rows whose V scales are far below one that they do not see: it has set the power of two.
      bool bad = S::kQuant && v_exp > 9 && seen_scale > 0.0f && seen_scale < 1.0f / 4096;
      float largest = 0.0f;  // of O, where that has to be known
#pragma unroll 1
      for (int piece = 0; piece < DP / 32; ++piece) {
        uint32_t s[32];
        tmem_load32(s, o_at + piece * 32);
        tmem_wait_load(s);
        if (S::kQuant && far) {
#pragma unroll
          for (int x = 0; x < 32; ++x) largest = fmaxf(largest, fabsf(__uint_as_float(s[x])));
        }
#pragma unroll
        for (int x = 0; x < 32; ++x) {
          bad = bad || !isfinite(__uint_as_float(s[x]));
          s[x] = __float_as_uint(__uint_as_float(s[x]) * times);
        }
        if (mine && it.slot >= 0) {
#pragma unroll
          for (int x = 0; x < 32; ++x) part[(2 + piece * 32 + x) * kTileRows] = __uint_as_float(s[x]);
        } else if (mine) {
#pragma unroll
          for (int x = 0; x < 32; x += 8) {
            if (piece * 32 + x < int(c.head_dim)) {
              uint4 y;
              constexpr bool kOutBf16 = Q == PF_DTYPE_BF16;
              y.x = pack_pair<kOutBf16>(__uint_as_float(s[x]), __uint_as_float(s[x + 1]));
              y.y = pack_pair<kOutBf16>(__uint_as_float(s[x + 2]), __uint_as_float(s[x + 3]));
              y.z = pack_pair<kOutBf16>(__uint_as_float(s[x + 4]), __uint_as_float(s[x + 5]));
              y.w = pack_pair<kOutBf16>(__uint_as_float(s[x + 6]), __uint_as_float(s[x + 7]));
              *reinterpret_cast<uint4*>(out + piece * 32 + x) = y;
            }
          }
        }
        __syncwarp();
      }
      tmem_before_sync();
      bar_arrive(&sh.o_free[h]);
      // And rows whose result is so small that the rounding of what is far below the unit shows in it.
      if (S::kQuant && far) {
        bad = bad || largest < kSmallRow * (S::kScaledValues ? l : float((it.unit1 - it.unit0) * kTileKeys));
      }
      if (mine) {
        if (it.slot >= 0) {
          part[0] = m, part[kTileRows] = l;
        } else if (k.a.lse) {
          reinterpret_cast<float*>(k.a.lse)[token * k.a.q_heads + qh] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kLn2;
        }
      }
      uint32_t again = __ballot_sync(0xffffffffu, mine && bad && l == l);
      __syncwarp();
      while (again) {
        const int src = __ffs(again) - 1;
        again &= again - 1;
        const int32_t row_r = it.row0 + (r & ~31) + src, i_r = row_r / it.group, qh_r = it.head * it.group + row_r - i_r * it.group;
        const int64_t token_r = int64_t(it.s.first) + i_r;
        float m_r, l_r;
        float4 v;
        attend_row_exactly<Q, STORE>(k, it.seq, token_r, uint32_t(qh_r), uint32_t(it.head),
                                     max(it.begin + it.unit0 * kTileKeys, kv_row_begin(k, it.s, i_r)),
                                     min(it.begin + it.unit1 * kTileKeys, kv_row_end(k, it.s, i_r)), m_r, l_r, v, &sh.watch.alive);
        if (it.slot >= 0) {
          float* to = reinterpret_cast<float*>(reinterpret_cast<char*>(k.a.workspace) + plan.parts_at) +
                      int64_t(it.slot) * kTileRows * (DP + 2) + (r & ~31) + src;
          if (lane == 0) to[0] = m_r, to[kTileRows] = l_r;
          if (lane * 4 < DP) {
            float* at = to + (2 + lane * 4) * kTileRows;
            at[0] = v.x, at[kTileRows] = v.y, at[2 * kTileRows] = v.z, at[3 * kTileRows] = v.w;
          }
        } else {
          const float inv = l_r == 0.0f ? 0.0f : 1.0f / l_r;
          if (lane * 4 < int(c.head_dim)) {
            KvPack<T, 4> y;
            y.v[0] = kv_from_float<Q>(v.x * inv), y.v[1] = kv_from_float<Q>(v.y * inv);
            y.v[2] = kv_from_float<Q>(v.z * inv), y.v[3] = kv_from_float<Q>(v.w * inv);
            *reinterpret_cast<KvPack<T, 4>*>(reinterpret_cast<T*>(k.a.out.data) + token_r * k.a.out.token_stride +
                                             int64_t(qh_r) * k.a.out.head_stride + lane * 4) = y;
          }
          if (lane == 0 && k.a.lse) {
            reinterpret_cast<float*>(k.a.lse)[token_r * k.a.q_heads + qh_r] = l_r == 0.0f ? -INFINITY : (m_r + log2f(l_r)) * kLn2;
          }
        }
      }
    }
  }
  __syncthreads();
  if (warp == kMmaWarp) {
    if (sh.watch.failed) kv_flag(reinterpret_cast<int32_t*>(k.a.status), PF_KV_TIMED_OUT);
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(sh.tmem));
  }
}

// Joins the parts of an item that lies in several spans: blocks of the CTA in whose
// span it begins, 32 rows each. A part is stored value by value, 256 rows side by
// side, as the threads that hold a row each write it; here a lane has a row and a
// warp an eighth of its values, and the results change places in shared memory.
template <uint32_t Q, int DP>
__global__ void __launch_bounds__(256) kv_join_tiles_kernel(const __grid_constant__ KvAttendArgs k, const KvTilePlan plan) {
  using T = typename KvElem<Q>::type;
  constexpr int kValues = DP / 8;  // of a warp
  __shared__ float rows[32][DP + 1];
  wait_for_previous_kernel();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t cta = blockIdx.x;
  int64_t span;
  const KvSpan next = find_span(k, plan, cta + 1, &span);
  if (next.seq >= int32_t(k.a.n_seqs) || next.unit == 0) return;
  const int64_t at = (cta + 1) * span - next.unit;  // where the item begins
  if (at / span != cta) return;
  const KvSeq s = kv_sequence(k, uint32_t(next.seq));
  const int32_t group = int32_t(k.a.q_heads / k.cache.heads);
  const int32_t row0 = next.tile * kTileRows, count = min(kTileRows, s.n * group - row0);
  const KvSplit split =
      item_split(at, tile_units(kv_row_begin(k, s, row0 / group) & -kTileKeys, kv_row_end(k, s, (row0 + count - 1) / group)), span);
  const int32_t first = int32_t(blockIdx.y) * 32;
  if (first >= count) return;
  const float* parts = reinterpret_cast<const float*>(reinterpret_cast<const char*>(k.a.workspace) + plan.parts_at) + first + lane;
  float top = -INFINITY, sum = 0.0f, o[kValues];
#pragma unroll
  for (int x = 0; x < kValues; ++x) o[x] = 0.0f;
  for (int64_t p = split.first; p <= split.last; ++p) {
    const float* part = parts + part_slot(at, p, span) * kTileRows * (DP + 2);
    float v[kValues];
    const float m = part[0], l = part[kTileRows];
#pragma unroll
    for (int x = 0; x < kValues; ++x) v[x] = part[(2 + warp * kValues + x) * kTileRows];
    const float now = fmaxf(top, m), base = now == -INFINITY ? 0.0f : now;
    const float keep = exp2f(top - base), by = exp2f(m - base);
    sum = sum * keep + l * by;
#pragma unroll
    for (int x = 0; x < kValues; ++x) o[x] = o[x] * keep + v[x] * by;
    top = now;
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
  for (int x = 0; x < kValues; ++x) rows[lane][warp * kValues + x] = o[x] * inv;
  if (warp == 0 && k.a.lse && first + lane < count) {
    const int32_t row = row0 + first + lane, i = row / group;
    reinterpret_cast<float*>(k.a.lse)[(int64_t(s.first) + i) * k.a.q_heads + next.head * group + row - i * group] =
        sum == 0.0f ? -INFINITY : (top + log2f(sum)) * kLn2;
  }
  __syncthreads();
  for (int r = warp; r < 32 && first + r < count; r += 8) {
    const int32_t row = row0 + first + r, i = row / group;
    T* out = reinterpret_cast<T*>(k.a.out.data) + (int64_t(s.first) + i) * k.a.out.token_stride +
             int64_t(next.head * group + row - i * group) * k.a.out.head_stride;
    if (lane * 4 < int(k.cache.head_dim)) {
      KvPack<T, 4> y;
#pragma unroll
      for (int x = 0; x < 4; ++x) y.v[x] = kv_from_float<Q>(rows[r][lane * 4 + x]);
      *reinterpret_cast<KvPack<T, 4>*>(out + lane * 4) = y;
    }
  }
}

template <typename... A>
cudaError_t launch_early(void (*kernel)(A...), dim3 grid, int threads, size_t shm, cudaStream_t stream, A... args) {
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = shm;
  cfg.stream = stream;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// The rows of a block as TMA sees them: [blocks][heads][tokens][values], boxes of
// up to 128 tokens x 64 values in the operands' swizzle. False: copied instead.
bool box_map(const pf_kv_cache& c, const pf_kv_side& s, CUtensorMap* map) {
  using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static const Encode encode = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult found{};
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess) {
      cudaGetLastError();
      f = nullptr;
    }
    return reinterpret_cast<Encode>(f);
  }();
  if (!encode) return false;
  const uint32_t rows = std::min<uint32_t>(c.block_size, kTileKeys);
  const cuuint64_t dims[4] = {c.head_dim, c.block_size, c.heads, c.num_blocks};
  // An axis of one element may have any stride; the map wants a real one.
  auto stride = [](int64_t elements, uint64_t n) { return n > 1 ? cuuint64_t(elements) * 2 : cuuint64_t(16); };
  const cuuint64_t strides[3] = {stride(s.token_stride, c.block_size), stride(s.head_stride, c.heads),
                                 stride(s.block_stride, c.num_blocks)};
  for (cuuint64_t x : strides) {
    if (x == 0 || x >= (1ull << 40)) return false;
  }
  const cuuint32_t box[4] = {64, rows, 1, 1}, steps[4] = {1, 1, 1, 1};
  return encode(map, c.dtype == PF_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                reinterpret_cast<void*>(s.data), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <uint32_t Q, uint32_t STORE, int DP>
cudaError_t launch_as(const KvAttendArgs& k, const KvTilePlan& p, cudaStream_t stream) {
  const auto kernel = kv_attend_tiles_kernel<Q, STORE, DP>;
  const size_t shm = sizeof(typename Tiles<Q, STORE, DP>::Shared) + 1024;
  static_assert(sizeof(typename Tiles<Q, STORE, DP>::Shared) + 1024 <= 227 * 1024, "tile kernel shared memory");
  cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(shm));
  if (err != cudaSuccess) return err;
  KvBoxMaps maps{};
  KvTilePlan plan = p;
  if (Tiles<Q, STORE, DP>::kQuant || !box_map(k.cache, k.cache.key, &maps.key) || !box_map(k.cache, k.cache.value, &maps.value)) {
    plan.box_rows = 0;
  }
  kv_tile_costs_kernel<<<1, 1024, 0, stream>>>(k, p);
  if ((err = cudaGetLastError()) != cudaSuccess) return err;
  if ((err = launch_early(kernel, dim3(p.ctas), Tiles<Q, STORE, DP>::kThreads, shm, stream, k, plan, maps)) != cudaSuccess) return err;
  return launch_early(kv_join_tiles_kernel<Q, DP>, dim3(p.ctas, kTileRows / 32), 256, 0, stream, k, p);
}

template <uint32_t Q, uint32_t STORE>
cudaError_t launch_dims(const KvAttendArgs& k, const KvTilePlan& p, cudaStream_t stream) {
  return k.cache.head_dim <= 64 ? launch_as<Q, STORE, 64>(k, p, stream) : launch_as<Q, STORE, 128>(k, p, stream);
}

template <uint32_t Q>
cudaError_t launch_store(const KvAttendArgs& k, const KvTilePlan& p, cudaStream_t stream) {
  switch (k.cache.dtype) {
    case PF_DTYPE_E4M3: return launch_dims<Q, PF_DTYPE_E4M3>(k, p, stream);
    case PF_DTYPE_INT8: return launch_dims<Q, PF_DTYPE_INT8>(k, p, stream);
    default: return launch_dims<Q, Q>(k, p, stream);
  }
}

}  // namespace

KvTilePlan tile_plan(const KvAttendArgs& k, int num_sms) {
  KvTilePlan p{};
  p.ctas = uint32_t(num_sms);
  const uint32_t page = k.cache.block_size;
  p.page_shift = page_shift(k.cache);
  // Boxes of whole swizzle groups (8 rows) that tile 128 rows.
  p.box_rows = page % kTileKeys == 0 ? kTileKeys : page >= 8 && kTileKeys % page == 0 ? page : 0;
  auto take = [&p](uint64_t bytes) {
    const uint64_t at = p.bytes;
    p.bytes += (bytes + 255) / 256 * 256;
    return at;
  };
  p.costs_at = take((uint64_t(k.a.n_seqs) + 1) * sizeof(int64_t));
  const uint64_t dp = k.cache.head_dim <= 64 ? 64 : 128;
  p.parts_at = take(2 * uint64_t(p.ctas) * kTileRows * (dp + 2) * sizeof(float));
  return p;
}

cudaError_t launch_attend_tiles(const KvAttendArgs& k, const KvTilePlan& p, cudaStream_t stream) {
  return k.a.dtype == PF_DTYPE_BF16 ? launch_store<PF_DTYPE_BF16>(k, p, stream) : launch_store<PF_DTYPE_FP16>(k, p, stream);
}

}  // namespace pf
