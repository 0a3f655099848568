// Paged-cache operators (pf_kv_* in pegaflow.h): what the host entry points
// and the kernels share.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "pegaflow.h"

namespace pf {

constexpr uint32_t kKvMaxHeadDim = 256;
constexpr uint32_t kKvMaxAttentionDim = 128;
// Tokens that a block table's row may name: positions rounded up to tiles still fit an int32.
constexpr uint64_t kKvMaxTokens = (1ull << 31) - (1ull << 16);
// Query rows (tokens times heads) of a call: rounded up to tiles they still fit one as well.
constexpr uint64_t kKvMaxRows = (1ull << 31) - (1ull << 16);
// Smallest scale a quantised row gets: the smallest normal fp32, so that 1 /
// scale is finite and a row of zeros stores zeros.
constexpr float kKvSmallestScale = 1.17549435e-38f;

inline bool kv_quantised(uint32_t dtype) { return dtype == PF_DTYPE_E4M3 || dtype == PF_DTYPE_INT8; }
inline uint32_t kv_dtype_bytes(uint32_t dtype) {
  return dtype == PF_DTYPE_FP32 ? 4 : kv_quantised(dtype) ? 1 : 2;
}

// log2 of the block size, -1 if it is no power of two.
inline int32_t page_shift(const pf_kv_cache& c) {
  for (int32_t i = 0; i < 31; ++i) {
    if (c.block_size == 1u << i) return i;
  }
  return -1;
}

struct KvWriteArgs {
  pf_kv_cache cache;
  pf_kv_rows key;
  pf_kv_rows value;
  const int64_t* slots;
  uint64_t n;
  int32_t* status;
  uint32_t dtype;
  uint32_t given_scales;
  uint32_t num_sms;
};

struct KvReadArgs {
  pf_kv_cache cache;
  pf_kv_rows key;
  pf_kv_rows value;
  const int32_t* block_table;
  const int32_t* starts;
  int32_t* status;
  int64_t table_stride;
  uint64_t n_rows;
  uint32_t max_blocks;
  uint32_t n_seqs;
  uint32_t dtype;
  uint32_t num_sms;
};

struct KvAttendArgs {
  pf_kv_cache cache;
  pf_kv_attention a;
};

cudaError_t launch_kv_write(const KvWriteArgs& args, cudaStream_t stream);
cudaError_t launch_kv_read(const KvReadArgs& args, cudaStream_t stream);

uint64_t kv_attention_workspace(const KvAttendArgs& args, int num_sms);
cudaError_t launch_kv_attention(const KvAttendArgs& args, int num_sms, cudaStream_t stream);

}  // namespace pf
