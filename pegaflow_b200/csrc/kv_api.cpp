// pf_kv_* entry points: argument checks, then one launcher each.
#include <cuda_runtime.h>

#include <climits>
#include <cmath>
#include <mutex>
#include <string>

#include "common.h"
#include "kv_ops.h"

namespace pf {
namespace {

[[noreturn]] void refuse(const std::string& msg) { throw invalid_argument(msg); }

void check_side(const pf_kv_cache& c, const pf_kv_side& s, const char* name) {
  const std::string n = name;
  if (!s.data) refuse(n + " cache has no address");
  if (s.data % kv_dtype_bytes(c.dtype)) refuse(n + " cache address is not aligned to its elements");
  if (s.block_stride < 0 || s.token_stride < 0 || s.head_stride < 0 || s.scale_block_stride < 0 || s.scale_token_stride < 0 ||
      s.scale_head_stride < 0) {
    refuse(n + " cache has a negative stride");
  }
  if (kv_quantised(c.dtype)) {
    if (!s.scale) refuse(n + " cache of 8 bits needs scales");
    if (s.scale % 4) refuse(n + " scale address is not aligned to 4 bytes");
  }
}

void check_cache(const pf_kv_cache& c) {
  if (c.dtype == PF_DTYPE_FP32 || c.dtype > PF_DTYPE_INT8) refuse("cache dtype must be bf16, fp16, e4m3 or int8");
  if (!c.num_blocks || !c.block_size || !c.heads) refuse("cache must have blocks, tokens and heads");
  if (c.num_blocks > INT32_MAX) refuse("cache has more blocks than an int32 can name");
  if (c.block_size > (1u << 20) || c.heads > (1u << 14)) refuse("cache block_size or heads out of range");
  if (!c.head_dim || c.head_dim > kKvMaxHeadDim) refuse("head_dim must be 1 to 256");
  check_side(c, c.key, "key");
  check_side(c, c.value, "value");
}

void check_rows(const pf_kv_rows& r, uint32_t dtype, const char* name) {
  if (!r.data) refuse(std::string(name) + " has no address");
  if (r.data % kv_dtype_bytes(dtype)) refuse(std::string(name) + " address is not aligned to its elements");
  if (r.token_stride < 0 || r.head_stride < 0) refuse(std::string(name) + " has a negative stride");
}

// Rows that are written: each in a place of its own.
void check_results(const pf_kv_rows& r, uint32_t dtype, uint64_t n, uint64_t heads, const char* name) {
  check_rows(r, dtype, name);
  if ((n > 1 && !r.token_stride) || (heads > 1 && !r.head_stride)) refuse(std::string(name) + " has rows that share their place");
}

bool aligned_rows(uint64_t data, int64_t a, int64_t b, int64_t c, uint32_t elt) {
  const int64_t step = 16 / elt;
  return data % 16 == 0 && a % step == 0 && b % step == 0 && c % step == 0;
}

void check_attention(const pf_kv_cache& c, const pf_kv_attention& a) {
  check_cache(c);
  if (a.dtype != PF_DTYPE_BF16 && a.dtype != PF_DTYPE_FP16) refuse("query must be bf16 or fp16");
  if (!kv_quantised(c.dtype) && c.dtype != a.dtype) refuse("a 16-bit cache must have the query's type");
  if (c.head_dim % 16 || c.head_dim > kKvMaxAttentionDim) refuse("attention head_dim must be a multiple of 16 up to 128");
  if (!a.q_heads || a.q_heads % c.heads) refuse("query heads must be a multiple of the cache's heads");
  if (a.q_heads > (1u << 16)) refuse("query heads out of range");
  if (a.n_tokens > INT32_MAX / 2 || a.n_tokens * a.q_heads > kKvMaxRows) refuse("too many query tokens");
  if (uint64_t(a.n_seqs) * c.heads > INT32_MAX / 2 || a.max_blocks > INT32_MAX) refuse("too many sequences or blocks");
  if (uint64_t(a.max_blocks) * c.block_size > kKvMaxTokens) refuse("block table names more tokens than an int32 can count");
  if (!std::isfinite(a.scale)) refuse("scale must be finite");
  const uint32_t elt = kv_dtype_bytes(c.dtype);
  if (!aligned_rows(c.key.data, c.key.block_stride, c.key.token_stride, c.key.head_stride, elt) ||
      !aligned_rows(c.value.data, c.value.block_stride, c.value.token_stride, c.value.head_stride, elt)) {
    refuse("attention needs cache rows aligned to 16 bytes");
  }
}

int num_sms(int device) {
  static std::mutex mu;
  static int sms[64] = {0};
  std::lock_guard<std::mutex> g(mu);
  if (device < 0 || device >= 64) refuse("device id out of range");
  if (!sms[device]) cuda_check(cudaDeviceGetAttribute(&sms[device], cudaDevAttrMultiProcessorCount, device), "cudaDeviceGetAttribute");
  return sms[device];
}

}  // namespace
}  // namespace pf

namespace {
int null_arg(const char* what) {
  pf::set_last_error(std::string("invalid argument: null ") + what);
  return PF_ERR_INVALID_ARGUMENT;
}
}  // namespace

extern "C" {

int pf_kv_write(int32_t device_id, const pf_kv_cache* cache, uint64_t key, int64_t key_token_stride,
                int64_t key_head_stride, uint64_t value, int64_t value_token_stride, int64_t value_head_stride,
                uint32_t dtype, const int64_t* slots, uint64_t n, int given_scales, int32_t* status, void* stream) {
  if (!cache) return null_arg("cache");
  return pf::guarded([&] {
    using namespace pf;
    check_cache(*cache);
    if (dtype > PF_DTYPE_FP32) refuse("rows must be bf16, fp16 or fp32");
    if (given_scales && !kv_quantised(cache->dtype)) refuse("a 16-bit cache has no scales to be given");
    if (!given_scales && kv_quantised(cache->dtype)) {
      for (const pf_kv_side* s : {&cache->key, &cache->value}) {
        if ((cache->num_blocks > 1 && !s->scale_block_stride) || (cache->block_size > 1 && !s->scale_token_stride) ||
            (cache->heads > 1 && !s->scale_head_stride)) {
          refuse("shared scales cannot be written for each token: pass given_scales");
        }
      }
    }
    if (n > INT32_MAX || n * cache->heads > UINT32_MAX) refuse("too many tokens");
    if (!n) return;
    const pf_kv_rows k{key, key_token_stride, key_head_stride}, v{value, value_token_stride, value_head_stride};
    check_rows(k, dtype, "key");
    check_rows(v, dtype, "value");
    for (const pf_kv_side* s : {&cache->key, &cache->value}) {
      if ((cache->num_blocks > 1 && !s->block_stride) || (cache->block_size > 1 && !s->token_stride) ||
          (cache->heads > 1 && !s->head_stride)) {
        refuse("a cache whose rows share their place cannot be written");
      }
    }
    if (!slots) refuse("no slots");
    DeviceGuard g(device_id);
    const KvWriteArgs args{*cache, k, v, slots, n, status, dtype, given_scales ? 1u : 0u, uint32_t(num_sms(device_id))};
    cuda_check(launch_kv_write(args, static_cast<cudaStream_t>(stream)), "kv_write launch");
  });
}

int pf_kv_read(int32_t device_id, const pf_kv_cache* cache, const int32_t* block_table, int64_t table_stride,
               uint32_t max_blocks, uint32_t n_seqs, const int32_t* starts, uint64_t key, int64_t key_token_stride,
               int64_t key_head_stride, uint64_t value, int64_t value_token_stride, int64_t value_head_stride,
               uint32_t dtype, uint64_t n_rows, int32_t* status, void* stream) {
  if (!cache) return null_arg("cache");
  return pf::guarded([&] {
    using namespace pf;
    check_cache(*cache);
    if (dtype > PF_DTYPE_FP32) refuse("rows must be bf16, fp16 or fp32");
    if (n_rows > INT32_MAX || n_rows * cache->heads > UINT32_MAX) refuse("too many rows");
    if (n_seqs > INT32_MAX / 2) refuse("too many sequences");
    if (!n_rows || !n_seqs) return;
    if (uint64_t(max_blocks) * cache->block_size > kKvMaxTokens) refuse("block table names more tokens than an int32 can count");
    const pf_kv_rows k{key, key_token_stride, key_head_stride}, v{value, value_token_stride, value_head_stride};
    check_results(k, dtype, n_rows, cache->heads, "key");
    check_results(v, dtype, n_rows, cache->heads, "value");
    if ((!block_table && max_blocks) || !starts) refuse("no block table or starts");
    DeviceGuard g(device_id);
    const KvReadArgs args{*cache, k, v, block_table, starts, status, table_stride, n_rows, max_blocks, n_seqs, dtype, uint32_t(num_sms(device_id))};
    cuda_check(launch_kv_read(args, static_cast<cudaStream_t>(stream)), "kv_read launch");
  });
}

int pf_kv_attention_workspace(int32_t device_id, const pf_kv_cache* cache, const pf_kv_attention* args,
                              uint64_t* out_bytes) {
  if (!cache || !args || !out_bytes) return null_arg("cache, arguments or result");
  return pf::guarded([&] {
    using namespace pf;
    check_attention(*cache, *args);
    *out_bytes = kv_attention_workspace(KvAttendArgs{*cache, *args}, num_sms(device_id));
  });
}

int pf_kv_attention_run(int32_t device_id, const pf_kv_cache* cache, const pf_kv_attention* args, void* stream) {
  if (!cache || !args) return null_arg("cache or arguments");
  return pf::guarded([&] {
    using namespace pf;
    check_attention(*cache, *args);
    const pf_kv_attention& a = *args;
    if (!a.n_tokens || !a.n_seqs) return;
    check_rows(a.query, a.dtype, "query");
    check_results(a.out, a.dtype, a.n_tokens, a.q_heads, "out");
    const uint32_t elt = kv_dtype_bytes(a.dtype);
    if (!aligned_rows(a.query.data, a.query.token_stride, a.query.head_stride, 0, elt) ||
        !aligned_rows(a.out.data, a.out.token_stride, a.out.head_stride, 0, elt)) {
      refuse("attention needs query and out rows aligned to 16 bytes");
    }
    if (!a.q_start || !a.kv_len || (a.max_blocks && !a.block_table)) refuse("no q_start, kv_len or block table");
    const KvAttendArgs k{*cache, a};
    const int sms = num_sms(device_id);
    if (a.workspace % 16 || a.workspace_bytes < kv_attention_workspace(k, sms) ||
        (a.workspace_bytes && !a.workspace)) {
      refuse("attention workspace is too small or not aligned to 16 bytes");
    }
    if (a.out.data == a.query.data) refuse("out cannot be the query: rows are read again after others are written");
    DeviceGuard g(device_id);
    cuda_check(launch_kv_attention(k, sms, static_cast<cudaStream_t>(stream)), "kv_attention launch");
  });
}

}  // extern "C"
