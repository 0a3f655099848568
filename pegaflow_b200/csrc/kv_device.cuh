// Device helpers of the paged-cache operators: types, 8-bit codes, addresses.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "kv_ops.h"

namespace pf {

template <uint32_t T> struct KvElem;
template <> struct KvElem<PF_DTYPE_BF16> { using type = __nv_bfloat16; };
template <> struct KvElem<PF_DTYPE_FP16> { using type = __half; };
template <> struct KvElem<PF_DTYPE_FP32> { using type = float; };
template <> struct KvElem<PF_DTYPE_E4M3> { using type = __nv_fp8_storage_t; };
template <> struct KvElem<PF_DTYPE_INT8> { using type = int8_t; };

// N consecutive elements as one or more loads of up to 16 bytes.
template <typename T, int N>
struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) KvPack {
  T v[N];
};

template <uint32_t T>
__device__ __forceinline__ float kv_to_float(typename KvElem<T>::type x) {
  if constexpr (T == PF_DTYPE_BF16) return __bfloat162float(x);
  if constexpr (T == PF_DTYPE_FP16) return __half2float(x);
  if constexpr (T == PF_DTYPE_FP32) return x;
  if constexpr (T == PF_DTYPE_E4M3) return __half2float(__half(__nv_cvt_fp8_to_halfraw(x, __NV_E4M3)));
  if constexpr (T == PF_DTYPE_INT8) return static_cast<float>(x);
}

// Rounds to the type; 8-bit types saturate (the value is already within
// +-qmax, or NaN: E4M3 keeps a NaN, INT8 stores 0 for it).
template <uint32_t T>
__device__ __forceinline__ typename KvElem<T>::type kv_from_float(float x) {
  if constexpr (T == PF_DTYPE_BF16) return __float2bfloat16_rn(x);
  if constexpr (T == PF_DTYPE_FP16) return __float2half_rn(x);
  if constexpr (T == PF_DTYPE_FP32) return x;
  if constexpr (T == PF_DTYPE_E4M3) return __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3);
  if constexpr (T == PF_DTYPE_INT8) return static_cast<int8_t>(x == x ? __float2int_rn(x) : 0);
}

__device__ __forceinline__ void kv_flag(int32_t* status, int32_t bit) {
  if (status) atomicOr(status, bit);
}

// The s in [0, n) with starts[s] <= x < starts[s + 1], or n. Offsets out of
// order give some s or n, never an index outside the array.
__device__ __forceinline__ uint32_t kv_find_seq(const int32_t* starts, uint32_t n, int64_t x) {
  uint32_t lo = 0, hi = n;  // starts[lo] <= x is kept for lo > 0
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) >> 1;
    if (starts[mid] <= x) lo = mid; else hi = mid;
  }
  return starts[lo] <= x && x < starts[lo + 1] ? lo : n;
}

}  // namespace pf
