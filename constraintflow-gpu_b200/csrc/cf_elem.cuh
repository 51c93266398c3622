// Element types of the operators that take float32, bfloat16 or float16 data: loads to
// float32, stores rounded once to nearest even; and what their entry points share.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <atomic>

#include "cf_common.cuh"

namespace cf {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }

template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) {
  return x;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) {
  return __float2half_rn(x);
}

// Allow `bytes` of dynamic shared memory to a kernel, once a device (`done`: one word a kernel).
template <typename F>
cf_status allow_smem(F* kern, int bytes, std::atomic<uint64_t>& done, const char* what) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  const uint64_t bit = dev < 64 ? (uint64_t)1 << dev : 0;
  if (e == cudaSuccess && !(done.load(std::memory_order_relaxed) & bit)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  }
  CF_REQUIRE(e == cudaSuccess, CF_ERR_CUDA, "%s: cudaFuncSetAttribute: %s", what, cudaGetErrorString(e));
  return CF_OK;
}

// Whether rows of a (at a_rs elements) and rows of b share memory: their ranges do, unless the rows
// lie beside one another at one stride.
inline bool rows_overlap(const void* a, int64_t a_rs, int64_t a_cols, const void* b, int64_t b_rs, int64_t b_cols,
                         int64_t rows, int64_t size) {
  const int64_t d = ((int64_t)(uintptr_t)b - (int64_t)(uintptr_t)a) / size;  // b's place, in elements
  if (d >= (rows - 1) * a_rs + a_cols || -d >= (rows - 1) * b_rs + b_cols) return false;
  if (rows <= 1 || a_rs != b_rs || a_rs <= 0) return true;
  const int64_t at = (d % a_rs + a_rs) % a_rs;
  return at < a_cols || at + b_cols > a_rs;
}

}  // namespace cf
