// Element types of the operators that take float32, bfloat16 or float16 data: loads to
// float32, stores rounded once to nearest even.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

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
