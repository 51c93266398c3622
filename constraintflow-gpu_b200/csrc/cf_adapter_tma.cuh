// What the TMA kernels of the adapter product share: tensor-map loads, 16-bit MMAs, tensor maps.
#pragma once
#include <cuda.h>

#include "cf_adapter_dev.cuh"

namespace cf {
namespace adapter {

__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], "
      "[%2];" ::"r"(dst),
      "l"(map), "r"(tc::smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// Fetch a tensor map ahead of the first load through it.
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

__device__ __forceinline__ void mma_f16(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// MN-major, 128-byte swizzle: 64 columns (128 B) x 8 contraction steps an atom; groups of 8 steps
// 1024 B apart, blocks of 64 columns 64 steps x 128 B = 8192 B apart.
__device__ __forceinline__ uint64_t mn_desc(uint32_t smem_addr) {
  return (uint64_t)((smem_addr & 0x3FFFFu) >> 4) | ((uint64_t)(8192 >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

struct Maps {
  CUtensorMap x, b, v_hi, v_lo, q;
};

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                             const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeFn encoder() {
  static EncodeFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess) f = nullptr;
    return (EncodeFn)f;
  }();
  return fn;
}

// [z][y][x] of 16-bit elements, x contiguous, boxes of 64 x box_y, 128-byte swizzle, zeros outside
inline cf_status encode(CUtensorMap* map, int dtype, const void* base, int64_t nx, int64_t ny, int64_t nz, int64_t ys,
                 int64_t zs, int box_y) {
  EncodeFn fn = encoder();
  CF_REQUIRE(fn, CF_ERR_CUDA, "adapter_matmul: cuTensorMapEncodeTiled is not available");
  const cuuint64_t dims[3] = {(cuuint64_t)nx, (cuuint64_t)ny, (cuuint64_t)nz};
  const cuuint64_t strides[2] = {(cuuint64_t)ys * 2, (cuuint64_t)(nz > 1 ? zs : ys * ny) * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)box_y, 1}, ones[3] = {1, 1, 1};
  CUresult r = fn(map, dtype == CF_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                  const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  CF_REQUIRE(r == CUDA_SUCCESS, CF_ERR_CUDA, "adapter_matmul: tensor map: error %d", (int)r);
  return CF_OK;
}

// The maps of M and Q_e for tiles of bn columns: n-contiguous ones in boxes of 64 x 64.
inline cf_status encode_weights(const Problem& p, int dtype, bool substitute, int bn, bool q_tma, Maps* maps) {
  if (substitute)
    CF_TRY(encode(&maps->b, dtype, p.M, p.N, p.K, 1, p.m_ks, p.m_ks * p.K, 64));
  else
    CF_TRY(encode(&maps->b, dtype, p.M, p.K, p.N, 1, p.m_ns, p.m_ns * p.N, bn));
  if (!q_tma || p.R == 0) return CF_OK;
  if (substitute) return encode(&maps->q, dtype, p.Qm, p.N, p.R, p.E, p.q_rs, p.q_es, 64);
  return encode(&maps->q, dtype, p.Qm, p.R, p.N, p.E, p.q_ns, p.q_es, bn);
}

// The 16-bit product in 128 x 256 tiles (cf_adapter_wide.cu); maps.x, v_hi and v_lo are set, with
// boxes of x_rows rows.
cf_status launch_wide(const Problem& p, int dtype, bool substitute, Maps maps, bool q_tma, int x_rows,
                      cudaStream_t st);

}  // namespace adapter
}  // namespace cf
