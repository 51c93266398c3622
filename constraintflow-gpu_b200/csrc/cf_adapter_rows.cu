// v = s_e x P_e row by row on the CUDA cores, for requests of few rows.
#include "cf_adapter_dev.cuh"

namespace cf {
namespace adapter {
namespace {

// v for rows whose requests are short (a tile of the tensor cores would hold few rows of each):
// one CTA per row and kRows columns of v.  Behind the rows, CTAs that plan row tiles.
constexpr int kRowThreads = 256;
template <bool kSub>
constexpr int kRowCols = kSub ? 16 : kRowThreads / 32;

template <typename T, bool kSub>
__global__ void __launch_bounds__(kRowThreads) k_adapter_shrink_rows(const Problem p, int64_t m_tiles, int whole) {
  launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t t = blockIdx.x;
  if (t >= p.T) {
    const int64_t tile = (t - p.T) * (kRowThreads / 32) + warp;
    if (blockIdx.y == 0 && tile < m_tiles) plan_tile(p, tile, whole);
    return;
  }
  const int e = adapter_of(p, request_of(p, t)), rank = rank_of(p, e);
  const int r0 = blockIdx.y * kRowCols<kSub>;
  if (r0 >= rank) return;
  const T* x = (const T*)p.x + t * p.x_rs;
  const T* P = (const T*)p.P + e * p.p_es;
  if constexpr (kSub) {  // rows of r: 16 columns x 16 steps of k at a time
    __shared__ float sums[kRowThreads / 32][16];
    const int r = r0 + (threadIdx.x & 15);
    float acc = 0.0f;
    if (r < rank) {
#pragma unroll 8
      for (int64_t k = threadIdx.x >> 4; k < p.K; k += kRowThreads / 16)
        acc = fmaf(to_f32(x[k]), to_f32(P[k * p.p_ks + r]), acc);
    }
    acc += __shfl_xor_sync(0xffffffffu, acc, 16);
    if (lane < 16) sums[warp][lane] = acc;
    __syncthreads();
    if (threadIdx.x < 16 && r < rank) {
      float v = 0.0f;
      for (int i = 0; i < kRowThreads / 32; ++i) v += sums[i][threadIdx.x];
      store_v(p, t, r, p.scale[e] * v);
    }
  } else {  // rows of k: a warp a column
    constexpr int E = 16 / sizeof(T);
    const int r = r0 + warp;
    if (r >= rank) return;
    P += r * p.p_rs;
    float acc = 0.0f;
#pragma unroll 4
    for (int64_t k = lane * E; k < p.K; k += 32 * E) {
      alignas(16) T a[E], b[E];
      *(uint4*)a = load16<T>(x, k, p.K, p.x_vec);
      *(uint4*)b = load16<T>(P, k, p.K, p.p_vec);
#pragma unroll
      for (int i = 0; i < E; ++i) acc = fmaf(to_f32(a[i]), to_f32(b[i]), acc);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, off);
    if (lane == 0) store_v(p, t, r, p.scale[e] * acc);
  }
}

template <typename T, bool kSub>
cf_status run(const Problem& p, int whole, cudaStream_t st) {
  const int64_t m_tiles = ceil_div(p.T, kBM), blocks = p.T + ceil_div(m_tiles, kRowThreads / 32);
  CF_REQUIRE(blocks <= 0x7fffffff, CF_ERR_SHAPE, "adapter_matmul: too many rows");
  const dim3 grid((unsigned)blocks, (unsigned)ceil_div(p.R, kRowCols<kSub>));
  k_adapter_shrink_rows<T, kSub><<<grid, kRowThreads, 0, st>>>(p, m_tiles, whole);
  return check_launch("k_adapter_shrink_rows");
}

}  // namespace

cf_status launch_row_shrink(const Problem& p, int dtype, bool substitute, int whole, cudaStream_t st) {
  if (dtype == CF_F32) return substitute ? run<float, true>(p, whole, st) : run<float, false>(p, whole, st);
  if (dtype == CF_BF16)
    return substitute ? run<__nv_bfloat16, true>(p, whole, st) : run<__nv_bfloat16, false>(p, whole, st);
  return substitute ? run<__half, true>(p, whole, st) : run<__half, false>(p, whole, st);
}

}  // namespace adapter
}  // namespace cf
