// The adapter product for a few rows, on the CUDA cores: the weights are read once, at the memory's
// rate, and a tile of the tensor cores would be filled by few rows (one row of 4096 x 4096
// float32: the tiles took 38 us, this 8; bfloat16 11 and 5.4, from the L2 cache; memory gives 33 MB in 5.2).
//
//   project:    M = W^T, rows of k.  A CTA has four columns; its eight warps share the contraction.
//   substitute: M = W, rows of n, float32.  A CTA has 32 columns, eight lanes of 16 bytes a row of W;
//               its warps, and the CTAs of a cluster, share the contraction.
//
// Up to kRows rows of x at a time (more in further CTAs, which find the weights in L2).  Every sum
// is one of float32 FMAs in a fixed order.  v Q_e is added at the end, behind the shrink kernel.
#include <cooperative_groups.h>

#include <type_traits>

#include "cf_adapter_dev.cuh"

namespace cg = cooperative_groups;

namespace cf {
namespace adapter {
namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kCols = 4;    // of a CTA, project
constexpr int kSubCols = 32;  // of a CTA, substitute: eight lanes of 16 bytes
constexpr int kMaxSplit = 8;  // CTAs of a cluster, substitute

// y[t, n] = sum + bias + v[t] Q_e[:, n]
template <typename T, bool kSub>
__device__ __forceinline__ void finish(const Problem& p, int64_t t, int64_t n, float sum) {
  if (t >= p.T || n >= p.N || !is_owned(p, t)) return;
  if (p.bias) sum += to_f32(((const T*)p.bias)[n]);
  if (p.R > 0) {
    const int e = adapter_of(p, request_of(p, t)), rank = rank_of(p, e);
    const float* v = p.v + t * p.v_rs;
    const T* q = (const T*)p.Qm + e * p.q_es + n * p.q_ns;
    int r = 0;
    if constexpr (!kSub) {
      constexpr int E = 16 / sizeof(T);
      if (p.q_vec)
#pragma unroll 2
        for (; r + E <= rank; r += E) {
          const uint4 d = *(const uint4*)(q + r);
#pragma unroll
          for (int i = 0; i < E; ++i) sum = fmaf(v[r + i], to_f32(((const T*)&d)[i]), sum);
        }
    }
#pragma unroll 4
    for (; r < rank; ++r) sum = fmaf(v[r], to_f32(q[r * p.q_rs]), sum);
  }
  ((T*)p.y)[t * p.y_rs + n] = from_f32<T>(sum);
}

template <typename T, int kRows>
__global__ void __launch_bounds__(kThreads) k_adapter_gemv(const Problem p, int dependent) {
  constexpr int E = 16 / sizeof(T);
  __shared__ float part[kWarps][kRows * kCols];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t n0 = (int64_t)blockIdx.x * kCols, t0 = (int64_t)blockIdx.y * kRows;
  const int K = (int)p.K;
  const T* M = (const T*)p.M;
  float acc[kRows][kCols] = {};
  // warp w takes every eighth 16-byte chunk group of 32
  auto chunk = [&](int k, auto whole) {
    uint4 m[kCols], x[kRows];
#pragma unroll
    for (int c = 0; c < kCols; ++c)
      m[c] = n0 + c < p.N ? (decltype(whole)::value ? *(const uint4*)(M + (n0 + c) * p.m_ns + k)
                                                    : load16<T>(M + (n0 + c) * p.m_ns, k, K, false))
                          : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int r = 0; r < kRows; ++r)
      x[r] = t0 + r < p.T ? (decltype(whole)::value ? *(const uint4*)((const T*)p.x + (t0 + r) * p.x_rs + k)
                                                    : load16<T>((const T*)p.x + (t0 + r) * p.x_rs, k, K, false))
                          : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < E; ++i)
#pragma unroll
      for (int r = 0; r < kRows; ++r)
#pragma unroll
        for (int c = 0; c < kCols; ++c)
          acc[r][c] = fmaf(to_f32(((const T*)&x[r])[i]), to_f32(((const T*)&m[c])[i]), acc[r][c]);
  };
  constexpr int step = kThreads * E;
  static_assert(step + E <= kMaxStep, "k stays an int");
  int k = threadIdx.x * E;
  if (p.x_vec && p.m_vec) {
#pragma unroll 4
    for (; k + E <= K; k += step) chunk(k, std::true_type{});
  }
  for (; k < K; k += step) chunk(k, std::false_type{});
#pragma unroll
  for (int r = 0; r < kRows; ++r)
#pragma unroll
    for (int c = 0; c < kCols; ++c) {
      float v = acc[r][c];
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
      if (lane == 0) part[warp][r * kCols + c] = v;
    }
  __syncthreads();
  if (dependent) dependency_wait();
  if (threadIdx.x < kRows * kCols) {
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) v += part[i][threadIdx.x];
    finish<T, false>(p, t0 + threadIdx.x / kCols, n0 + threadIdx.x % kCols, v);
  }
}

template <int kRows>
__global__ void __launch_bounds__(kThreads) k_adapter_gemv_sub(const Problem p, int split, int dependent) {
  using T = float;
  constexpr int E = 4, kUnroll = kRows <= 2 ? 8 : 4;
  __shared__ float part[kWarps][kRows][kSubCols];
  __shared__ float total[kRows][kSubCols];
  cg::cluster_group cl = cg::this_cluster();
  const int rank = split > 1 ? (int)cl.block_rank() : 0;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t n0 = (int64_t)(blockIdx.x / split) * kSubCols, t0 = (int64_t)blockIdx.y * kRows;
  const int64_t n = n0 + (lane & 7) * E;
  const int K = (int)p.K;
  const int kb = (int)((int64_t)K * rank / split), ke = (int)((int64_t)K * (rank + 1) / split);
  const T *M = (const T*)p.M + n, *x = (const T*)p.x + t0 * p.x_rs;
  const bool vec = p.m_vec && n + E <= p.N;
  float acc[kRows][E] = {};
  constexpr int kStep = kThreads / 8;  // rows of W a turn
  static_assert(kStep * (kUnroll + 1) <= kMaxStep, "k stays an int");
  for (int k0 = kb + warp * 4 + (lane >> 3); k0 < ke; k0 += kStep * kUnroll) {
    uint4 m[kUnroll];
    float w[kUnroll][kRows];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int k = k0 + u * kStep;
#pragma unroll
      for (int r = 0; r < kRows; ++r) w[u][r] = k < ke && t0 + r < p.T ? to_f32(x[r * p.x_rs + k]) : 0.0f;
      m[u] = k < ke ? load16<T>(M + (int64_t)k * p.m_ks, 0, vec ? E : (n < p.N ? p.N - n : 0), vec)
                    : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int r = 0; r < kRows; ++r)
#pragma unroll
        for (int i = 0; i < E; ++i) acc[r][i] = fmaf(w[u][r], to_f32(((const T*)&m[u])[i]), acc[r][i]);
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r)
#pragma unroll
    for (int i = 0; i < E; ++i) {
      float v = acc[r][i];
      v += __shfl_xor_sync(0xffffffffu, v, 8);
      v += __shfl_xor_sync(0xffffffffu, v, 16);
      if (lane < 8) part[warp][r][lane * E + i] = v;
    }
  __syncthreads();
  for (int i = threadIdx.x; i < kRows * kSubCols; i += kThreads) {
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) v += (&part[w][0][0])[i];
    (&total[0][0])[i] = v;
  }
  if (split > 1)
    cl.sync();
  else
    __syncthreads();
  if (dependent) dependency_wait();
  for (int i = rank * kThreads + threadIdx.x; i < kRows * kSubCols; i += split * kThreads) {
    float v = 0.0f;
    for (int s = 0; s < split; ++s) v += (split > 1 ? cl.map_shared_rank(&total[0][0], s) : &total[0][0])[i];
    finish<T, true>(p, t0 + i / kSubCols, n0 + i % kSubCols, v);
  }
  if (split > 1) cl.sync();  // nobody leaves while its part is read
}

template <typename T, bool kSub, int kRows>
cf_status launch(const Problem& p, cudaStream_t st) {
  const int64_t cols = ceil_div(p.N, kSub ? kSubCols : kCols), groups = ceil_div(p.T, kRows);
  // substitute: as many CTAs a column block as make six an SM, 256 rows of W each at least
  int split = 1;
  while (kSub && split < kMaxSplit && cols * groups * split * 2 <= 148 * 6 && p.K >= split * 2 * 256) split *= 2;
  CF_REQUIRE(cols * split <= 0x7fffffff && groups <= 65535, CF_ERR_SHAPE, "k_adapter_gemv: too many columns");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(cols * split), (unsigned)groups);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  int n = 0;
  if (kSub) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = (unsigned)split;
    at[n].val.clusterDim.y = at[n].val.clusterDim.z = 1;
    ++n;
  }
  if (p.R > 0) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = at;
  cfg.numAttrs = n;
  cudaError_t e;
  if constexpr (kSub)
    e = cudaLaunchKernelEx(&cfg, k_adapter_gemv_sub<kRows>, p, split, (int)(p.R > 0));
  else
    e = cudaLaunchKernelEx(&cfg, k_adapter_gemv<T, kRows>, p, (int)(p.R > 0));
  if (e != cudaSuccess) {
    set_error("k_adapter_gemv: %s", cudaGetErrorString(e));
    return CF_ERR_CUDA;
  }
  return check_launch("k_adapter_gemv");
}

template <typename T, bool kSub>
cf_status run(const Problem& p, int dtype, cudaStream_t st) {
  if (p.R > 0) CF_TRY(launch_row_shrink(p, dtype, kSub, 0, st));
  if (p.T <= 1) return launch<T, kSub, 1>(p, st);
  if (p.T <= 2) return launch<T, kSub, 2>(p, st);
  if (p.T <= 4) return launch<T, kSub, 4>(p, st);
  return launch<T, kSub, 8>(p, st);
}

}  // namespace

cf_status launch_gemv(const Problem& p, int dtype, bool substitute, cudaStream_t st) {
  if (dtype == CF_F32) return substitute ? run<float, true>(p, dtype, st) : run<float, false>(p, dtype, st);
  return dtype == CF_BF16 ? run<__nv_bfloat16, false>(p, dtype, st) : run<__half, false>(p, dtype, st);
}

}  // namespace adapter
}  // namespace cf
