// v = s_e x P_e row by row on the CUDA cores, for requests of few rows; and the layout of 16-bit
// operands that lie where the tensor-core kernels cannot read them.
#include "cf_adapter_dev.cuh"

namespace cf {
namespace adapter {
namespace {

// v for rows whose requests are short (a tile of the tensor cores would hold few rows of each):
// one CTA per row and kRows columns of v.  Behind the rows, CTAs that plan row tiles.
constexpr int kRowThreads = 256;
template <bool kSub>
constexpr int kRowCols = kSub ? 16 : kRowThreads / 32;
static_assert(kMaxRowRank <= 65535 * kRowCols<false> && kMaxRowRank <= 65535 * kRowCols<true>, "a grid's rows");

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
  // the request: the first that ends behind the row, if the row is any request's
  const int64_t q = warp_search(0, p.Q, [&](int64_t i) { return p.offsets[i + 1] > t; });
  const int e = q < p.Q && p.offsets[q] <= t ? adapter_of(p, q) : kNone, rank = rank_of(p, e);
  const int r0 = blockIdx.y * kRowCols<kSub>;
  if (r0 >= rank) return;
  const T* x = (const T*)p.x + t * p.x_rs;
  const T* P = (const T*)p.P + e * p.p_es;
  if constexpr (kSub) {  // rows of r: 16 columns x 16 steps of k at a time
    __shared__ float sums[kRowThreads / 32][16];
    const int K = (int)p.K;
    float v = 0.0f;
    if (p.p_vec && p.R % 8 == 0 && sizeof(T) == 2) {  // eight columns a load, two threads a row
      constexpr int kBatch = 8, kRows = kRowThreads / 2;
      static_assert((kBatch + 1) * kRows <= kMaxStep, "k stays an int");
      const int c = (threadIdx.x & 1) * 8;
      const bool in = r0 + c < p.R;
      const T* at = P + r0 + c;
      float acc[8] = {};
      for (int k = threadIdx.x >> 1; k < K; k += kBatch * kRows) {
        uint4 d[kBatch];
        T xv[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const bool ok = in && k + i * kRows < K;
          d[i] = ok ? *(const uint4*)(at + (int64_t)(k + i * kRows) * p.p_ks) : make_uint4(0, 0, 0, 0);
          xv[i] = ok ? x[k + i * kRows] : from_f32<T>(0.0f);
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i)
#pragma unroll
          for (int j = 0; j < 8; ++j) acc[j] = fmaf(to_f32(xv[i]), to_f32(((const T*)&d[i])[j]), acc[j]);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
#pragma unroll
        for (int off = 16; off > 1; off >>= 1) acc[j] += __shfl_xor_sync(0xffffffffu, acc[j], off);
        if (lane < 2) sums[warp][lane * 8 + j] = acc[j];
      }
    } else {
      const int r = r0 + (threadIdx.x & 15);
      float acc = 0.0f;
      if (r < rank) {
#pragma unroll 8
        for (int k = threadIdx.x >> 4; k < K; k += kRowThreads / 16)
          acc = fmaf(to_f32(x[k]), to_f32(P[k * p.p_ks + r]), acc);
      }
      acc += __shfl_xor_sync(0xffffffffu, acc, 16);
      if (lane < 16) sums[warp][lane] = acc;
    }
    __syncthreads();
    const int r = r0 + threadIdx.x;
    if (threadIdx.x < 16 && r < rank) {
      for (int i = 0; i < kRowThreads / 32; ++i) v += sums[i][threadIdx.x];
      store_v(p, t, r, p.scale[e] * v);
    }
  } else {  // rows of k: a warp a column
    constexpr int E = 16 / sizeof(T);
    const int r = r0 + warp;
    if (r >= rank) return;
    P += r * p.p_rs;
    float acc = 0.0f;
    const int K = (int)p.K;
    int k = lane * E;
    if (p.x_vec && p.p_vec) {  // kBatch pairs of loads in flight
      constexpr int kBatch = 8;
      static_assert((kBatch + 1) * 32 * E <= kMaxStep, "k stays an int");
      for (; k + (kBatch - 1) * 32 * E + E <= K; k += kBatch * 32 * E) {
        uint4 a[kBatch], b[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          a[i] = *(const uint4*)(x + k + i * 32 * E);
          b[i] = *(const uint4*)(P + k + i * 32 * E);
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const T *u = (const T*)&a[i], *v = (const T*)&b[i];
#pragma unroll
          for (int j = 0; j < E; ++j) acc = fmaf(to_f32(u[j]), to_f32(v[j]), acc);
        }
      }
    }
    for (; k < K; k += 32 * E) {
      alignas(16) T a[E], b[E];
      *(uint4*)a = load16<T>(x, k, K, p.x_vec);
      *(uint4*)b = load16<T>(P, k, K, p.p_vec);
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

// 16 bytes of a copy at a time: rows padded with zeros to a multiple of 8 elements, for TMA.  Eight
// 2-byte loads of neighbouring addresses a thread (4095 x 4096: 33 MB in 15 us).
__global__ void __launch_bounds__(kRowThreads) k_adapter_pack(const Pack pack) {
  for (int i = 0; i < pack.n; ++i) {
    const Pack::Item& it = pack.item[i];
    const int64_t row_chunks = it.dst_rs / 8, chunks = it.entries * it.rows * row_chunks;
    for (int64_t c = (int64_t)blockIdx.x * kRowThreads + threadIdx.x; c < chunks; c += (int64_t)gridDim.x * kRowThreads) {
      const int64_t row = c / row_chunks, col = (c - row * row_chunks) * 8;
      const int64_t e = row / it.rows, r = row - e * it.rows;
      const uint16_t* src = (const uint16_t*)it.src + e * it.src_es + r * it.src_rs + col;
      alignas(16) uint16_t d[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) d[k] = col + k < it.cols ? src[k] : (uint16_t)0;
      *(uint4*)((uint16_t*)it.dst + c * 8) = *(const uint4*)d;
    }
  }
}

}  // namespace

cf_status launch_pack(const Pack& pack, cudaStream_t st) {
  if (pack.n == 0) return CF_OK;
  int64_t chunks = 0;
  for (int i = 0; i < pack.n; ++i) {
    const Pack::Item& it = pack.item[i];
    const int64_t c = it.entries * it.rows * (it.dst_rs / 8);
    chunks = c > chunks ? c : chunks;
  }
  int64_t blocks = ceil_div(chunks, kRowThreads);
  if (blocks > 148 * 8) blocks = 148 * 8;
  k_adapter_pack<<<(unsigned)blocks, kRowThreads, 0, st>>>(pack);
  return check_launch("k_adapter_pack");
}

cf_status launch_row_shrink(const Problem& p, int dtype, bool substitute, int whole, cudaStream_t st) {
  if (dtype == CF_F32) return substitute ? run<float, true>(p, whole, st) : run<float, false>(p, whole, st);
  if (dtype == CF_BF16)
    return substitute ? run<__nv_bfloat16, true>(p, whole, st) : run<__nv_bfloat16, false>(p, whole, st);
  return substitute ? run<__half, true>(p, whole, st) : run<__half, false>(p, whole, st);
}

}  // namespace adapter
}  // namespace cf
