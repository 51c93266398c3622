// Rows of many requests through an affine layer with per-request low-rank adapters
// (cf_adapter_matmul).  With x [T, K], y [T, N] and, for the rows of a request with adapter e,
//   v = s_e x P_e   [T, R]      P_e: A_e^T (project) or B_e (substitute)
//   y = x M + b + v Q_e         M: W^T or W;  Q_e: B_e^T or A_e
// the shrink kernel writes v to the workspace and the product kernel adds v Q_e to its tile.
#include "cf_common.cuh"
#include "cf_elem.cuh"

namespace cf {
namespace {

// The problem as both kernels see it.  Element (k, n) of M is at M + k*m_ks + n*m_ns; of P_e
// (k, r) at P + e*p_es + k*p_ks + r*p_rs; of Q_e (r, n) at Q + e*q_es + r*q_rs + n*q_ns.
struct Problem {
  int64_t T, K, N;
  int32_t R, E;
  int64_t Q;
  const void *x, *M, *bias, *P, *Qm;
  int64_t x_rs, m_ks, m_ns, p_es, p_ks, p_rs, q_es, q_rs, q_ns;
  const float* scale;
  const int32_t* ranks;
  const int64_t* offsets;
  const int32_t* ids;
  void* y;
  int64_t y_rs;
  float* v;  // [T, R]
};

// The request of row t: -1 for a row of no request.
__device__ __forceinline__ int64_t request_of(const Problem& p, int64_t t) {
  if (t < p.offsets[0] || t >= p.offsets[p.Q]) return -1;
  int64_t lo = 0, hi = p.Q;  // offsets[lo] <= t < offsets[hi]
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) / 2;
    if (p.offsets[mid] <= t)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

__device__ __forceinline__ int adapter_of(const Problem& p, int64_t q) {
  if (q < 0) return -1;
  const int e = p.ids[q];
  return e >= 0 && e < p.E ? e : -1;
}

__device__ __forceinline__ int rank_of(const Problem& p, int e) {
  if (e < 0) return 0;
  return p.ranks ? min(max(p.ranks[e], 0), p.R) : p.R;
}

// one warp per (row, r)
template <typename T>
__global__ void k_adapter_shrink(const Problem p) {
  const int64_t w = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (w >= p.T * p.R) return;
  const int64_t t = w / p.R;
  const int r = (int)(w - t * p.R);
  const int e = adapter_of(p, request_of(p, t));
  if (r >= rank_of(p, e)) return;
  const T* x = (const T*)p.x + t * p.x_rs;
  const T* P = (const T*)p.P + e * p.p_es + r * p.p_rs;
  float acc = 0.0f;
  for (int64_t k = lane; k < p.K; k += 32) acc = fmaf(to_f32(x[k]), to_f32(P[k * p.p_ks]), acc);
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, off);
  if (lane == 0) p.v[w] = p.scale[e] * acc;
}

// 64 x 64 tile of y, 256 threads, 4 x 4 outputs a thread
template <typename T>
__global__ void __launch_bounds__(256) k_adapter_product(const Problem p) {
  __shared__ float sx[16][65], sm[16][65];
  const int64_t t0 = (int64_t)blockIdx.y * 64, n0 = (int64_t)blockIdx.x * 64;
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  float acc[4][4] = {};
  for (int64_t k0 = 0; k0 < p.K; k0 += 16) {
    for (int i = threadIdx.x; i < 64 * 16; i += 256) {
      const int64_t t = t0 + i / 16, k = k0 + i % 16;
      sx[i % 16][i / 16] = t < p.T && k < p.K ? to_f32(((const T*)p.x)[t * p.x_rs + k]) : 0.0f;
      const int64_t n = n0 + i % 64, kk = k0 + i / 64;
      sm[i / 64][i % 64] = n < p.N && kk < p.K ? to_f32(((const T*)p.M)[kk * p.m_ks + n * p.m_ns]) : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sx[k][ty * 4 + i], sm[k][tx + 16 * j], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i) {
    const int64_t t = t0 + ty * 4 + i;
    if (t >= p.T) break;
    const int64_t q = request_of(p, t);
    if (q < 0) continue;
    const int e = adapter_of(p, q), rank = rank_of(p, e);
    for (int j = 0; j < 4; ++j) {
      const int64_t n = n0 + tx + 16 * j;
      if (n >= p.N) break;
      float a = acc[i][j];
      if (p.bias) a += to_f32(((const T*)p.bias)[n]);
      for (int r = 0; r < rank; ++r)
        a = fmaf(p.v[t * p.R + r], to_f32(((const T*)p.Qm)[e * p.q_es + r * p.q_rs + n * p.q_ns]), a);
      ((T*)p.y)[t * p.y_rs + n] = from_f32<T>(a);
    }
  }
}

template <typename T>
cf_status run(const Problem& p, cudaStream_t st) {
  if (p.R > 0 && p.E > 0) {
    const int64_t blocks = ceil_div(p.T * p.R * 32, 256);
    CF_REQUIRE(blocks <= 0x7fffffff, CF_ERR_SHAPE, "adapter_matmul: too many rows");
    k_adapter_shrink<T><<<(unsigned)blocks, 256, 0, st>>>(p);
    CF_TRY(check_launch("k_adapter_shrink"));
  }
  const int64_t gx = ceil_div(p.N, 64), gy = ceil_div(p.T, 64);
  CF_REQUIRE(gx <= 0x7fffffff && gy <= 65535, CF_ERR_SHAPE, "adapter_matmul: too many rows");
  k_adapter_product<T><<<dim3((unsigned)gx, (unsigned)gy), 256, 0, st>>>(p);
  return check_launch("k_adapter_product");
}

int elem_bytes(int dtype) { return dtype == CF_F32 ? 4 : 2; }

cf_status check_layer(const cf_adapter_layer* L) {
  CF_REQUIRE(L, CF_ERR_NULL, "adapter_matmul: NULL layer");
  CF_REQUIRE(L->dtype == CF_F32 || L->dtype == CF_BF16 || L->dtype == CF_F16, CF_ERR_UNSUPPORTED,
             "adapter_matmul: dtype %d", L->dtype);
  CF_REQUIRE(L->n_out >= 0 && L->n_in >= 0 && L->n_adapters >= 0 && L->rank >= 0, CF_ERR_SHAPE,
             "adapter_matmul: negative size");
  CF_REQUIRE(L->n_out <= 0x7fffff00 && L->n_in <= 0x7fffff00, CF_ERR_SHAPE, "adapter_matmul: layer too wide");
  CF_REQUIRE(L->w_rs >= L->n_in, CF_ERR_SHAPE, "adapter_matmul: rows of W overlap");
  if (L->n_adapters > 0 && L->rank > 0)
    CF_REQUIRE(L->a_rs >= L->n_in && L->b_rs >= L->rank && L->a_es >= 0 && L->b_es >= 0, CF_ERR_SHAPE,
               "adapter_matmul: rows of A or B overlap");
  return CF_OK;
}

}  // namespace
}  // namespace cf

using namespace cf;

extern "C" size_t cf_adapter_workspace_bytes(const cf_adapter_layer* L, int32_t, int64_t T, int64_t) {
  if (!L || T <= 0 || L->rank <= 0) return 0;
  return (size_t)T * L->rank * 4;
}

extern "C" cf_status cf_adapter_matmul(const cf_adapter_layer* L, int32_t substitute, int64_t T, const void* x,
                                       int64_t x_rs, int64_t n_requests, const int64_t* offsets, const int32_t* ids,
                                       void* y, int64_t y_rs, void* ws, size_t ws_bytes, void* stream) {
  clear_error();
  CF_INJECT("adapter_matmul");
  CF_TRY(check_layer(L));
  const int64_t K = substitute ? L->n_out : L->n_in, N = substitute ? L->n_in : L->n_out;
  CF_REQUIRE(T >= 0 && n_requests >= 0, CF_ERR_SHAPE, "adapter_matmul: negative size");
  CF_REQUIRE(T <= 1 || (x_rs >= 0 && y_rs >= N), CF_ERR_SHAPE, "adapter_matmul: rows of y overlap");
  if (T == 0 || N == 0 || n_requests == 0) return CF_OK;
  const bool adapters = L->n_adapters > 0 && L->rank > 0;
  CF_REQUIRE(y && offsets && ids && (K == 0 || (x && L->W_dev)), CF_ERR_NULL, "adapter_matmul: NULL argument");
  CF_REQUIRE(!adapters || (L->A_dev && L->B_dev && L->scale_dev), CF_ERR_NULL, "adapter_matmul: NULL adapters");
  const size_t need = cf_adapter_workspace_bytes(L, substitute, T, n_requests);
  CF_REQUIRE(ws_bytes >= need && (need == 0 || ws), CF_ERR_WORKSPACE, "adapter_matmul: workspace of %zu bytes, needs %zu",
             ws_bytes, need);
  CF_REQUIRE((uintptr_t)ws % 16 == 0, CF_ERR_WORKSPACE, "adapter_matmul: unaligned workspace");
  CF_REQUIRE(((uintptr_t)x | (uintptr_t)y | (uintptr_t)L->W_dev | (uintptr_t)L->A_dev | (uintptr_t)L->B_dev |
              (uintptr_t)L->bias_dev) % elem_bytes(L->dtype) == 0,
             CF_ERR_SHAPE, "adapter_matmul: unaligned data");
  Problem p = {};
  p.T = T, p.K = K, p.N = N;
  p.R = adapters ? L->rank : 0, p.E = adapters ? L->n_adapters : 0, p.Q = n_requests;
  p.x = x, p.x_rs = x_rs, p.M = L->W_dev, p.y = y, p.y_rs = y_rs;
  p.scale = L->scale_dev, p.ranks = L->ranks_dev, p.offsets = offsets, p.ids = ids, p.v = (float*)ws;
  if (substitute) {
    p.m_ks = L->w_rs, p.m_ns = 1;
    p.P = L->B_dev, p.p_es = L->b_es, p.p_ks = L->b_rs, p.p_rs = 1;
    p.Qm = L->A_dev, p.q_es = L->a_es, p.q_rs = L->a_rs, p.q_ns = 1;
  } else {
    p.bias = L->bias_dev;
    p.m_ks = 1, p.m_ns = L->w_rs;
    p.P = L->A_dev, p.p_es = L->a_es, p.p_ks = 1, p.p_rs = L->a_rs;
    p.Qm = L->B_dev, p.q_es = L->b_es, p.q_rs = 1, p.q_ns = L->b_rs;
  }
  if (L->dtype == CF_F32) return run<float>(p, as_stream(stream));
  if (L->dtype == CF_BF16) return run<__nv_bfloat16>(p, as_stream(stream));
  return run<__half>(p, as_stream(stream));
}
