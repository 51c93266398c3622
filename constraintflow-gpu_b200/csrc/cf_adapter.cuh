// The adapter product as its kernels see it (cf_adapter.cu: entry point, checks and
// workspace; the kernels: cf_adapter_tile.cu, cf_adapter_f32.cu, cf_adapter_rows.cu).
#pragma once
#include "cf_common.cuh"
#include "cf_elem.cuh"

namespace cf {
namespace adapter {

constexpr int kBM = 128;  // rows of a tile
// tile_e: what a tile's rows carry
constexpr int kNone = -1;   // no adapter
constexpr int kMixed = -2;  // several, or one that the tensor cores do not add: row by row

// Element (k, n) of M is at M + k*m_ks + n*m_ns; (k, r) of P_e at P + e*p_es + k*p_ks + r*p_rs;
// (r, n) of Q_e at Qm + e*q_es + r*q_rs + n*q_ns.
struct Problem {
  int64_t T, K, N;
  int32_t R, E;
  int64_t Q;  // requests
  const void *x, *M, *bias, *P, *Qm;
  int64_t x_rs, m_ks, m_ns, p_es, p_ks, p_rs, q_es, q_rs, q_ns;
  const float* scale;
  const int32_t* ranks;
  const int64_t* offsets;
  const int32_t* ids;
  void* y;
  int64_t y_rs;
  // 16-byte loads of x, M, P and Q_e rows are aligned; vector stores of y are
  int32_t x_vec, m_vec, p_vec, q_vec, y_vec;
  // workspace: v [T, v_rs] float32; its halves [T, v_rs] bfloat16 (TMA path); tile_e, tile_q [row tiles]: what
  // the tile's rows carry, and the first request that reaches into it
  float* v;
  __nv_bfloat16 *v_hi, *v_lo;
  int64_t v_rs;
  int32_t *tile_e, *tile_q;
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
  if (q < 0) return kNone;
  const int e = p.ids[q];
  return e >= 0 && e < p.E ? e : kNone;
}

__device__ __forceinline__ int rank_of(const Problem& p, int e) {
  if (e < 0) return 0;
  return p.ranks ? min(max(p.ranks[e], 0), p.R) : p.R;
}

// tile_e and tile_q of row tile m, by one warp.  One adapter for all of the tile's rows can be added by the
// tensor cores: a tile of several would multiply each row with every one of them, and an
// infinity or NaN of one would reach the others' rows.  `whole`: the ranks that the tensor
// cores take are R and the multiples of `whole` (0: none), so that nothing beyond an adapter's
// own rank is multiplied.
__device__ __forceinline__ void plan_tile(const Problem& p, int64_t m, int whole) {
  const int lane = threadIdx.x & 31;
  int lo = INT32_MAX, hi = INT32_MIN;
  for (int i = lane; i < kBM; i += 32) {
    const int64_t t = m * kBM + i;
    const int64_t q = t < p.T ? request_of(p, t) : -1;
    if (q < 0) continue;
    int e = adapter_of(p, q);
    if (rank_of(p, e) == 0) e = kNone;
    lo = min(lo, e);
    hi = max(hi, e);
  }
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  int e = hi < 0 ? kNone : (lo == hi ? lo : kMixed);
  if (e >= 0) {
    const int r = rank_of(p, e);
    if (!(whole > 0 && (r == p.R || r % whole == 0))) e = kMixed;
  }
  int64_t a = 0, b = p.Q;  // the first request that ends behind the tile's start
  while (a < b) {
    const int64_t mid = (a + b) / 2;
    if (p.offsets[mid + 1] > m * kBM)
      b = mid;
    else
      a = mid + 1;
  }
  if (lane == 0) {
    p.tile_e[m] = e;
    p.tile_q[m] = (int32_t)a;
  }
}

__device__ __forceinline__ void store_v(const Problem& p, int64_t t, int r, float v) {
  p.v[t * p.v_rs + r] = v;
  if (p.v_hi) {
    const __nv_bfloat16 hi = __float2bfloat16_rn(v);
    p.v_hi[t * p.v_rs + r] = hi;
    p.v_lo[t * p.v_rs + r] = __float2bfloat16_rn(v - __bfloat162float(hi));
  }
}

__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void dependency_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// 16-bit data (cf_adapter_tile.cu).  tma: 16-byte aligned operands, read by TMA; lowrank_tma: the
// adapters too.  row_shrink: v row by row on the CUDA cores (requests of few rows).
cf_status launch_tiles(const Problem& p, int dtype, bool substitute, bool tma, bool row_shrink, bool lowrank_tma,
                       cudaStream_t st);
// float32 data (cf_adapter_f32.cu)
cf_status launch_f32(const Problem& p, bool substitute, bool row_shrink, cudaStream_t st);
// v row by row, and the plan of the row tiles (cf_adapter_rows.cu)
cf_status launch_row_shrink(const Problem& p, int dtype, bool substitute, int whole, cudaStream_t st);
// the first site at which a bounded device wait gave up since the last call on this device (0: none)
cf_status take_site_tiles(int* site, cudaStream_t st);
cf_status take_site_f32(int* site, cudaStream_t st);

}  // namespace adapter
}  // namespace cf
