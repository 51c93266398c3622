// The adapter product as its kernels see it (cf_adapter.cu: entry point, checks and
// workspace; the kernels: cf_adapter_tile.cu,
// cf_adapter_wide.cu, cf_adapter_f32.cu, cf_adapter_rows.cu).
#pragma once
#include "cf_common.cuh"
#include "cf_elem.cuh"

namespace cf {
namespace adapter {

// Widths of a layer: the kernels step an int through the contraction and the columns, at most kMaxStep
// past their end.
constexpr int kMaxStep = 1 << 16, kMaxWidth = 0x7fffffff - kMaxStep;
constexpr int kMaxRowRank = 65535 * 8;  // v row by row: eight columns a CTA, dealt out over gridDim.y
constexpr int kBM = 128;  // rows of a tile
// tile_e: what a tile's rows carry
constexpr int kNone = -1;   // no adapter
constexpr int kMixed = -2;  // several, or one that the tensor cores do not add: row by row
constexpr int kFew = -3;    // several, of at most kFewRequests requests, all of them for the tensor cores
constexpr int kFewRequests = 8;

// Element (k, n) of M is at M + k*m_ks + n*m_ns; (k, r) of P_e at P + e*p_es + k*p_ks + r*p_rs;
// (r, n) of Q_e at Qm + e*q_es + r*q_rs + n*q_ns.
struct Problem {
  int64_t T, K, N;
  int32_t R, E;
  uint32_t max_polls;  // of every bounded wait
  uint32_t withhold;   // 1: the first stage of operands is never released (the failure-path tests)
  int64_t Q;           // requests
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

// Whether row t is some request's.
__device__ __forceinline__ bool is_owned(const Problem& p, int64_t t) {
  return t >= p.offsets[0] && t < p.offsets[p.Q];
}

// The first index in [lo, hi) at which `pred`, false up to some point and true from there on, is
// true, else hi.  A warp together: 32 places a turn, where a binary search would wait for one
// load after the other.
template <typename F>
__device__ __forceinline__ int64_t warp_search(int64_t lo, int64_t hi, F&& pred) {
  const int lane = threadIdx.x & 31;
  while (lo < hi) {
    const int64_t step = (hi - lo + 31) / 32, at = lo + (lane + 1) * step - 1;
    const uint32_t found = __ballot_sync(0xffffffffu, at >= hi - 1 ? at < hi + step && pred(hi - 1) : pred(at));
    if (!found) return hi;  // the last lane in range tried hi - 1
    const int first = __ffs(found) - 1;
    hi = min(lo + (first + 1) * step - 1, hi - 1);
    lo = lo + first * step;
    if (step == 1) return hi;
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

// A lane's request of 32 that may reach into a row tile: its adapter and rank (0: none, or no row of
// the tile) and its rows [a, b) of the tile.
struct Reach {
  int e, r, a, b;
  bool past;  // this request and those behind it start behind the tile
};

__device__ __forceinline__ Reach reach(const Problem& p, int64_t m, int64_t base) {
  const int64_t t0 = m * kBM, t1 = min(t0 + kBM, p.T), q = base + (threadIdx.x & 31);
  Reach w{kNone, 0, 0, 0, true};
  if (q < p.Q) {
    const int64_t o0 = p.offsets[q], o1 = p.offsets[q + 1];
    const int e = adapter_of(p, q);
    w.past = o0 >= t1;
    w.a = (int)(max(o0, t0) - t0);
    w.b = (int)(max(min(o1, t1), t0) - t0);
    if (!w.past && w.a < w.b) {
      w.e = e;
      w.r = rank_of(p, e);
    }
  }
  return w;
}

// f(adapter, rank, first row, end row) for the requests with an adapter that reach into row tile
// m, in order, from request `from` on (the first that ends behind the tile's start; `w`: its and
// the next 31's reach); a warp together, every lane with the same arguments.  f returns false to
// stop.
template <typename F>
__device__ __forceinline__ bool for_requests(const Problem& p, int64_t m, int64_t from, Reach w, F&& f) {
  for (;;) {
    for (uint32_t todo = __ballot_sync(0xffffffffu, w.r > 0); todo; todo &= todo - 1) {
      const int i = __ffs(todo) - 1;
      if (!f(__shfl_sync(0xffffffffu, w.e, i), __shfl_sync(0xffffffffu, w.r, i), __shfl_sync(0xffffffffu, w.a, i),
             __shfl_sync(0xffffffffu, w.b, i)))
        return false;
    }
    if (__any_sync(0xffffffffu, w.past)) return true;
    from += 32;
    w = reach(p, m, from);
  }
}

// tile_e and tile_q of row tile m, by one warp.  One adapter for all of the tile's rows can be added by the
// tensor cores: a tile of several would multiply each row with every one of them, and an
// infinity or NaN of one would reach the others' rows.  `whole`: the ranks that the tensor
// cores take are R and the multiples of `whole` (0: none), so that nothing beyond an adapter's
// own rank is multiplied.
__device__ __forceinline__ void plan_tile(const Problem& p, int64_t m, int whole) {
  // the first request that ends behind the tile's start
  const int64_t from = warp_search(0, p.Q, [&](int64_t q) { return p.offsets[q + 1] > m * kBM; });
  int first = kNone, requests = 0;
  int64_t rows = 0;
  bool one = true, fit = true;
  for_requests(p, m, from, reach(p, m, from), [&](int e, int r, int a, int b) {
    if (requests == 0) first = e;
    one &= e == first;
    fit &= whole > 0 && (r == p.R || r % whole == 0);
    rows += b - a;
    ++requests;
    return true;
  });
  // rows of requests: all of [offsets[0], offsets[Q]) within the tile
  const int64_t t0 = m * kBM, t1 = min(t0 + kBM, p.T);
  const int64_t owned = max(min(p.offsets[p.Q], t1) - max(p.offsets[0], t0), (int64_t)0);
  int e = kMixed;
  if (requests == 0)
    e = kNone;
  else if (fit && one && rows == owned)
    e = first;
  else if (fit && requests <= kFewRequests)
    e = kFew;
  if ((threadIdx.x & 31) == 0) {
    p.tile_e[m] = e;
    p.tile_q[m] = (int32_t)from;
  }
}

// For the tensor cores v is a bfloat16 pair: 16 bits of it, off by 2^-16 at most where the result is
// rounded to 2^-8, for two passes of Q_e (float32 itself would take three).
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

// Copies of 16-bit matrices [entries][rows][cols] with rows of dst_rs elements, a multiple of 8.
struct Pack {
  struct Item {
    const void* src;
    void* dst;
    int64_t entries, rows, cols, src_es, src_rs, dst_rs;
  } item[4];
  int n;
};
cf_status launch_pack(const Pack& pack, cudaStream_t st);  // cf_adapter_rows.cu

// 16-bit data, x and M 16-byte aligned (cf_adapter_tile.cu).  row_shrink: v row by row on the CUDA
// cores (requests of few rows); lowrank_tma: the adapters are 16-byte aligned too, as they must
// be without row_shrink.
cf_status launch_tiles(const Problem& p, int dtype, bool substitute, bool row_shrink, bool lowrank_tma,
                       cudaStream_t st);
// float32 data (cf_adapter_f32.cu)
cf_status launch_f32(const Problem& p, bool substitute, bool row_shrink, cudaStream_t st);
// a few rows, whatever the alignment, with v row by row (cf_adapter_gemv.cu); substitute: float32
cf_status launch_gemv(const Problem& p, int dtype, bool substitute, cudaStream_t st);
// v row by row, and the plan of the row tiles (cf_adapter_rows.cu)
cf_status launch_row_shrink(const Problem& p, int dtype, bool substitute, int whole, cudaStream_t st);
// the first site at which a bounded device wait gave up since the last call on this device (0: none)
cf_status take_site_tiles(int* site, cudaStream_t st);
cf_status take_site_wide(int* site, cudaStream_t st);
cf_status take_site_f32(int* site, cudaStream_t st);

}  // namespace adapter
}  // namespace cf
