// Tensor-core tiles of the adapter product (cf_adapter.cuh): 128 rows x kBN columns of
// x [M | Q_e], float32 accumulators in TMEM.
//
//   k_adapter_tile<.., kShrink = true>   v = s_e x P_e for the rows of one request in one row tile
//   k_adapter_tile<.., kShrink = false>  y = x M + b + v Q_e
//
// The contraction is dealt out to the CTAs of a cluster (few tiles: one token's product is as
// wide as the weights, so the cluster makes enough CTAs to read them at full bandwidth); the
// parts meet in shared memory, each CTA summing every rank's part of its own rows in rank order.
// A row tile whose rows all carry one adapter takes v Q_e as further steps of the contraction;
// other tiles add it row by row on the CUDA cores, where a row reads its own adapter only.
//
// Operands in shared memory are 128-byte-swizzled images, 128 bytes of the contraction a row:
// loaded by tensor maps; M and Q_e with n contiguous (substitution) stay as they lie, as MN-major
// images.  v is a bfloat16 pair (hi, lo), two passes of the same Q_e.  The accumulator truncates and is kept
// for all of a CTA's steps, as in the wide tiles.
//
// 64 rows of 4096 x 4096, each with its own adapter of rank 16: 19.0 us, 47 MB at 2.5 TB/s: a chain of
// launch, v, weights, sums and the rows' own adapters.  Of these only v Q_e needs v: the adapters' rows
// are still read behind the contraction, not under it.
#include <cooperative_groups.h>

#include "cf_adapter_tma.cuh"

namespace cg = cooperative_groups;

namespace cf {
namespace adapter {
namespace {

using namespace tc;

constexpr int kWorkers = 256;  // warps 0-7: epilogue
constexpr int kProducerWarp = 8, kMmaWarp = 9;
constexpr int kThreads = 320;

// The site at which a bounded wait gave up (cf_adapter_check); kernels only write it.
__device__ int g_err;

struct Tiling {
  int64_t m_tiles, units;  // units: clusters that work on tiles; behind them, clusters that plan tiles
  int32_t split;           // CTAs of a cluster
  int32_t x_rows;          // rows of a TMA box of x
  int32_t whole;           // plan_tile
  int32_t q_tma;           // v Q_e can be a further step of the contraction
  int32_t dependent;       // launched while the shrink kernel may still run
};

template <int kStages>
struct Bars {
  uint64_t full[kStages], empty[kStages], done;
  uint32_t tmem;
  int err;  // the site at which a wait of this CTA gave up: the others follow
};

template <typename T, bool kSub, bool kShrink, int kBN, int kStages>
__global__ void __launch_bounds__(kThreads, 2) k_adapter_tile(const Problem p, const __grid_constant__ Maps maps,
                                                           const Tiling g) {
  constexpr int kStep = Kind<T>::kStep;
  constexpr bool kMn = kSub;  // B images lie n-contiguous
  constexpr uint32_t kABytes = kBM * 128, kBBytes = kBN * 128;
  constexpr uint32_t kStageBytes = kABytes + kBBytes;
  static_assert((kBM * (kBN + 4)) * 4 <= kStageBytes * kStages, "the tile is staged where the operands were");
  extern __shared__ uint8_t smem_raw[];
  __shared__ Bars<kStages> bars;
  // each row's adapter, kMixed for a row of no request, and that adapter's rank
  __shared__ int row_e[kShrink ? 1 : kBM], row_rank[kShrink ? 1 : kBM];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const uint32_t sbase = smem_u32(smem);
  cg::cluster_group cl = cg::this_cluster();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == kProducerWarp * 32) {
    prefetch_map(&maps.x);
    prefetch_map(&maps.b);
  }
  const int split = g.split;
  const int rank = split > 1 ? (int)cl.block_rank() : 0;
  const int64_t unit = blockIdx.x / split;

  // ---- which tile
  int64_t m, n0 = 0, row0 = 0, row1 = 0;  // rows [row0, row1) of the tile are this unit's (shrink)
  int e = kNone, e_rank = 0, r0 = 0;
  if constexpr (kShrink) {
    launch_dependents();
    const int64_t blocks_r = (p.R + kBN - 1) / kBN;
    if (unit >= g.units) {
      const int64_t tile = ((unit - g.units) * split + rank) * (kThreads / 32) + warp;
      if (tile < g.m_tiles) plan_tile(p, tile, g.whole);
      return;
    }
    const int64_t u = unit / blocks_r;
    r0 = (int)(unit - u * blocks_r) * kBN;
    // Units are the steps of the staircase of (tile, request) pairs: tile + request is different
    // for each pair that overlaps.  Request q of unit u: the first that ends behind tile u - q's start.
    const int64_t lo = warp_search(0, p.Q, [&](int64_t q) { return p.offsets[q + 1] + kBM * q > kBM * u; });
    if (lo >= p.Q) return;
    m = u - lo;
    if (m < 0 || m >= g.m_tiles) return;
    row0 = max(p.offsets[lo], m * kBM);
    row1 = min(min(p.offsets[lo + 1], (m + 1) * kBM), p.T);
    e = adapter_of(p, lo);
    e_rank = rank_of(p, e);
    if (row0 >= row1 || e < 0 || r0 >= e_rank) return;  // the whole cluster returns
  } else {
    m = unit % g.m_tiles;
    n0 = unit / g.m_tiles * kBN;
  }
  const int64_t t0 = m * kBM;
  const int rows = (int)min((int64_t)kBM, p.T - t0);
  // columns that the MMAs take, a multiple of 16
  const int cols = kShrink ? min(kBN, (min(p.R - r0, kBN) + 15) / 16 * 16) : kBN;

  const int n_k = (int)((p.K + kStep - 1) / kStep);
  const int kb = (int)((int64_t)n_k * rank / split), ke = (int)((int64_t)n_k * (rank + 1) / split);

  // ---- set-up
  if (warp == kMmaWarp) tmem_alloc(&bars.tmem, kBN < 32 ? 32 : kBN);
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&bars.full[i], 1);
      mbar_init(&bars.empty[i], i == 0 ? 1 + p.withhold : 1);
    }
    mbar_init(&bars.done, 1);
    bars.err = 0;
    fence_mbar_init();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars.tmem;
  int* err = &bars.err;

  // The low-rank steps behind the contraction: only known once the shrink kernel is done.
  auto lowrank_steps = [&](int& te, int& tr) {
    te = kNone, tr = 0;
    if (kShrink || rank != 0 || p.R == 0 || !g.q_tma) return 0;
    dependency_wait();
    te = *(volatile int*)(p.tile_e + m);
    if (te < 0) return 0;
    tr = rank_of(p, te);
    const int steps = (tr + kStep - 1) / kStep;
    return 2 * steps;
  };

  bool ok = true;
  if (warp == kProducerWarp && lane == 0) {
    int it = 0, te, tr;
    auto stage_for = [&](uint32_t bytes) -> int {
      const int s = it % kStages, round = it / kStages;
      if (!mbar_wait(&bars.empty[s], (round & 1) ^ 1, err, 11, p.max_polls)) return -1;
      mbar_arrive_expect_tx(&bars.full[s], bytes);
      ++it;
      return s;
    };
    const uint32_t a_bytes = (uint32_t)g.x_rows * 128;
    // B image: `bcols` columns from column c on, contraction from k on, of map entry z
    auto load_b = [&](uint32_t dst, const CUtensorMap* map, int c, int k, int z, int bcols, uint64_t* bar) {
      if constexpr (kMn) {
        for (int j = 0; j < bcols; j += 64) tma_3d(dst + j * 128, map, c + j, k, z, bar);
      } else {
        tma_3d(dst, map, k, c, z, bar);
      }
    };
    const int bcols = kMn ? (cols + 63) / 64 * 64 : kBN;
    for (int k = kb; k < ke && ok; ++k) {
      const int s = stage_for(a_bytes + bcols * 128);
      if (s < 0) {
        ok = false;
        break;
      }
      const uint32_t a = sbase + s * kStageBytes, b = a + kABytes;
      tma_3d(a, &maps.x, k * kStep, (int)t0, 0, &bars.full[s]);
      load_b(b, &maps.b, (int)(kShrink ? r0 : n0), k * kStep, kShrink ? e : 0, bcols, &bars.full[s]);
    }
    if constexpr (!kShrink) {
      const int extra = ok ? lowrank_steps(te, tr) : 0;
      for (int i = 0; i < extra && ok; ++i) {
        const int s = stage_for(a_bytes + kBN * 128);
        if (s < 0) {
          ok = false;
          break;
        }
        const uint32_t a = sbase + s * kStageBytes, b = a + kABytes;
        const int r = i / 2 * kStep;
        tma_3d(a, i & 1 ? &maps.v_lo : &maps.v_hi, r, (int)t0, 0, &bars.full[s]);
        load_b(b, &maps.q, (int)n0, r, te, kBN, &bars.full[s]);
      }
    }
    // Copies in flight land before shared memory is given up: the others may have given up on them.
    for (int i = max(0, it - kStages); i < it; ++i)
      mbar_wait_drain(&bars.full[i % kStages], (i / kStages) & 1, err, 12);
  } else if (warp == kMmaWarp && lane == 0) {
    int it = 0, te = kNone, tr = 0;
    const uint32_t id = idesc(Kind<T>::kAb, cols, kMn);
    auto step = [&](int k16) -> bool {  // k16: MMAs of this step
      const int s = it % kStages, round = it / kStages;
      if (!mbar_wait(&bars.full[s], round & 1, err, 21, p.max_polls)) return false;
      tc_fence_after();
      const uint32_t a = sbase + s * kStageBytes, b = a + kABytes;
      const uint64_t ad = sw128_desc(a), bd = kMn ? mn_desc(b) : sw128_desc(b);
      constexpr uint64_t kAStep = 32 >> 4, kBStep = kMn ? (16 * 128) >> 4 : 32 >> 4;
      for (int j = 0; j < k16; ++j) {
        const uint32_t acc = it > 0 || j > 0;
        mma_f16(tmem, ad + j * kAStep, bd + j * kBStep, id, acc);
      }
      mma_commit(&bars.empty[s]);
      ++it;
      return true;
    };
    for (int k = kb; k < ke && ok; ++k) ok = step(4);
    if constexpr (!kShrink) {
      const int extra = ok ? lowrank_steps(te, tr) : 0;
      constexpr int kMma = kStep / 4;  // contraction of one MMA
      for (int i = 0; i < extra && ok; ++i) {
        const int r = i / 2 * kStep;
        ok = step((min(tr - r, kStep) + kMma - 1) / kMma);
      }
    }
    mma_commit(&bars.done);
    mbar_wait_drain(&bars.done, 0, err, 22);  // every MMA has run before tensor memory is given up
  }

  // ---- the accumulators, staged in shared memory
  __syncwarp();
  if constexpr (!kShrink) {
    if (warp < 4)
      for (int i = threadIdx.x; i < rows; i += kBM) {
        const int64_t t = t0 + i;
        row_e[i] = !is_owned(p, t) ? kMixed : p.R > 0 ? adapter_of(p, request_of(p, t)) : kNone;
        row_rank[i] = rank_of(p, row_e[i]);
      }
  }
  float* part = (float*)smem;
  constexpr int kLd = kBN + 4;
  int te = kNone;
  if (warp < kProducerWarp) {
    ok = warp_wait(&bars.done, 0, err, 41, p.max_polls);
    tc_fence_after();
    const int row = (warp & 3) * 32 + lane;
    const bool any = kb < ke;  // else the accumulators were never written (or by low-rank steps only)
    bool low = false;
    if (!kShrink && p.R > 0) {
      if (g.dependent) dependency_wait();
      te = p.tile_e[m];
      low = te >= 0 && g.q_tma && rank == 0;
    }
    const uint32_t src = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    for (int c = (warp >> 2) * 16; c < cols; c += 32) {
      float v[16];
      tmem_ld16(src + c, v);
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        *(float4*)(part + row * kLd + c + i) = any || low ? make_float4(v[i], v[i + 1], v[i + 2], v[i + 3])
                                                          : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_relinquish();
    tmem_dealloc(tmem, kBN < 32 ? 32 : kBN);
    report(bars.err, &g_err);
  }
  if (split > 1) cl.sync();
  if (warp < kProducerWarp) {
    auto sum4 = [&](int row, int c) -> float4 {
      float4 s = *(const float4*)((split > 1 ? cl.map_shared_rank(part, 0) : part) + row * kLd + c);
      for (int i = 1; i < split; ++i) {
        const float4 q = *(const float4*)(cl.map_shared_rank(part, i) + row * kLd + c);
        s.x += q.x, s.y += q.y, s.z += q.z, s.w += q.w;
      }
      return s;
    };
    if constexpr (kShrink) {
      const int a = (int)(row0 - t0), b = (int)(row1 - t0), quads = cols / 4;
      const float scale = p.scale[e];
      for (int i = rank * kWorkers + threadIdx.x; i < (b - a) * quads; i += split * kWorkers) {
        const int row = a + i / quads, c = i % quads * 4;
        const float4 s = sum4(row, c);
        const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (r0 + c + j < e_rank) store_v(p, t0 + row, r0 + c + j, scale * v[j]);
      }
    } else {
      const int64_t n = n0 + lane * 4;
      float bias[4] = {};
      if (p.bias)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (n + i < p.N) bias[i] = to_f32(((const T*)p.bias)[n + i]);
#pragma unroll 2
      for (int row = rank + warp * split; row < rows; row += 8 * split) {
        const int64_t t = t0 + row;
        const int re = row_e[row];
        if (re == kMixed || n >= p.N) continue;
        const float4 s = sum4(row, lane * 4);
        float a[4] = {s.x + bias[0], s.y + bias[1], s.z + bias[2], s.w + bias[3]};
        if (te == kMixed || te == kFew) add_lowrank<T, kSub>(p, t, re, row_rank[row], n, a);
        store4<T>(p, t, n, a);
      }
    }
  }
  __syncwarp();
  if (split > 1) cl.sync();  // nobody leaves while its part is read
}

template <typename T, bool kSub, bool kShrink, int kBN, int kStages>
cf_status launch(const char* what, const Problem& p, const Maps& maps, const Tiling& g, int64_t clusters,
                 cudaStream_t st) {
  constexpr int smem = (kBM + kBN) * 128 * kStages + 1024;
  auto* kern = k_adapter_tile<T, kSub, kShrink, kBN, kStages>;
  static std::atomic<uint64_t> allowed{0};
  CF_TRY(allow_smem(kern, smem, allowed, what));
  const int64_t blocks = clusters * g.split;
  CF_REQUIRE(blocks <= 0x7fffffff, CF_ERR_SHAPE, "%s: too many tiles", what);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)g.split;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = g.dependent ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p, maps, g);
  if (e != cudaSuccess) {
    set_error("%s: %s", what, cudaGetErrorString(e));
    return CF_ERR_CUDA;
  }
  return check_launch(what);
}

template <typename T, bool kSub>
cf_status run(const Problem& p, int dtype, bool row_shrink, bool lowrank_tma, cudaStream_t st) {
  constexpr int kStep = Kind<T>::kStep, kStages = 3;
  const int64_t steps = ceil_div(p.K, kStep), m_tiles = ceil_div(p.T, kBM);
  Maps maps = {};
  Tiling g = {};
  g.m_tiles = m_tiles;
  g.x_rows = (int)(p.T < kBM ? ceil_div(p.T, 8) * 8 : kBM);
  // Row by row: requests of few rows, and float16, whose range does not hold every intermediate that
  // float32 does.
  g.q_tma = dtype == CF_BF16 && lowrank_tma && !row_shrink;
  g.whole = g.q_tma ? 16 : 0;
  CF_TRY(encode(&maps.x, dtype, p.x, p.K, p.T, 1, p.x_rs, p.x_rs * p.T, g.x_rows));
  if (p.R > 0 && row_shrink) {
    CF_TRY(launch_row_shrink(p, dtype, kSub, g.whole, st));
  } else if (p.R > 0) {
    const int bn = p.R <= 64 ? 64 : 128;
    if (kSub)
      CF_TRY(encode(&maps.b, dtype, p.P, p.R, p.K, p.E, p.p_ks, p.p_es, 64));
    else
      CF_TRY(encode(&maps.b, dtype, p.P, p.K, p.R, p.E, p.p_rs, p.p_es, bn));
    g.units = (m_tiles + p.Q - 1) * ceil_div(p.R, bn);
    g.split = split_for(m_tiles, steps);
    const int64_t clusters = g.units + ceil_div(m_tiles, (int64_t)g.split * (kThreads / 32));
    const char* what = "k_adapter_tile (shrink)";
    CF_TRY(bn == 64 ? (launch<T, kSub, true, 64, kStages>(what, p, maps, g, clusters, st))
                    : (launch<T, kSub, true, 128, kStages>(what, p, maps, g, clusters, st)));
  }
  constexpr int bn = 128;
  if (g.q_tma && p.R > 0) {
    CF_TRY(encode(&maps.v_hi, dtype, p.v_hi, p.R, p.T, 1, p.v_rs, p.v_rs * p.T, g.x_rows));
    CF_TRY(encode(&maps.v_lo, dtype, p.v_lo, p.R, p.T, 1, p.v_rs, p.v_rs * p.T, g.x_rows));
  }
  g.dependent = p.R > 0;
  g.units = m_tiles * ceil_div(p.N, bn);
  // More 128-column tiles than a wave: 256-column ones, one CTA an SM (1024 x 4096 x 4096: 29 us
  // against 52; 512 x 4096 x 4096, 128 tiles: 28 both).  Where row tiles may hold several requests,
  // whose low-rank parts the wide kernel puts on the tensor cores and this one does not, from a
  // quarter of a wave on (384 x 4096 x 4096, 5 requests, rank 16: 36 against 54).
  if (g.units > (g.q_tma && p.R > 0 && !row_shrink ? 64 : 128)) 
    return launch_wide(p, dtype, kSub, maps, g.q_tma, g.x_rows, st);
  CF_TRY(encode_weights(p, dtype, kSub, bn, g.q_tma, &maps));
  g.split = split_for(g.units, steps);
  // Tiles for more than half of the SMs: three CTAs a tile, two an SM, where the contraction repays the
  // sums (66 / 88 tiles, us with three and with one: K = 4096 27.1 and 30.4 / 30.2 and 32.5, 2560 20.9 and 21.5 / 21.6
  // and 21.9, 2048 18.8 and 18.5 / 20.0 and 18.6, 768 13.9 and 10.5 / 14.1 and 10.5).  From 89 tiles on two an SM do
  // not hold all CTAs at once.
  if (g.units > 64 && g.units <= 88 && steps >= 36) g.split = 3;
  return launch<T, kSub, false, bn, kStages>("k_adapter_tile", p, maps, g, g.units, st);
}

}  // namespace

cf_status launch_tiles(const Problem& p, int dtype, bool substitute, bool row_shrink, bool lowrank_tma,
                       cudaStream_t st) {
  if (dtype == CF_BF16)
    return substitute ? run<__nv_bfloat16, true>(p, dtype, row_shrink, lowrank_tma, st)
                      : run<__nv_bfloat16, false>(p, dtype, row_shrink, lowrank_tma, st);
  return substitute ? run<__half, true>(p, dtype, row_shrink, lowrank_tma, st)
                    : run<__half, false>(p, dtype, row_shrink, lowrank_tma, st);
}

cf_status take_site_tiles(int* site, cudaStream_t st) { return take_site(&g_err, site, st); }

}  // namespace adapter
}  // namespace cf
