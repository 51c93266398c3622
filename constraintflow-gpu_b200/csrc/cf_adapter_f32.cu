// The adapter product for float32 data: 128 x kBN tiles on tcgen05 as 3xTF32.
//
//   k_adapter_f32<.., kShrink = true>   v = s_e x P_e for the rows of one request in one row tile
//   k_adapter_f32<.., kShrink = false>  y = x M + b + v Q_e
//
// 3xTF32: an operand is split into tf32 hi + lo, and hi*hi + hi*lo + lo*hi is summed.  The tensor
// core adds into its accumulator with truncation, an error that grows with every addition and
// always points towards zero, so a sum stays in the accumulator for kChunk steps of 32 only; the
// epilogue's warps add the chunks in registers, rounded to nearest.  The error of a sum is then
// that of 24 truncated additions of a chunk, not of 3 K / 8.  It is above that of float32 FMAs all the
// same, as an operand keeps 22 bits and lo*lo is left out: 4.6e-7 of y against 64 bits where FMAs are
// 2.6e-7 off (51200 x 200 x 784).
//
// The chunks also keep requests apart: the low-rank part of each request that reaches into the
// tile is a chunk of its own, added to that request's rows only (a masked operand would not do:
// 0 * inf of another request's adapter is NaN).  Requests of few rows would make many such chunks;
// their low-rank part is added row by row on the CUDA cores instead.
//
// Warps 0-7 drain chunks and write the tile, warps 8-15 load operands of any stride and alignment
// (the next step's loads in flight while this step's are split and stored), warp 16 issues the
// MMAs.  One CTA an SM walks over the tiles, the epilogue of a tile under the MMAs of the next;
// with few tiles the contraction is dealt out to the CTAs of a cluster instead, which sum their
// parts in rank order.
//
// 4096 x 4096 x 4096, rank 64: 971 us, 146 TFLOP/s, 0.53 of the rate of 3xTF32 alone (276): a step's images
// are written, read for three products and loaded through the same 128 bytes a cycle of the SM, about
// as long as its MMAs take to issue.  A third stage takes the L1 cache that the loads go through (1104 us, 975
// with two at that time).
// 51200 x 200 x 784 with 256 requests of rank 8: 257 us, substituted 283, without adapters 166 and 176.
// About 3% of these times is the lanes' agreement on the outcome of each wait.
#include <cooperative_groups.h>

#include <type_traits>

#include "cf_adapter_dev.cuh"

namespace cg = cooperative_groups;

namespace cf {
namespace adapter {
namespace {

using namespace tc;

constexpr int kDrain = 256, kLoad = 256;  // threads of the two groups
constexpr int kMmaWarp = 16;
constexpr int kThreads = 640;  // five warpgroups; warps 17-19 idle
// Registers a thread: 96 at launch (640 x 96 = 61440).  What the MMA group gives up goes to the drain, which
// holds a tile's sums, 128 (2 x 112 + 2 x 96 + 64) = 61440; for v, with half a tile and less, to the loads.
constexpr int kMmaRegs = 64;
template <bool kShrink, int kBN>
struct Regs {
  static constexpr int kDrain = kShrink ? (kBN == 64 ? 96 : 104) : 112, kLoad = 208 - kDrain;
};
constexpr int kStep = 32;   // contraction of a stage: 128 bytes
constexpr int kChunk = 2;   // steps of one accumulation
constexpr int kStages = 2, kBufs = 2;

// The site at which a bounded wait gave up (cf_adapter_check); kernels only write it.
__device__ int g_err;

template <int kRegs>
__device__ __forceinline__ void more_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
}
template <int kRegs>
__device__ __forceinline__ void fewer_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}

struct Tiling {
  int64_t m_tiles, units, clusters;  // clusters: on tiles; behind them, clusters that plan row tiles
  int32_t split;                     // CTAs of a cluster
  int32_t rowwise;                   // the low-rank part row by row
  int32_t dependent;                 // launched while the shrink kernel may still run
};

struct Tile {
  int32_t m, t0, n0, row0, row1;  // shrink: rows [row0, row1) of the tile
  int32_t e, e_rank, r0, cols;
};

// The tile of a unit, by a warp together; false: nothing to do.
template <bool kShrink, int kBN>
__device__ __forceinline__ bool tile_of(const Problem& p, const Tiling& g, int64_t unit, Tile& w) {
  w.n0 = w.row0 = w.row1 = 0;
  w.e = kNone, w.e_rank = w.r0 = 0;
  if constexpr (kShrink) {
    const int64_t blocks_r = (p.R + kBN - 1) / kBN, u = unit / blocks_r;
    w.r0 = (int)(unit - u * blocks_r) * kBN;
    // tile + request numbers the overlapping (tile, request) pairs; request q of unit u is the
    // first that ends behind tile u - q's start
    const int64_t lo = warp_search(0, p.Q, [&](int64_t q) { return p.offsets[q + 1] + kBM * q > kBM * u; });
    if (lo >= p.Q) return false;
    const int64_t m = u - lo;
    if (m < 0 || m >= g.m_tiles) return false;
    const int64_t t0 = m * kBM, row0 = max(p.offsets[lo], t0), row1 = min(min(p.offsets[lo + 1], t0 + kBM), p.T);
    w.e = adapter_of(p, lo);
    w.e_rank = rank_of(p, w.e);
    if (row0 >= row1 || w.r0 >= w.e_rank) return false;
    w.m = (int)m;
    w.row0 = (int)(row0 - t0);
    w.row1 = (int)(row1 - t0);
    w.cols = min(kBN, (w.e_rank - w.r0 + 15) / 16 * 16);
  } else {
    const int n_tile = (int)(unit / g.m_tiles);
    w.m = (int)(unit - n_tile * g.m_tiles);
    w.n0 = n_tile * kBN;
    w.cols = kBN;
  }
  w.t0 = w.m * kBM;
  return true;
}

struct Bars {
  uint64_t full[kStages], empty[kStages], acc_full[kBufs], acc_empty[kBufs], done;
  uint32_t tmem;
  int err;  // the site at which a wait of this CTA gave up: the others follow
};

template <int kBN>
struct Chunks {  // one step's operand chunks of a loading thread
  uint4 x[kBM * 8 / kLoad], b[kBN * 8 / kLoad];
};

template <bool kSub, bool kShrink, int kBN>
__global__ void __launch_bounds__(kThreads, 1) k_adapter_f32(const Problem p, const Tiling g) {
  constexpr uint32_t kABytes = kBM * 128, kBBytes = kBN * 128, kStageBytes = 2 * (kABytes + kBBytes);
  constexpr int kLd = kBN + 4;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Bars bars;
  __shared__ int row_e[kShrink ? 1 : kBM];  // each row's adapter, kMixed for a row of no request
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const uint32_t sbase = smem_u32(smem);
  float* part = (float*)smem;  // a cluster's tile, [kBM][kLd], where its operands were
  static_assert(kBM * kLd * 4 <= kStages * kStageBytes, "the tile is staged where the operands were");
  cg::cluster_group cl = cg::this_cluster();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = g.split, rank = split > 1 ? (int)cl.block_rank() : 0;
  const int64_t cluster = blockIdx.x / split;
  if constexpr (kShrink) {
    launch_dependents();
    if (cluster >= g.clusters) {
      const int64_t tile = ((cluster - g.clusters) * split + rank) * (kThreads / 32) + warp;
      if (tile < g.m_tiles) plan_tile(p, tile, 1);
      return;
    }
  }
  if (warp == kMmaWarp) tmem_alloc(&bars.tmem, kBufs * kBN);
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&bars.full[i], kLoad);
      mbar_init(&bars.empty[i], i == 0 ? 1 + p.withhold : 1);
    }
    for (int i = 0; i < kBufs; ++i) {
      mbar_init(&bars.acc_full[i], 1);
      mbar_init(&bars.acc_empty[i], kDrain / 32);
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
  const int n_k = (int)((p.K + kStep - 1) / kStep);
  const int kb = (int)((int64_t)n_k * rank / split), ke = (int)((int64_t)n_k * (rank + 1) / split);
  // the requests' low-rank parts as chunks
  const bool lowrank = !kShrink && p.R > 0 && !g.rowwise && rank == 0;
  Tile w = {};
  // v up to the adapter's rank, and zeros up to the next multiple of 4
  auto put_v4 = [&](int64_t t, int r, float scale, float a, float b, float c, float d) {
    if (r >= w.e_rank) return;
    *(float4*)(p.v + t * p.v_rs + r) = make_float4(scale * a, r + 1 < w.e_rank ? scale * b : 0.0f,
                                                   r + 2 < w.e_rank ? scale * c : 0.0f, r + 3 < w.e_rank ? scale * d : 0.0f);
  };
  bool waited = !g.dependent;
  bool ok = true;

  if (warp >= 8 && warp < kMmaWarp) {
    // ---------------------------------------------------------------- loads
    more_registers<Regs<kShrink, kBN>::kLoad>();
    const int tid = threadIdx.x - kDrain, chunk = tid & 7, prow = tid >> 3;
    int it = 0;
    // four elements of a row with contiguous k from k on, of n_kk; vec: 16-byte aligned, n_kk a
    // multiple of 4
    auto row4 = [&](auto vec, const float* row, int k, int n_kk, bool ok) -> uint4 {
      if constexpr (decltype(vec)::value) {
        return ldg16_if(row + k, ok && k < n_kk);
      } else {
        uint4 d;
        d.x = ldg4_if(row + k, ok && k < n_kk);
        d.y = ldg4_if(row + k + 1, ok && k + 1 < n_kk);
        d.z = ldg4_if(row + k + 2, ok && k + 2 < n_kk);
        d.w = ldg4_if(row + k + 3, ok && k + 3 < n_kk);
        return d;
      }
    };
    auto fetch_x = [&](auto vec, uint4(&d)[kBM * 8 / kLoad], const float* x, int64_t rs, int t0, int k,
                       int n_kk) {
      const float* row = x + (int64_t)(t0 + prow) * rs;
      const int rows = (int)min(p.T - t0, (int64_t)kBM);
#pragma unroll
      for (int j = 0; j < kBM * 8 / kLoad; ++j)
        d[j] = row4(vec, row + j * (kLoad / 8) * rs, k + chunk * 4, n_kk, prow + j * (kLoad / 8) < rows);
    };
    // columns [0, n_c) of B, contraction k .. of n_kk
    auto fetch_b = [&](auto vec, uint4(&d)[kBN * 8 / kLoad], const float* B, int64_t ks, int64_t ns, int n_c, int k,
                       int n_kk) {
#pragma unroll
      for (int j = 0; j < kBN * 8 / kLoad; ++j) {
        if constexpr (kSub) {  // columns contiguous: consecutive threads, consecutive columns
          const int task = j * kLoad + tid, c = task % kBN, kk = k + task / kBN * 4;
          const float* at = B + kk * ks + c;
          const bool ok = c < n_c;
          d[j].x = ldg4_if(at, ok && kk < n_kk);
          d[j].y = ldg4_if(at + ks, ok && kk + 1 < n_kk);
          d[j].z = ldg4_if(at + 2 * ks, ok && kk + 2 < n_kk);
          d[j].w = ldg4_if(at + 3 * ks, ok && kk + 3 < n_kk);
        } else {
          const int c = prow + j * (kLoad / 8);
          d[j] = row4(vec, B + c * ns, k + chunk * 4, n_kk, c < n_c);
        }
      }
    };
    const int K = (int)p.K;
    auto fetch = [&](auto vec, Chunks<kBN>& d, const Tile& w, int k) {
      fetch_x(vec, d.x, (const float*)p.x, p.x_rs, w.t0, k * kStep, K);
      if constexpr (kShrink)
        fetch_b(vec, d.b, (const float*)p.P + w.e * p.p_es + w.r0 * p.p_rs, p.p_ks, p.p_rs, w.e_rank - w.r0, k * kStep,
                K);
      else
        fetch_b(vec, d.b, (const float*)p.M + w.n0 * p.m_ns, p.m_ks, p.m_ns, (int)min(p.N - w.n0, (int64_t)kBN),
                k * kStep, K);
    };
    auto store = [&](const Chunks<kBN>& d) -> bool {
      const int s = it % kStages, round = it / kStages;
      if (!warp_wait(&bars.empty[s], (round & 1) ^ 1, err, 51, p.max_polls)) return false;
      const uint32_t a = sbase + s * kStageBytes, b = a + 2 * kABytes;
#pragma unroll
      for (int j = 0; j < kBM * 8 / kLoad; ++j) put(a, kABytes, prow + j * (kLoad / 8), chunk, d.x[j]);
#pragma unroll
      for (int j = 0; j < kBN * 8 / kLoad; ++j) {
        if constexpr (kSub) {
          const int task = j * kLoad + tid;
          put(b, kBBytes, task % kBN, task / kBN, d.b[j]);
        } else {
          put(b, kBBytes, prow + j * (kLoad / 8), chunk, d.b[j]);
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(&bars.full[s]);
      ++it;
      return true;
    };
    // A tile's steps: the contraction's, then those of its requests' low-rank parts, the next one's
    // loads in flight while a step's are split and stored.
    int k = 0;
    uint32_t todo = 0;  // of the 32 requests from `from` on, those that have an adapter and rows here
    int from = 0, e = kNone, r = 0, r0 = 0;
    bool begun = false, past = true;
    auto look = [&] {
      const Reach at = reach(p, w.m, from);
      todo = __ballot_sync(0xffffffffu, at.r > 0);
      past = __any_sync(0xffffffffu, at.past);
    };
    auto next = [&](auto vec, Chunks<kBN>& d) -> bool {
      if (k < ke) {
        fetch(vec, d, w, k++);
        return true;
      }
      if (!lowrank) return false;
      if (!begun) {
        begun = true;
        if (!waited) dependency_wait();
        waited = true;
        from = p.tile_q[w.m];
        r = 0;
        look();
      }
      r0 += kStep;
      if (r0 >= r) {
        while (todo == 0) {
          if (past) return false;
          from += 32;
          look();
        }
        const int i = __ffs(todo) - 1;
        todo &= todo - 1;
        e = adapter_of(p, from + i);
        r = rank_of(p, e);
        r0 = 0;
      }
      // rows of v are 16-byte aligned and zero from the rank to the next multiple of 4
      fetch_x(std::true_type{}, d.x, p.v, p.v_rs, w.t0, r0, r);
      fetch_b(std::false_type{}, d.b, (const float*)p.Qm + e * p.q_es + w.n0 * p.q_ns, p.q_rs, p.q_ns,
              (int)min(p.N - w.n0, (int64_t)kBN), r0, r);
      return true;
    };
    auto tiles = [&](auto vec) {
      for (int64_t unit = cluster; unit < g.units && ok; unit += g.clusters) {
        if (!tile_of<kShrink, kBN>(p, g, unit, w)) continue;
        k = kb;
        begun = false;
        Chunks<kBN> one, two;
        bool more = next(vec, one);
        while (more) {
          more = next(vec, two);
          ok = store(one);
          if (!ok || !more) break;
          more = next(vec, one);
          ok = store(two);
          if (!ok) break;
        }
      }
    };
    const bool vec = p.x_vec && (kShrink ? p.p_vec : p.m_vec) && p.K % 4 == 0;
    if (vec || (kSub && p.x_vec && p.K % 4 == 0))
      tiles(std::true_type{});
    else
      tiles(std::false_type{});
  } else if (warp >= kMmaWarp) {
    // ---------------------------------------------------------------- MMAs
    fewer_registers<kMmaRegs>();
    if (warp == kMmaWarp) {
    int it = 0, ch = 0;
    // one step into chunk ch; first / last of its chunk
    auto step = [&](int mmas, bool first, bool last, uint32_t id) -> bool {
      const int s = it % kStages, buf = ch % kBufs;
      const bool ok = (!first || mbar_wait(&bars.acc_empty[buf], ((ch / kBufs) & 1) ^ 1, err, 61, p.max_polls)) &&
                      mbar_wait(&bars.full[s], (it / kStages) & 1, err, 62, p.max_polls);
      tc_fence_after();
      if (ok && lane == 0) {
        const uint32_t a = sbase + s * kStageBytes, d = tmem + buf * kBN;
        const uint64_t ad = sw128_desc(a), bd = sw128_desc(a + 2 * kABytes);
        constexpr uint64_t kALo = kABytes >> 4, kBLo = kBBytes >> 4;
        for (int j = 0; j < mmas; ++j) {
          mma_tf32(d, ad + kALo + 2 * j, bd + 2 * j, id, !first || j > 0);  // the small terms first
          mma_tf32(d, ad + 2 * j, bd + kBLo + 2 * j, id, 1);
          mma_tf32(d, ad + 2 * j, bd + 2 * j, id, 1);
        }
        mma_commit(&bars.empty[s]);
        if (last) mma_commit(&bars.acc_full[buf]);
      }
      ++it;
      ch += last;
      return __all_sync(0xffffffffu, ok);  // all lanes go on, or none; behind the MMAs, which it would delay
    };
    for (int64_t unit = cluster; unit < g.units && ok; unit += g.clusters) {
      if (!tile_of<kShrink, kBN>(p, g, unit, w)) continue;
      const uint32_t id = idesc(Kind<float>::kAb, w.cols, false);
      for (int k = kb; k < ke && ok; ++k)
        ok = step(4, (k - kb) % kChunk == 0, (k - kb) % kChunk == kChunk - 1 || k + 1 == ke, id);
      if (lowrank && ok) {
        if (!waited) dependency_wait();
        waited = true;
        const int from = p.tile_q[w.m];
        ok = for_requests(p, w.m, from, reach(p, w.m, from), [&](int, int r, int, int) {
          for (int r0 = 0; r0 < r; r0 += kStep)
            if (!step((min(r - r0, kStep) + 7) / 8, true, true, id)) return false;
          return true;
        });
      }
    }
    if (lane == 0) mma_commit(&bars.done);
    mbar_wait_drain(&bars.done, 0, err, 63);  // every MMA has run before tensor memory is given up
    }
  } else {
    // ---------------------------------------------------------------- chunks, tiles
    more_registers<Regs<kShrink, kBN>::kDrain>();  // the compiler allots by it
    const int row = (warp & 3) * 32 + lane, c0 = (warp >> 2) * (kBN / 2);
    const uint32_t src = tmem + ((uint32_t)((warp & 3) * 32) << 16) + c0;
    int ch = 0;
    for (int64_t unit = cluster; unit < g.units && ok; unit += g.clusters) {
      if (!tile_of<kShrink, kBN>(p, g, unit, w)) continue;
      const int rows = (int)min((int64_t)kBM, p.T - w.t0);
      if constexpr (!kShrink) {
        if (split > 1 && threadIdx.x < rows) {
          const int64_t t = w.t0 + (int)threadIdx.x;
          row_e[threadIdx.x] = !is_owned(p, t) ? kMixed : g.rowwise ? adapter_of(p, request_of(p, t)) : kNone;
        }
      }
      float acc[kBN / 2];
#pragma unroll
      for (int i = 0; i < kBN / 2; ++i) acc[i] = 0.0f;
      auto drain = [&](bool mine) -> bool {
        const int buf = ch % kBufs;
        const bool ok = mbar_wait(&bars.acc_full[buf], (ch / kBufs) & 1, err, 71, p.max_polls);
        // (a chunk that a lane gave up on is read all the same, and is worth nothing: the lanes agree behind it)
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < kBN / 2; c += 16) {
          if (kShrink && c0 + c >= w.cols) break;
          float v[16];
          tmem_ld16(src + buf * kBN + c, v);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i) acc[c + i] = mine ? acc[c + i] + v[i] : acc[c + i];
        }
        tc_fence_before();
        const bool all = __all_sync(0xffffffffu, ok);
        if (lane == 0) mbar_arrive(&bars.acc_empty[buf]);
        ++ch;
        return all;
      };
      for (int k = kb; k < ke && ok; k += kChunk) ok = drain(true);
      if (!kShrink && p.R > 0 && !waited) {
        dependency_wait();
        waited = true;
      }
      if (lowrank && ok) {
        const int from = p.tile_q[w.m];
        ok = for_requests(p, w.m, from, reach(p, w.m, from), [&](int, int r, int a, int b) {
          for (int r0 = 0; r0 < r; r0 += kStep)
            if (!drain(row >= a && row < b)) return false;
          return true;
        });
      }
      if (split > 1) {  // one tile: the cluster's parts are summed below
        if (!ok) break;
#pragma unroll
        for (int i = 0; i < kBN / 2; i += 4)
          *(float4*)(part + row * kLd + c0 + i) = make_float4(acc[i], acc[i + 1], acc[i + 2], acc[i + 3]);
        break;
      }
      if (!ok) break;
      if constexpr (kShrink) {
        if (row >= w.row0 && row < w.row1) {
          const float scale = p.scale[w.e];
#pragma unroll
          for (int i = 0; i < kBN / 2; i += 4) put_v4(w.t0 + row, w.r0 + c0 + i, scale, acc[i], acc[i + 1], acc[i + 2], acc[i + 3]);
        }
      } else {
        // The warp's rows, 32 columns at a time: turned in its own shared memory, written four rows of 128
        // bytes a turn.
        const int64_t t = w.t0 + row;
        const int mine = row >= rows || !is_owned(p, t) ? kMixed : g.rowwise ? adapter_of(p, request_of(p, t)) : kNone;
        float* turn = (float*)(smem + kStages * kStageBytes) + warp * 1024;
#pragma unroll
        for (int c = 0; c < kBN / 2; c += 32) {
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 8; ++i)
            *(float4*)(turn + lane * 32 + ((i ^ (lane & 7)) << 2)) =
                make_float4(acc[c + 4 * i], acc[c + 4 * i + 1], acc[c + 4 * i + 2], acc[c + 4 * i + 3]);
          __syncwarp();
          const int64_t n = w.n0 + c0 + c + (lane & 7) * 4;
          float bias[4] = {};
          if (p.bias)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (n + i < p.N) bias[i] = ((const float*)p.bias)[n + i];
#pragma unroll 1
          for (int i = 0; i < 8; ++i) {
            const int r = i * 4 + (lane >> 3), re = __shfl_sync(0xffffffffu, mine, r);
            if (re == kMixed || n >= p.N) continue;
            const float4 d = *(const float4*)(turn + r * 32 + (((lane & 7) ^ (r & 7)) << 2));
            float a[4] = {d.x + bias[0], d.y + bias[1], d.z + bias[2], d.w + bias[3]};
            const int64_t tr = w.t0 + (warp & 3) * 32 + r;
            if (g.rowwise) add_lowrank<float, kSub>(p, tr, re, rank_of(p, re), n, a);
            store4<float>(p, tr, n, a);
          }
        }
      }
    }
  }
  __syncwarp();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_relinquish();
    tmem_dealloc(tmem, kBufs * kBN);
    report(bars.err, &g_err);
  }
  if (split == 1) return;

  // ---- the parts of the cluster's one tile
  cl.sync();
  if (warp < 8 && tile_of<kShrink, kBN>(p, g, cluster, w)) {
    auto sum4 = [&](int row, int c) -> float4 {
      float4 s = *(const float4*)(cl.map_shared_rank(part, 0) + row * kLd + c);
      for (int i = 1; i < split; ++i) {
        const float4 q = *(const float4*)(cl.map_shared_rank(part, i) + row * kLd + c);
        s.x += q.x, s.y += q.y, s.z += q.z, s.w += q.w;
      }
      return s;
    };
    if constexpr (kShrink) {
      const int a = w.row0, b = w.row1, quads = w.cols / 4;
      const float scale = p.scale[w.e];
      for (int i = rank * kDrain + threadIdx.x; i < (b - a) * quads; i += split * kDrain) {
        const int r = a + i / quads, c = i % quads * 4;
        const float4 s = sum4(r, c);
        put_v4(w.t0 + r, w.r0 + c, scale, s.x, s.y, s.z, s.w);
      }
    } else {
      const int rows = (int)min((int64_t)kBM, p.T - w.t0);
      const int64_t n = w.n0 + lane * 4;
      float bias[4] = {};
      if (p.bias)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (n + i < p.N) bias[i] = ((const float*)p.bias)[n + i];
      for (int r = rank + warp * split; r < rows; r += 8 * split) {
        const int re = row_e[r];
        if (re == kMixed || n >= p.N) continue;
        const float4 s = sum4(r, lane * 4);
        float a[4] = {s.x + bias[0], s.y + bias[1], s.z + bias[2], s.w + bias[3]};
        if (g.rowwise) add_lowrank<float, kSub>(p, w.t0 + r, re, rank_of(p, re), n, a);
        store4<float>(p, w.t0 + r, n, a);
      }
    }
  }
  __syncwarp();
  cl.sync();  // nobody leaves while its part is read
}

template <bool kSub, bool kShrink, int kBN>
cf_status launch(const Problem& p, Tiling g, cudaStream_t st) {
  constexpr int smem = kStages * 2 * (kBM + kBN) * 128 + (kShrink ? 0 : kDrain / 32 * 4096) + 1024;
  auto* kern = k_adapter_f32<kSub, kShrink, kBN>;
  static std::atomic<uint64_t> allowed{0};
  CF_TRY(allow_smem(kern, smem, allowed, "k_adapter_f32"));
  g.split = split_for(kShrink ? g.m_tiles : g.units, ceil_div(p.K, kStep));
  // one CTA an SM walks over the tiles; a cluster has one
  g.clusters = g.split > 1 ? g.units : (g.units < 148 ? g.units : 148);
  const int64_t plans = kShrink ? ceil_div(g.m_tiles, (int64_t)g.split * (kThreads / 32)) : 0;
  const int64_t blocks = (g.clusters + plans) * g.split;
  CF_REQUIRE(blocks <= 0x7fffffff, CF_ERR_SHAPE, "k_adapter_f32: too many tiles");
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
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p, g);
  if (e != cudaSuccess) {
    set_error("k_adapter_f32: %s", cudaGetErrorString(e));
    return CF_ERR_CUDA;
  }
  return check_launch("k_adapter_f32");
}

template <bool kSub>
cf_status run(const Problem& p, bool row_shrink, cudaStream_t st) {
  Tiling g = {};
  g.m_tiles = ceil_div(p.T, kBM);
  g.rowwise = row_shrink && p.R > 0;
  if (p.R > 0 && row_shrink) {
    CF_TRY(launch_row_shrink(p, CF_F32, kSub, 1, st));
  } else if (p.R > 0) {
    const int bn = p.R <= 64 ? 64 : 128;
    g.units = (g.m_tiles + p.Q - 1) * ceil_div(p.R, bn);
    CF_TRY(bn == 64 ? (launch<kSub, true, 64>(p, g, st)) : (launch<kSub, true, 128>(p, g, st)));
  }
  g.dependent = p.R > 0;
  g.units = g.m_tiles * ceil_div(p.N, 128);
  return launch<kSub, false, 128>(p, g, st);
}

}  // namespace

cf_status launch_f32(const Problem& p, bool substitute, bool row_shrink, cudaStream_t st) {
  return substitute ? run<true>(p, row_shrink, st) : run<false>(p, row_shrink, st);
}

cf_status take_site_f32(int* site, cudaStream_t st) { return take_site(&g_err, site, st); }

}  // namespace adapter
}  // namespace cf
