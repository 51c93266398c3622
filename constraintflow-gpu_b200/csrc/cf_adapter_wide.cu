// The adapter product for 16-bit data in 128 x 256 tiles, for grids that fill the GPU: one CTA an
// SM walks over the tiles, the epilogue of one tile under the MMAs of the next.
//
//   y = x M + b + v Q_e:  ceil(K / 64) steps of x M; where all of the tile's rows carry one adapter,
//   two more for every 64 of its rank (v as a bfloat16 pair hi, lo against the same Q_e).  In a
//   tile of a few requests, v Q_e of each goes into the other accumulator, one request after the
//   other, and the epilogue adds it to that request's rows: an infinity or NaN of one adapter does
//   not reach another's rows.  Else the epilogue adds v Q_e row by row on the CUDA cores.
//
// A step of 64 takes 512 cycles of MMAs, for which 48 KB are written to shared memory and 48 KB read: 128 x 128
// tiles would move 32 KB each way for half the work.  8192 x 4096 x 4096: 205 us, 1341 TFLOP/s, 0.96 of what a
// library's product of that size sustains under the power limit (1395); tensor pipe active 0.6 of the time.
// Two CTAs on one 256 x 256 tile (half of B each) took 223 us where this took 200.
//
// Products of 16-bit data stay in the accumulator, which truncates, for all of K: for K = 4096 0.25% of
// the results round to the neighbour of the nearest bfloat16 (float32 FMAs 0.04%, a library's product
// 0.23%).  Against 64 bits both are 1.66e-3 off, the rounding to bfloat16; emptying it, as the float32 tiles
// do, would buy nothing that the result can hold.
// Four stages of 48 KB, two accumulators of 256 columns (all of TMEM), 32 KB through which each
// warp turns its rows into 128-byte stores.
//
// Warps 0-7 epilogue (two a TMEM lane quadrant, 128 columns each), warp 8 TMA, warp 9 MMA.
#include "cf_adapter_tma.cuh"

namespace cf {
namespace adapter {
namespace {

using namespace tc;

constexpr int kBN = 256, kStages = 4, kStep = 64;
constexpr int kEpilogue = 256, kProducerWarp = 8, kMmaWarp = 9, kThreads = 320;
constexpr uint32_t kABytes = kBM * 128, kBBytes = kBN * 128, kStageBytes = kABytes + kBBytes;
constexpr int kSmem = kStages * kStageBytes + 8 * 4096 + 1024;

// The site at which a bounded wait gave up (cf_adapter_check); kernels only write it.
__device__ int g_err;

// Tiles go through the row tiles of a group of kGroup first, then through the columns: what 148 CTAs read
// at a time is then 16 MB of x and 18 MB of M (of 4096 rows), and L2 keeps it (8192 x 4096 x 4096: 214 us in one
// group, 198 to 201 in groups of 8, 16 and 32).
constexpr int kGroup = 16;

struct Bars {
  uint64_t full[kStages], empty[kStages], acc_full[2], acc_empty[2], done;
  uint32_t tmem;
  int err;  // the site at which a wait of this CTA gave up: the others follow
};

template <typename T, bool kSub>
__global__ void __launch_bounds__(kThreads, 1)
    k_adapter_wide(const Problem p, const __grid_constant__ Maps maps, int64_t m_tiles, int64_t units, int q_tma,
                   uint32_t x_bytes) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ Bars bars;
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  const uint32_t sbase = smem_u32(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == kProducerWarp * 32) {
    prefetch_map(&maps.x);
    prefetch_map(&maps.b);
  }
  if (warp == kMmaWarp) tmem_alloc(&bars.tmem, 512);
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&bars.full[i], 1);
      mbar_init(&bars.empty[i], i == 0 ? 1 + p.withhold : 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars.acc_full[i], 1);
      mbar_init(&bars.acc_empty[i], kEpilogue / 32);
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
  bool ok = true, waited = false;
  const int64_t n_tiles = units / m_tiles;
  auto tile_at = [&](int64_t unit, int64_t& m, int64_t& n0) {
    const int64_t g = unit / (kGroup * n_tiles), rest = unit - g * kGroup * n_tiles;
    const int64_t rows = min(m_tiles - g * kGroup, (int64_t)kGroup), n = rest / rows;
    m = g * kGroup + rest - n * rows;
    n0 = n * kBN;
  };
  // What the low-rank part of row tile m takes: the adapter and its rank.  Known once the
  // shrink kernel is done, so the first tile asks behind its contraction.
  auto ask = [&](int64_t m, int& te, int& tr) {
    te = *(volatile int*)(p.tile_e + m);
    tr = rank_of(p, te);
  };

  if (warp == kProducerWarp) {
    int it = 0, loads = 0;  // steps; those that lane 0 has loaded
    // x map entry at (xk, t0) and 256 columns from n0 on of b at contraction bk
    auto load = [&](const CUtensorMap* x, int xk, int64_t t0, const CUtensorMap* b, int bk, int64_t n0, int z) {
      const int s = it % kStages;
      const bool ok = mbar_wait(&bars.empty[s], ((it / kStages) & 1) ^ 1, err, 81, p.max_polls);
      if (ok && lane == 0) {
        mbar_arrive_expect_tx(&bars.full[s], x_bytes + kBBytes);
        const uint32_t dst = sbase + s * kStageBytes;
        tma_3d(dst, x, xk, (int)t0, 0, &bars.full[s]);
        if constexpr (kSub) {
#pragma unroll
          for (int j = 0; j < kBN; j += 64) tma_3d(dst + kABytes + j * 128, b, (int)n0 + j, bk, z, &bars.full[s]);
        } else {
          tma_3d(dst + kABytes, b, bk, (int)n0, z, &bars.full[s]);
        }
        ++loads;
      }
      ++it;
      return (bool)__all_sync(0xffffffffu, ok);  // all lanes go on, or none; behind the loads, which it would delay
    };
    for (int64_t unit = blockIdx.x; unit < units && ok; unit += gridDim.x) {
      int64_t m, n0;
      tile_at(unit, m, n0);
      const int64_t t0 = m * kBM;
      int te = kNone, tr = 0;
      if (q_tma && waited) ask(m, te, tr);
      for (int k = 0; k < n_k && ok; ++k) ok = load(&maps.x, k * kStep, t0, &maps.b, k * kStep, n0, 0);
      if (q_tma && !waited) {
        dependency_wait();
        waited = true;
        ask(m, te, tr);
      }
      auto lowrank = [&](int e, int rank, int, int) {
        for (int r = 0; r < rank; r += kStep)
          if (!load(&maps.v_hi, r, t0, &maps.q, r, n0, e) || !load(&maps.v_lo, r, t0, &maps.q, r, n0, e)) return false;
        return true;
      };
      if (ok && te >= 0) ok = lowrank(te, tr, 0, 0);
      if (ok && te == kFew) ok = for_requests(p, m, p.tile_q[m], reach(p, m, p.tile_q[m]), lowrank);
    }
    // Copies in flight land before shared memory is given up: the others may have given up on them.
    for (int i = max(0, loads - kStages); i < loads; ++i)
      mbar_wait_drain(&bars.full[i % kStages], (i / kStages) & 1, err, 82);
  } else if (warp == kMmaWarp) {
    int it = 0, n_tile = 0, uses[2] = {0, 0};  // uses of each accumulator
    const uint32_t id = idesc(Kind<T>::kAb, kBN, kSub);
    auto claim = [&](int buf) {
      if (!warp_wait(&bars.acc_empty[buf], (uses[buf] & 1) ^ 1, err, 83, p.max_polls)) return false;
      tc_fence_after();
      ++uses[buf];
      return true;
    };
    // k16 MMAs of the next stage into accumulator buf; first: it starts there
    auto step = [&](int buf, int k16, bool first) {
      const int s = it % kStages;
      const bool ok = mbar_wait(&bars.full[s], (it / kStages) & 1, err, 84, p.max_polls);
      tc_fence_after();
      if (ok && lane == 0) {
        const uint32_t a = sbase + s * kStageBytes;
        const uint64_t ad = sw128_desc(a), bd = kSub ? mn_desc(a + kABytes) : sw128_desc(a + kABytes);
        constexpr uint64_t kAStep = 32 >> 4, kBStep = kSub ? (16 * 128) >> 4 : 32 >> 4;
        for (int j = 0; j < k16; ++j)
          mma_f16(tmem + buf * kBN, ad + j * kAStep, bd + j * kBStep, id, !first || j > 0);
        mma_commit(&bars.empty[s]);
      }
      ++it;
      return (bool)__all_sync(0xffffffffu, ok);
    };
    auto lowrank = [&](int buf, int rank, bool first) {
      for (int r = 0; r < rank; r += kStep) {
        const int k16 = (min(rank - r, kStep) + 15) / 16;
        if (!step(buf, k16, first && r == 0) || !step(buf, k16, false)) return false;
      }
      return true;
    };
    auto publish = [&](int buf) {
      if (lane == 0) mma_commit(&bars.acc_full[buf]);
      __syncwarp();
    };
    for (int64_t unit = blockIdx.x; unit < units && ok; unit += gridDim.x, ++n_tile) {
      int64_t m, n0;
      tile_at(unit, m, n0);
      const int buf = n_tile & 1;
      int te = kNone, tr = 0;
      if (q_tma && waited) ask(m, te, tr);
      ok = claim(buf);
      for (int k = 0; k < n_k && ok; ++k) ok = step(buf, 4, k == 0);
      if (q_tma && !waited) {
        dependency_wait();
        waited = true;
        ask(m, te, tr);
      }
      if (ok && te >= 0) ok = lowrank(buf, tr, false);
      if (!ok) break;
      publish(buf);
      if (te == kFew)
        ok = for_requests(p, m, p.tile_q[m], reach(p, m, p.tile_q[m]), [&](int, int rank, int, int) {
          if (!claim(buf ^ 1) || !lowrank(buf ^ 1, rank, true)) return false;
          publish(buf ^ 1);
          return true;
        });
    }
    if (lane == 0) mma_commit(&bars.done);
    __syncwarp();
    mbar_wait_drain(&bars.done, 0, err, 85);
  } else if (warp < kProducerWarp) {
    const int row = (warp & 3) * 32 + lane, half = warp >> 2;
    uint8_t* stage = smem + kStages * kStageBytes + warp * 4096;  // 32 rows x 128 B, swizzled
    int n_tile = 0, uses[2] = {0, 0};
    auto full = [&](int buf) {
      if (!warp_wait(&bars.acc_full[buf], uses[buf] & 1, err, 86, p.max_polls)) return false;
      tc_fence_after();
      ++uses[buf];
      return true;
    };
    auto release = [&](int buf) {
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.acc_empty[buf]);
    };
    for (int64_t unit = blockIdx.x; unit < units && ok; unit += gridDim.x, ++n_tile) {
      int64_t m, n0;
      tile_at(unit, m, n0);
      n0 += half * 128;
      const int64_t t = m * kBM + row;
      const int buf = n_tile & 1;
      if (p.R > 0 && !waited) {
        dependency_wait();
        waited = true;
      }
      const bool own = t < p.T && is_owned(p, t);
      const int te = p.R > 0 ? p.tile_e[m] : kNone;
      const int e = own && (te == kMixed || te == kFew) ? adapter_of(p, request_of(p, t)) : kNone;
      const int rank = rank_of(p, e);
      const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
      // The warp's rows in `rows` from accumulator buf, `more` added: kBoth: of the other accumulator,
      // kRows: v Q_e of each row's adapter.
      enum { kPlain, kRows, kBoth };
      auto write = [&](uint32_t rows, int more) {
#pragma unroll 1
        for (int c = 0; c < 128; c += 64) {
          const int64_t n = n0 + c;
          if (n >= p.N) break;
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            float a[16];
            const uint32_t at = tmem + lanes + half * 128 + c + g * 16;
            tmem_ld16(at + buf * kBN, a);
            tmem_ld_wait();
            if (more == kBoth) {
              float b[16];
              tmem_ld16(at + (buf ^ 1) * kBN, b);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) a[i] += b[i];
            }
            if (p.bias)
#pragma unroll
              for (int i = 0; i < 16; ++i)
                if (n + g * 16 + i < p.N) a[i] += to_f32(((const T*)p.bias)[n + g * 16 + i]);
            if (more == kRows && rank > 0) add_lowrank16<T, kSub>(p, t, e, rank, n + g * 16, a);
            __syncwarp();
            alignas(16) T o[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = from_f32<T>(a[i]);
            *(uint4*)(stage + lane * 128 + (((2 * g) ^ (lane & 7)) << 4)) = *(const uint4*)o;
            *(uint4*)(stage + lane * 128 + (((2 * g + 1) ^ (lane & 7)) << 4)) = *(const uint4*)(o + 8);
          }
          __syncwarp();
          const int64_t tw = m * kBM + (warp & 3) * 32;
#pragma unroll
          for (int i = 0; i < 8; ++i) {  // four rows of 128 B a turn
            const int r = i * 4 + (lane >> 3), chunk = lane & 7;
            if (!((rows >> r) & 1u)) continue;
            const uint4 d = *(const uint4*)(stage + r * 128 + ((chunk ^ (r & 7)) << 4));
            T* y = (T*)p.y + (tw + r) * p.y_rs + n + chunk * 8;
            if (p.y_vec && n + chunk * 8 + 8 <= p.N) {
              *(uint4*)y = d;
            } else {
              alignas(16) T o[8];
              *(uint4*)o = d;
#pragma unroll
              for (int j = 0; j < 8; ++j)
                if (n + chunk * 8 + j < p.N) y[j] = o[j];
            }
          }
          __syncwarp();
        }
      };
      const uint32_t owned = __ballot_sync(0xffffffffu, own);
      ok = full(buf);
      if (!ok) break;
      if (te != kFew) {
        write(owned, te == kMixed ? kRows : kPlain);
      } else {
        const uint32_t plain = owned & __ballot_sync(0xffffffffu, rank == 0);
        if (plain) write(plain, kPlain);
        ok = for_requests(p, m, p.tile_q[m], reach(p, m, p.tile_q[m]), [&](int, int, int a, int b) {
          if (!full(buf ^ 1)) return false;
          const uint32_t mine = __ballot_sync(0xffffffffu, row >= a && row < b);
          if (mine) write(mine, kBoth);
          release(buf ^ 1);
          return true;
        });
      }
      release(buf);
    }
  }
  __syncwarp();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_relinquish();
    tmem_dealloc(tmem, 512);
    report(bars.err, &g_err);
  }
}

template <typename T, bool kSub>
cf_status launch(const Problem& p, const Maps& maps, bool q_tma, int x_rows, cudaStream_t st) {
  auto* kern = k_adapter_wide<T, kSub>;
  static std::atomic<uint64_t> allowed{0};
  CF_TRY(allow_smem(kern, kSmem, allowed, "k_adapter_wide"));
  const int64_t m_tiles = ceil_div(p.T, kBM), units = m_tiles * ceil_div(p.N, kBN);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(units < 148 ? units : 148));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = p.R > 0 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p, maps, m_tiles, units, (int)(q_tma && p.R > 0),
                         (uint32_t)x_rows * 128u);
  if (e != cudaSuccess) {
    set_error("k_adapter_wide: %s", cudaGetErrorString(e));
    return CF_ERR_CUDA;
  }
  return check_launch("k_adapter_wide");
}

}  // namespace

cf_status launch_wide(const Problem& p, int dtype, bool substitute, Maps maps, bool q_tma, int x_rows,
                      cudaStream_t st) {
  CF_TRY(encode_weights(p, dtype, substitute, kBN, q_tma, &maps));
  if (dtype == CF_BF16)
    return substitute ? launch<__nv_bfloat16, true>(p, maps, q_tma, x_rows, st)
                      : launch<__nv_bfloat16, false>(p, maps, q_tma, x_rows, st);
  return substitute ? launch<__half, true>(p, maps, q_tma, x_rows, st) : launch<__half, false>(p, maps, q_tma, x_rows, st);
}

cf_status take_site_wide(int* site, cudaStream_t st) { return take_site(&g_err, site, st); }

}  // namespace adapter
}  // namespace cf
