// The rule by which an answer is taken from logits, per row (request, region): penalties for
// what the row's history holds, biases, and a set of allowed answers; applied to logits
// (cf_edit_logits) and to bounds of logits (cf_answer_margin).
//
//   v = x;  j in the history:            v = v > 0 ? v / repetition : v * repetition
//           c = times j was answered:    v = v - frequency * c,  v = v - presence (c > 0)
//           j has a bias:                v = v + bias (the last entry given for j)
//           j is not allowed:            v = -inf
//
// Each step is a float32 operation rounded on its own (no fused multiply-add), so every step
// is monotone in x for repetition > 0: the edit of a lower (upper) bound is a lower (upper)
// bound of the edit, rounding included, and no interval arithmetic is needed.
//
// Memory-bound: a row is read (and written) once.  What a row's history says about its n
// answers is a scatter; a cluster of CTAs takes a span of the answers, each CTA holding the
// counts of its own slice in shared memory, and the cluster walks the history once, every CTA
// a share of it, adding to the owner's counts through distributed shared memory.  Counts are
// integers and "the last entry" is a maximum, so the order of the atomics changes nothing.
#include <cooperative_groups.h>

#include "cf_common.cuh"
#include "cf_elem.cuh"

namespace cg = cooperative_groups;

namespace cf {
namespace {

constexpr uint32_t kSeen = 0x80000000u;  // in the history, prompt included
constexpr int kThreads = 512;
constexpr int kMinSlice = 512;
constexpr int kMaxCluster = 8;

// bytes of a slice's tables: counts, and the place of the last bias where biases are given
constexpr int kSliceBytes = 64 * 1024;

struct Row {
  int64_t h0, h1, answered;  // history, and where its answered part begins
  int64_t b0, b1;            // biases
  float rep, freq, pres;
  const uint32_t* allowed;  // nullptr: everything
};

__device__ __forceinline__ int64_t clamp64(int64_t x, int64_t lo, int64_t hi) {
  return x < lo ? lo : (x > hi ? hi : x);
}

__device__ Row load_row(const cf_answer_rules& R, int64_t r) {
  Row w;
  w.h0 = w.h1 = w.b0 = w.b1 = 0;
  if (R.tokens_dev) {
    w.h0 = clamp64(R.token_offsets_dev[r], 0, R.n_tokens);
    w.h1 = clamp64(R.token_offsets_dev[r + 1], w.h0, R.n_tokens);
  }
  w.answered = w.h0 + (R.prompt_len_dev ? (int64_t)max(R.prompt_len_dev[r], 0) : 0);
  if (R.bias_ids_dev) {
    w.b0 = clamp64(R.bias_offsets_dev[r], 0, R.n_biases);
    w.b1 = clamp64(R.bias_offsets_dev[r + 1], w.b0, R.n_biases);
  }
  w.rep = R.repetition_dev ? R.repetition_dev[r] : 1.0f;
  w.freq = R.frequency_dev ? R.frequency_dev[r] : 0.0f;
  w.pres = R.presence_dev ? R.presence_dev[r] : 0.0f;
  w.allowed = nullptr;
  if (R.allowed_dev) {
    const int64_t m = R.allowed_row_dev ? (int64_t)R.allowed_row_dev[r] : r;
    if (m >= 0 && m < R.n_masks) w.allowed = (const uint32_t*)R.allowed_dev + m * R.allowed_words;
  }
  return w;
}

__device__ __forceinline__ float edit(float v, uint32_t c, uint32_t bias_at, const Row& w, const float* biases) {
  if (c) {
    v = v > 0.0f ? __fdiv_rn(v, w.rep) : __fmul_rn(v, w.rep);
    const uint32_t times = c & ~kSeen;
    if (times) v = __fsub_rn(__fsub_rn(v, __fmul_rn(w.freq, (float)times)), w.pres);
  }
  if (bias_at) v = __fadd_rn(v, biases[w.b0 + bias_at - 1]);
  return v;
}

// The tables of answers [lo + rank * S, + S) of one span for this CTA; lo counts answers and may
// start before the first (the row's own alignment).  Every CTA of the cluster calls it.
__device__ void tables(const cf_answer_rules& R, const Row& w, int64_t lo, int log_s, uint32_t* cnt, uint32_t* pos,
                       cg::cluster_group& cl) {
  const int S = 1 << log_s;
  const uint32_t nc = cl.num_blocks(), rank = cl.block_rank();
  const bool bias = w.b1 > w.b0;
  for (int i = threadIdx.x * 4; i < S; i += blockDim.x * 4) {
    *(uint4*)(cnt + i) = make_uint4(0, 0, 0, 0);
    if (bias) *(uint4*)(pos + i) = make_uint4(0, 0, 0, 0);
  }
  cl.sync();
  const int64_t step = (int64_t)nc * blockDim.x, at = (int64_t)rank * blockDim.x + threadIdx.x;
  const uint64_t span = (uint64_t)nc << log_s;
  for (int64_t i = w.h0 + at; i < w.h1; i += step) {
    const int64_t j = R.tokens_dev[i];
    const uint64_t rel = (uint64_t)(j - lo);
    if (j < 0 || j >= R.n || rel >= span) continue;
    uint32_t* c = cl.map_shared_rank(cnt, (unsigned)(rel >> log_s)) + (rel & (S - 1));
    if (i < w.answered)
      atomicOr(c, kSeen);
    else
      atomicAdd(c, 1u);
  }
  for (int64_t i = w.b0 + at; i < w.b1; i += step) {
    const int64_t j = R.bias_ids_dev[i];
    const uint64_t rel = (uint64_t)(j - lo);
    if (j < 0 || j >= R.n || rel >= span) continue;
    atomicMax(cl.map_shared_rank(pos, (unsigned)(rel >> log_s)) + (rel & (S - 1)), (uint32_t)(i - w.b0) + 1u);
  }
  cl.sync();
}

template <typename T>
struct alignas(16) Vec {
  static constexpr int N = 16 / sizeof(T);
  T v[N];
};

// The bits of `allowed` for N answers from j on, all of them answers.
template <int N>
__device__ __forceinline__ uint32_t allowed_bits(const uint32_t* allowed, int64_t j) {
  if (!allowed) return 0xffffffffu;
  const int sh = (int)(j & 31);
  uint32_t bits = allowed[j >> 5] >> sh;
  if (sh + N > 32) bits |= allowed[(j >> 5) + 1] << (32 - sh);
  return bits;
}

// One cluster per (row, span) of the grid.  mis: answers between the 16-byte boundary below the
// row's start and the start, so that whole vectors fall on whole vectors of the tables.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    k_edit_logits(const cf_answer_rules R, const T* __restrict__ in, int64_t in_rs, T* out, int64_t out_rs,
                  int log_s, int spans) {
  extern __shared__ __align__(16) uint32_t smem[];
  constexpr int V = Vec<T>::N;
  cg::cluster_group cl = cg::this_cluster();
  const int S = 1 << log_s;
  uint32_t *cnt = smem, *pos = smem + S;
  const int64_t cluster = blockIdx.x / cl.num_blocks();
  const int64_t r = cluster / spans;
  const int span = (int)(cluster - r * spans);
  const Row w = load_row(R, r);
  const T* x = in + r * in_rs;
  T* y = out + r * out_rs;
  const int mis = (int)(((uintptr_t)x & 15) / sizeof(T));
  const int64_t lo = (int64_t)span * cl.num_blocks() * S - mis;
  const bool hist = w.h1 > w.h0, bias = w.b1 > w.b0;
  if (hist || bias) tables(R, w, lo, log_s, cnt, pos, cl);
  const int64_t mine = lo + (int64_t)cl.block_rank() * S;
  const bool aligned = (((uintptr_t)y - (uintptr_t)mis * sizeof(T)) & 15) == 0;
  for (int i = threadIdx.x * V; i < S; i += blockDim.x * V) {
    const int64_t j = mine + i;
    if (j >= R.n) break;
    if (j >= 0 && j + V <= R.n) {
      Vec<T> t = *(const Vec<T>*)(x + j);
      const uint32_t bits = allowed_bits<V>(w.allowed, j);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float v = edit(to_f32(t.v[e]), hist ? cnt[i + e] : 0u, bias ? pos[i + e] : 0u, w, R.bias_values_dev);
        t.v[e] = (bits >> e) & 1u ? from_f32<T>(v) : from_f32<T>(-INFINITY);
      }
      if (aligned) {
        *(Vec<T>*)(y + j) = t;
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) y[j + e] = t.v[e];
      }
    } else {
      for (int e = 0; e < V; ++e) {
        if (j + e < 0 || j + e >= R.n) continue;
        const float v =
            edit(to_f32(x[j + e]), hist ? cnt[i + e] : 0u, bias ? pos[i + e] : 0u, w, R.bias_values_dev);
        y[j + e] = allowed_bits<1>(w.allowed, j + e) & 1u ? from_f32<T>(v) : from_f32<T>(-INFINITY);
      }
    }
  }
}

struct Best {
  float v;
  int64_t j;
};

// the larger value; the lower answer on equal ones
__device__ __forceinline__ void take(Best& a, float v, int64_t j) {
  if (v > a.v || (v == a.v && j < a.j)) {
    a.v = v;
    a.j = j;
  }
}

constexpr int64_t kNone = INT64_MAX;

// One cluster per row: the label's edited lower bound less the best edited upper bound among the
// other answers.
__global__ void __launch_bounds__(kThreads)
    k_answer_margin(const cf_answer_rules R, const float* __restrict__ l, int64_t l_rs, const float* __restrict__ u,
                    int64_t u_rs, const int64_t* __restrict__ labels, float* margin, int32_t* rival, int log_s,
                    int spans) {
  extern __shared__ __align__(16) uint32_t smem[];
  __shared__ Best part[kThreads / 32];
  __shared__ Best joined[kMaxCluster];
  __shared__ float label_l;
  constexpr int V = 4;
  cg::cluster_group cl = cg::this_cluster();
  const int S = 1 << log_s;
  uint32_t *cnt = smem, *pos = smem + S;
  const int64_t r = blockIdx.x / cl.num_blocks();
  const Row w = load_row(R, r);
  const float* x = u + r * u_rs;
  const int64_t label = labels[r];
  const int mis = (int)(((uintptr_t)x & 15) / 4);
  const bool hist = w.h1 > w.h0, bias = w.b1 > w.b0;
  if (threadIdx.x == 0) label_l = -INFINITY;
  cl.sync();  // the label's bound is written to the first CTA below
  Best best{-INFINITY, kNone};
  for (int span = 0; span < spans; ++span) {
    const int64_t lo = (int64_t)span * cl.num_blocks() * S - mis;
    if (hist || bias) tables(R, w, lo, log_s, cnt, pos, cl);
    const int64_t mine = lo + (int64_t)cl.block_rank() * S;
    for (int i = threadIdx.x * V; i < S; i += blockDim.x * V) {
      const int64_t j = mine + i;
      if (j >= R.n) break;
      float t[V];
      uint32_t bits = 0;
      if (j >= 0 && j + V <= R.n) {
        const float4 f = *(const float4*)(x + j);
        t[0] = f.x, t[1] = f.y, t[2] = f.z, t[3] = f.w;
        bits = allowed_bits<V>(w.allowed, j);
      } else {
        for (int e = 0; e < V; ++e) {
          const bool in = j + e >= 0 && j + e < R.n;
          t[e] = in ? x[j + e] : 0.0f;
          if (in) bits |= (allowed_bits<1>(w.allowed, j + e) & 1u) << e;
        }
      }
#pragma unroll
      for (int e = 0; e < V; ++e) {
        if (!((bits >> e) & 1u)) continue;
        const uint32_t c = hist ? cnt[i + e] : 0u, p = bias ? pos[i + e] : 0u;
        if (j + e == label) {
          float v = edit(l[r * l_rs + label], c, p, w, R.bias_values_dev);
          *cl.map_shared_rank(&label_l, 0) = v != v ? -INFINITY : v;  // a bound that is no number bounds nothing
        } else {
          const float v = edit(t[e], c, p, w, R.bias_values_dev);
          take(best, v != v ? INFINITY : v, j + e);
        }
      }
    }
    if (span + 1 < spans) __syncthreads();  // the tables are rebuilt
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    const float v = __shfl_xor_sync(0xffffffffu, best.v, off);
    const int64_t j = __shfl_xor_sync(0xffffffffu, best.j, off);
    take(best, v, j);
  }
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = best;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < (int)blockDim.x / 32; ++i) take(best, part[i].v, part[i].j);
    cl.map_shared_rank(joined, 0)[cl.block_rank()] = best;
  }
  cl.sync();
  if (cl.block_rank() == 0 && threadIdx.x == 0) {
    for (int i = 0; i < (int)cl.num_blocks(); ++i) take(best, joined[i].v, joined[i].j);
    const bool any = best.v > -INFINITY;
    const float m = label_l - best.v;
    margin[r] = m != m ? -INFINITY : m;  // an infinite bound less itself says nothing
    rival[r] = any ? (int32_t)best.j : -1;
  }
}

struct Shape {
  int threads, cluster, log_s, spans;
  size_t smem;
};

// How a row's n answers are dealt out.  A slice is a CTA's share: as small as fills the GPU
// (three CTAs of 64 KB of tables fit an SM) but at least kMinSlice answers, at most what
// kSliceBytes of tables hold.  `mis` answers of slack cover a row that starts off a 16-byte
// boundary.  one_cluster: the whole row stays with one cluster (its results are joined there).
Shape shape_for(const cf_answer_rules& R, int64_t mis, bool one_cluster) {
  Shape s;
  const int64_t n = R.n + mis;
  const bool tables = (R.tokens_dev && R.n_tokens > 0) || (R.bias_ids_dev && R.n_biases > 0);
  const int entry = R.bias_ids_dev ? 8 : 4;
  const int64_t want = R.rows * n / (148 * 3);
  int log_s = 9;
  static_assert(kMinSlice == 1 << 9, "the smallest slice");
  while ((1 << log_s) < want && ((int64_t)entry << (log_s + 1)) <= kSliceBytes) ++log_s;
  const int64_t slices = ceil_div(n, (int64_t)1 << log_s);
  s.cluster = 1;
  while (s.cluster < kMaxCluster && s.cluster < slices) s.cluster *= 2;
  if (one_cluster)  // fewer, larger slices rather than many passes of the cluster
    while (((int64_t)s.cluster << log_s) < n && ((int64_t)entry << (log_s + 1)) <= kSliceBytes) ++log_s;
  s.log_s = log_s;
  s.spans = (int)ceil_div(n, (int64_t)s.cluster << log_s);
  s.smem = tables ? (size_t)entry << log_s : 0;
  s.threads = kThreads;
  while (s.threads > 64 && s.threads * 4 > (1 << log_s)) s.threads /= 2;
  if (n <= 256) s.threads = 64;
  return s;
}

template <typename F, typename... Args>
cf_status launch(const char* what, F* kern, const Shape& s, int64_t clusters, cudaStream_t st, Args... args) {
  const int64_t blocks = clusters * s.cluster;
  CF_REQUIRE(blocks <= 0x7fffffff, CF_ERR_SHAPE, "%s: too many rows", what);
  if (s.smem > 48 * 1024) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSliceBytes);
    CF_REQUIRE(e == cudaSuccess, CF_ERR_CUDA, "%s: cudaFuncSetAttribute: %s", what, cudaGetErrorString(e));
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3((unsigned)s.threads);
  cfg.dynamicSmemBytes = s.smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)s.cluster;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
  if (e != cudaSuccess) {
    set_error("%s: %s", what, cudaGetErrorString(e));
    return CF_ERR_CUDA;
  }
  return check_launch(what);
}

cf_status check_rules(const cf_answer_rules* R, const char* what) {
  CF_REQUIRE(R, CF_ERR_NULL, "%s: NULL rules", what);
  CF_REQUIRE(R->rows >= 0 && R->n >= 0 && R->n_tokens >= 0 && R->n_biases >= 0 && R->n_masks >= 0, CF_ERR_SHAPE,
             "%s: negative size", what);
  CF_REQUIRE(R->n < 0x7fffffff && R->n_tokens < 0x7fffffff && R->n_biases < 0x7fffffff, CF_ERR_SHAPE,
             "%s: answers, tokens and biases are counted in 31 bits", what);
  CF_REQUIRE((R->tokens_dev != nullptr) == (R->token_offsets_dev != nullptr), CF_ERR_NULL,
             "%s: tokens and their offsets go together", what);
  CF_REQUIRE(R->tokens_dev || (!R->prompt_len_dev && !R->repetition_dev && !R->frequency_dev && !R->presence_dev),
             CF_ERR_NULL, "%s: penalties without a history", what);
  CF_REQUIRE((R->bias_ids_dev != nullptr) == (R->bias_offsets_dev != nullptr) &&
                 (R->bias_ids_dev != nullptr) == (R->bias_values_dev != nullptr),
             CF_ERR_NULL, "%s: bias ids, values and offsets go together", what);
  if (R->allowed_dev) {
    CF_REQUIRE(R->allowed_words >= ceil_div(R->n, 32), CF_ERR_SHAPE, "%s: %lld mask words for %lld answers", what,
               (long long)R->allowed_words, (long long)R->n);
    CF_REQUIRE(R->allowed_row_dev || R->n_masks == R->rows, CF_ERR_SHAPE, "%s: %d masks for %lld rows", what,
               (int)R->n_masks, (long long)R->rows);
  } else {
    CF_REQUIRE(!R->allowed_row_dev, CF_ERR_NULL, "%s: mask rows without masks", what);
  }
  return CF_OK;
}

template <typename T>
cf_status edit_logits(const cf_answer_rules& R, const void* in, int64_t in_rs, void* out, int64_t out_rs,
                      cudaStream_t st) {
  CF_REQUIRE(((uintptr_t)in | (uintptr_t)out) % sizeof(T) == 0, CF_ERR_SHAPE, "edit_logits: unaligned rows");
  const bool flat = (uintptr_t)in % 16 == 0 && (R.rows == 1 || in_rs * sizeof(T) % 16 == 0);
  const Shape s = shape_for(R, flat ? 0 : Vec<T>::N - 1, false);
  return launch("k_edit_logits", k_edit_logits<T>, s, R.rows * s.spans, st, R, (const T*)in, in_rs, (T*)out, out_rs,
                s.log_s, s.spans);
}

}  // namespace
}  // namespace cf

using namespace cf;

extern "C" cf_status cf_edit_logits(const cf_answer_rules* R, int32_t dtype, const void* in, int64_t in_rs, void* out,
                                    int64_t out_rs, void* stream) {
  clear_error();
  CF_INJECT("edit_logits");
  CF_TRY(check_rules(R, "edit_logits"));
  CF_REQUIRE(in_rs >= 0 && (R->rows <= 1 || out_rs >= R->n), CF_ERR_SHAPE, "edit_logits: rows of %lld overlap",
             (long long)R->n);
  CF_REQUIRE(dtype == CF_F32 || dtype == CF_BF16 || dtype == CF_F16, CF_ERR_UNSUPPORTED, "edit_logits: dtype %d",
             dtype);
  if (R->rows * R->n == 0) return CF_OK;
  CF_REQUIRE(in && out, CF_ERR_NULL, "edit_logits: NULL argument");
  if (dtype == CF_F32) return edit_logits<float>(*R, in, in_rs, out, out_rs, as_stream(stream));
  if (dtype == CF_BF16) return edit_logits<__nv_bfloat16>(*R, in, in_rs, out, out_rs, as_stream(stream));
  return edit_logits<__half>(*R, in, in_rs, out, out_rs, as_stream(stream));
}

extern "C" cf_status cf_answer_margin(const cf_answer_rules* R, const float* l, int64_t l_rs, const float* u,
                                      int64_t u_rs, const int64_t* labels, float* margin, int32_t* rival,
                                      void* stream) {
  clear_error();
  CF_INJECT("answer_margin");
  CF_TRY(check_rules(R, "answer_margin"));
  CF_REQUIRE(R->n > 0 || R->rows == 0, CF_ERR_SHAPE, "answer_margin: no answers");
  CF_REQUIRE(l_rs >= 0 && u_rs >= 0, CF_ERR_SHAPE, "answer_margin: negative row stride");
  if (R->rows == 0) return CF_OK;
  CF_REQUIRE(l && u && labels && margin && rival, CF_ERR_NULL, "answer_margin: NULL argument");
  CF_REQUIRE(((uintptr_t)l | (uintptr_t)u) % 4 == 0, CF_ERR_SHAPE, "answer_margin: unaligned rows");
  const bool flat = (uintptr_t)u % 16 == 0 && (R->rows == 1 || u_rs % 4 == 0);
  const Shape s = shape_for(*R, flat ? 0 : 3, true);
  return launch("k_answer_margin", k_answer_margin, s, R->rows, as_stream(stream), *R, l, l_rs, u, u_rs, labels, margin,
                rival, s.log_s, s.spans);
}
