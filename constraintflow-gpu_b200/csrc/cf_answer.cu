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
// Memory-bound: a row is read (and written) once, and only its mask is looked at on the way.
// What the history and the biases touch is little, so it is put right afterwards: while a CTA has
// the logits of its slice of the answers on their way into registers, it counts in shared memory
// what they say about the slice, lists the touched answers, and edits those alone.  (A lookup for
// every answer on the way, with the edit under a branch, took 228 us for 256 x 131072 bfloat16:
// some lane of nearly every warp has one.)  Tables hold 16 bits an answer (seen, and 15 bits of
// times; the place of the last bias); a row with a longer history or more biases is put right in
// two halves of 32-bit tables.  Every CTA of a row walks its history, or, where histories are
// long, a cluster shares the walk and counts through distributed shared memory.  Counts are
// integers and "the last entry" is a maximum, so the order of the atomics changes nothing.
#include <cooperative_groups.h>

#include "cf_common.cuh"
#include "cf_elem.cuh"

namespace cg = cooperative_groups;

namespace cf {
namespace {

constexpr uint32_t kSeen = 0x80000000u;  // in the history, prompt included
constexpr int kThreads = 256;
constexpr int kMaxCluster = 8;
constexpr uint32_t kList = 1024;  // touched answers of a slice that are edited from a list
constexpr int kMaxTimes = 0x7fff, kMaxPlace = 0xffff;  // of the 16-bit tables

struct Row {
  uint32_t h0, h1, answered;  // history, and where its answered part begins
  uint32_t b0, b1;            // biases
  float rep, freq, pres;
  const uint32_t* allowed;  // nullptr: everything
};

// x within 0 .. n
__device__ __forceinline__ uint32_t clamp_to(int64_t x, int64_t n) { return (uint32_t)(x < 0 ? 0 : (x > n ? n : x)); }

__device__ Row load_row(const cf_answer_rules& R, int64_t r) {
  Row w;
  w.h0 = w.h1 = w.b0 = w.b1 = 0;
  if (R.tokens_dev) {
    w.h0 = clamp_to(R.token_offsets_dev[r], R.n_tokens);
    w.h1 = max(clamp_to(R.token_offsets_dev[r + 1], R.n_tokens), w.h0);
  }
  w.answered = w.h0 + (R.prompt_len_dev ? (uint32_t)max(R.prompt_len_dev[r], 0) : 0u);
  if (R.bias_ids_dev) {
    w.b0 = clamp_to(R.bias_offsets_dev[r], R.n_biases);
    w.b1 = max(clamp_to(R.bias_offsets_dev[r + 1], R.n_biases), w.b0);
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

__device__ __noinline__ float edit(float v, uint32_t c, uint32_t bias_at, const Row& w,
                                   const float* biases) {
  if (c) {
    v = v > 0.0f ? __fdiv_rn(v, w.rep) : __fmul_rn(v, w.rep);
    const uint32_t times = c & ~kSeen;
    if (times) v = __fsub_rn(__fsub_rn(v, __fmul_rn(w.freq, (float)times)), w.pres);
  }
  if (bias_at) v = __fadd_rn(v, biases[w.b0 + bias_at - 1]);
  return v;
}

// A slice's tables: S entries of 16 bits each or, wide, half of them of 32 bits; and the list of
// its touched entries.
struct Tables {
  uint32_t *cnt, *pos;
  uint32_t* listed;  // touched entries; the list holds the first kList
  uint16_t* list;    // an entry; kBias: because of a bias
  int log_s;
  bool wide, hist, bias;
};
constexpr uint32_t kBias = 0x8000u;

// Another CTA's tables.
__device__ __forceinline__ Tables of_rank(const Tables& t, cg::cluster_group& cl, uint32_t rank) {
  Tables o = t;
  o.cnt = cl.map_shared_rank(t.cnt, rank);
  o.pos = cl.map_shared_rank(t.pos, rank);
  o.listed = cl.map_shared_rank(t.listed, rank);
  o.list = cl.map_shared_rank(t.list, rank);
  return o;
}

__device__ __forceinline__ void put(const Tables& t, uint32_t i) {
  const uint32_t at = atomicAdd(t.listed, 1u);
  if (at < kList) t.list[at] = (uint16_t)i;
}

// Count a token of entry i of the slice (k: of its table), listed at the first.
__device__ __forceinline__ void add_times(const Tables& t, uint32_t i, uint32_t k, bool answered) {
  uint32_t old;
  if (t.wide) {
    old = answered ? atomicAdd(t.cnt + k, 1u) : atomicOr(t.cnt + k, kSeen);
  } else {
    const uint32_t sh = (k & 1) * 16;
    old = answered ? atomicAdd(t.cnt + (k >> 1), 1u << sh) : atomicOr(t.cnt + (k >> 1), 0x8000u << sh);
    old = (old >> sh) & 0xffffu;
  }
  if (old == 0) put(t, i);
}

__device__ __forceinline__ void max_place(const Tables& t, uint32_t i, uint32_t k, uint32_t place) {
  uint32_t first;
  if (t.wide) {
    first = atomicMax(t.pos + k, place);
  } else {
    const uint32_t sh = (k & 1) * 16;
    uint32_t old = *(volatile uint32_t*)(t.pos + (k >> 1));
    for (;;) {
      first = (old >> sh) & 0xffffu;
      if (first >= place) break;
      const uint32_t seen = atomicCAS(t.pos + (k >> 1), old, (old & ~(0xffffu << sh)) | (place << sh));
      if (seen == old) break;
      old = seen;
    }
  }
  if (first == 0) put(t, i | kBias);
}

__device__ __forceinline__ void sync_all(cg::cluster_group& cl) {
  if (cl.num_blocks() > 1)
    cl.sync();
  else
    __syncthreads();
}

// f(list[i], i) for this CTA's share of [from, end), kBatch loads in flight.
template <typename F>
__device__ __forceinline__ void walk(const int32_t* list, uint32_t from, uint32_t end, uint32_t nc, uint32_t rank,
                                     F&& f) {
  constexpr int kBatch = 4;
  const uint32_t step = nc * kThreads;
  for (uint32_t i = from + rank * kThreads + threadIdx.x; i < end; i += kBatch * step) {
    int32_t j[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) j[b] = i + b * step < end ? list[i + b * step] : -1;
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
      if (j[b] >= 0) f(j[b], i + b * step);
  }
}

// The slices [lo + rank * S, + S) of a cluster's CTAs; lo counts answers and may start before the
// first (the row's own alignment).  Wide: half `side` of each slice.
struct Span {
  int32_t lo, n;
  int side;
};

// Fill the tables.  Every CTA of the cluster calls it.
__device__ __forceinline__ void fill(const cf_answer_rules& R, const Row& w, const Tables& t, const Span& s,
                                     cg::cluster_group& cl) {
  const uint32_t S = 1u << t.log_s, nc = cl.num_blocks(), rank = cl.block_rank();
  for (uint32_t i = threadIdx.x * 4; i < S / 2; i += kThreads * 4) {
    if (t.hist) *(uint4*)(t.cnt + i) = make_uint4(0, 0, 0, 0);
    if (t.bias) *(uint4*)(t.pos + i) = make_uint4(0, 0, 0, 0);
  }
  if (threadIdx.x == 0) *t.listed = 0;
  sync_all(cl);
  const uint32_t mask = (S >> (t.wide ? 1 : 0)) - 1;
  // f(owner's tables, entry of the slice, of the table) where answer j is of this span and half
  auto at = [&](int32_t j, auto&& f) {
    const uint32_t rel = (uint32_t)(j - s.lo);
    if (j < 0 || j >= s.n || rel >= nc << t.log_s) return;
    const uint32_t i = rel & (S - 1);
    if (t.wide && (int)(i >> (t.log_s - 1)) != s.side) return;
    if (nc > 1)
      f(of_rank(t, cl, rel >> t.log_s), i, i & mask);
    else
      f(t, i, i & mask);
  };
  walk(R.tokens_dev, w.h0, w.h1, nc, rank, [&](int32_t j, uint32_t h) {
    at(j, [&](const Tables& o, uint32_t i, uint32_t k) { add_times(o, i, k, h >= w.answered); });
  });
  walk(R.bias_ids_dev, w.b0, w.b1, nc, rank, [&](int32_t j, uint32_t b) {
    at(j, [&](const Tables& o, uint32_t i, uint32_t k) { max_place(o, i, k, b - w.b0 + 1u); });
  });
  sync_all(cl);
}

// Entry i of the slice: its count (seen in the highest bit) and the place of its bias, or 0.
__device__ __forceinline__ void look(const Tables& t, uint32_t i, uint32_t& c, uint32_t& p) {
  c = p = 0;
  if (t.wide) {
    i &= (1u << (t.log_s - 1)) - 1;
    if (t.hist) c = t.cnt[i];
    if (t.bias) p = t.pos[i];
  } else {
    const uint32_t sh = (i & 1) * 16;
    if (t.hist) {
      c = (t.cnt[i >> 1] >> sh) & 0xffffu;
      c = (c & 0x7fffu) | (c & 0x8000u) << 16;
    }
    if (t.bias) p = (t.pos[i >> 1] >> sh) & 0xffffu;
  }
}

// Entry at place `at` of the list with what touches it; false: listed for its bias, and for its
// count as well.
__device__ __forceinline__ bool listed_entry(const Tables& t, uint32_t at, uint32_t& i, uint32_t& c, uint32_t& p) {
  const uint32_t e = t.list[at];
  i = e & ~kBias;
  look(t, i, c, p);
  return !(e & kBias) || c == 0;
}

// bit e: entry i + e of four is touched
__device__ __forceinline__ uint32_t touched4(const Tables& t, uint32_t i) {
  if (t.wide) {
    i &= (1u << (t.log_s - 1)) - 1;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (t.hist) v = *(const uint4*)(t.cnt + i);
    if (t.bias) {
      const uint4 q = *(const uint4*)(t.pos + i);
      v.x |= q.x, v.y |= q.y, v.z |= q.z, v.w |= q.w;
    }
    return (v.x != 0) | (v.y != 0) << 1 | (v.z != 0) << 2 | (v.w != 0) << 3;
  }
  uint2 v = make_uint2(0, 0);
  if (t.hist) v = *(const uint2*)(t.cnt + i / 2);
  if (t.bias) {
    const uint2 q = *(const uint2*)(t.pos + i / 2);
    v.x |= q.x, v.y |= q.y;
  }
  if (!(v.x | v.y)) return 0;
  return ((v.x & 0xffffu) != 0) | (v.x >> 16 != 0) << 1 | ((v.y & 0xffffu) != 0) << 2 | (v.y >> 16 != 0) << 3;
}

__device__ __forceinline__ Tables tables_of(const cf_answer_rules& R, const Row& w, uint32_t* smem, int log_s) {
  const uint32_t words = 1u << (log_s - 1);
  Tables t;
  t.log_s = log_s;
  t.hist = w.h1 > w.h0;
  t.bias = w.b1 > w.b0;
  t.wide = w.h1 - w.h0 > kMaxTimes || w.b1 - w.b0 > kMaxPlace;
  t.cnt = smem;
  t.pos = smem + words;
  t.listed = smem + words * (R.bias_ids_dev ? 2 : 1);
  t.list = (uint16_t*)(t.listed + 4);
  return t;
}

template <typename T>
struct alignas(16) Vec {
  static constexpr int N = 16 / sizeof(T);
  T v[N];
};

// The bits of `allowed` for N answers from j on, all of them answers.
template <int N>
__device__ __forceinline__ uint32_t allowed_bits(const uint32_t* allowed, int32_t j) {
  if (!allowed) return 0xffffffffu;
  const int sh = (int)(j & 31);
  uint32_t bits = allowed[j >> 5] >> sh;
  if (sh + N > 32) bits |= allowed[(j >> 5) + 1] << (32 - sh);
  return bits;
}

// Elements [j, j + V) of a row of n: whole vectors where they are, zeros outside.
template <typename T>
__device__ __forceinline__ Vec<T> load_vec(const T* x, int32_t j, int32_t n) {
  constexpr int V = Vec<T>::N;
  if (j >= 0 && j + V <= n) return *(const Vec<T>*)(x + j);
  Vec<T> t;
#pragma unroll
  for (int e = 0; e < V; ++e) t.v[e] = j + e >= 0 && j + e < n ? x[j + e] : from_f32<T>(0.0f);
  return t;
}

// bit e: answer j + e exists and is allowed
template <int V>
__device__ __forceinline__ uint32_t open_bits(const uint32_t* allowed, int32_t j, int32_t n) {
  if (j >= 0 && j + V <= n) return allowed_bits<V>(allowed, j);
  uint32_t bits = 0;
  for (int e = 0; e < V; ++e)
    if (j + e >= 0 && j + e < n) bits |= (allowed_bits<1>(allowed, j + e) & 1u) << e;
  return bits;
}

// One CTA per slice of a row, `spans` clusters of slices a row.  mis: answers between the 16-byte
// boundary below the row's start and the start, so that whole vectors are aligned.  A slice is
// kVpt vectors a thread.
template <typename T, int kVpt>
__global__ void __launch_bounds__(kThreads, 4)
    k_edit_logits(const cf_answer_rules R, const T* in, int64_t in_rs, T* out, int64_t out_rs, int log_s, int spans) {
  extern __shared__ __align__(16) uint32_t smem[];
  constexpr int V = Vec<T>::N;
  cg::cluster_group cl = cg::this_cluster();
  const int nc = (int)cl.num_blocks(), n = (int)R.n;
  const int64_t cluster = blockIdx.x / nc;
  const int64_t r = cluster / spans;
  const T* x = in + r * in_rs;
  T* y = out + r * out_rs;
  const int mis = (int)(((uintptr_t)x & 15) / sizeof(T));
  Span s;
  s.lo = (((int)(cluster - r * spans) * nc) << log_s) - mis;
  s.n = n;
  s.side = 0;
  const int mine = s.lo + ((int)cl.block_rank() << log_s);
  Vec<T> t[kVpt];
#pragma unroll
  for (int i = 0; i < kVpt; ++i) {
    const int j = mine + (i * kThreads + (int)threadIdx.x) * V;
    if (j < n) t[i] = load_vec(x, j, n);
  }
  const Row w = load_row(R, r);
  const Tables tab = tables_of(R, w, smem, log_s);
  const bool aligned = (((uintptr_t)y - (uintptr_t)mis * sizeof(T)) & 15) == 0;
  auto store = [&](int j, const Vec<T>& v) {
    if (aligned && j >= 0 && j + V <= n) {
      *(Vec<T>*)(y + j) = v;
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (j + e >= 0 && j + e < n) y[j + e] = v.v[e];
    }
  };
  const bool touch = tab.hist || tab.bias;
  if (touch) fill(R, w, tab, s, cl);
#pragma unroll
  for (int i = 0; i < kVpt; ++i) {
    const int j = mine + (i * kThreads + (int)threadIdx.x) * V;
    if (j >= n) break;
    const uint32_t bits = open_bits<V>(w.allowed, j, n);
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (!((bits >> e) & 1u)) t[i].v[e] = from_f32<T>(-INFINITY);
    store(j, t[i]);
  }
  if (!touch) return;
  // Answers that are not allowed stay as they are; the others' logits are as they were, also
  // where the result takes the logits' place.
  for (;;) {
    __syncthreads();
    const uint32_t listed = *tab.listed;
    uint32_t i, c, p;
    if (listed <= kList) {
      for (uint32_t k = threadIdx.x; k < listed; k += kThreads) {
        if (!listed_entry(tab, k, i, c, p)) continue;
        const int j = mine + (int)i;
        if (!(allowed_bits<1>(w.allowed, j) & 1u)) continue;
        y[j] = from_f32<T>(edit(to_f32(x[j]), c, p, w, R.bias_values_dev));
      }
    } else {  // many: vector by vector
#pragma unroll 1
      for (int k = 0; k < kVpt; ++k) {
        i = (k * kThreads + threadIdx.x) * V;
        const int j = mine + (int)i;
        if (j >= n || (tab.wide && (int)(i >> (log_s - 1)) != s.side)) continue;
        const uint32_t bits = open_bits<V>(w.allowed, j, n);
        Vec<T> v = load_vec(x, j, n);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          look(tab, i + e, c, p);
          if (!((bits >> e) & 1u))
            v.v[e] = from_f32<T>(-INFINITY);
          else if (c | p)
            v.v[e] = from_f32<T>(edit(to_f32(v.v[e]), c, p, w, R.bias_values_dev));
        }
        store(j, v);
      }
    }
    if (!tab.wide || s.side == 1) return;
    s.side = 1;
    sync_all(cl);  // the tables are filled anew
    fill(R, w, tab, s, cl);
  }
}

struct Best {
  float v;
  int32_t j;
};

// the larger value; the lower answer on equal ones
__device__ __forceinline__ void take(Best& a, float v, int32_t j) {
  if (v > a.v || (v == a.v && j < a.j)) {
    a.v = v;
    a.j = j;
  }
}

constexpr int32_t kNone = INT32_MAX;

// One cluster per row: the label's edited lower bound less the best edited upper bound among the
// other answers.
template <int kVpt>
__global__ void __launch_bounds__(kThreads, 3)
    k_answer_margin(const cf_answer_rules R, const float* __restrict__ l, int64_t l_rs, const float* __restrict__ u,
                    int64_t u_rs, const int64_t* __restrict__ labels, float* margin, int32_t* rival, int log_s,
                    int spans) {
  extern __shared__ __align__(16) uint32_t smem[];
  __shared__ Best part[kThreads / 32];
  __shared__ Best joined[kMaxCluster];
  __shared__ float label_l;
  constexpr int V = 4;
  cg::cluster_group cl = cg::this_cluster();
  const int nc = (int)cl.num_blocks(), n = (int)R.n;
  const int64_t r = blockIdx.x / nc;
  const float* x = u + r * u_rs;
  const int mis = (int)(((uintptr_t)x & 15) / 4);
  Vec<float> t[kVpt];
  auto first = [&](int span) {  // answer of this CTA's slice
    return ((span * nc + (int)cl.block_rank()) << log_s) - mis;
  };
  auto load = [&](int span) {
#pragma unroll
    for (int i = 0; i < kVpt; ++i) {
      const int j = first(span) + (i * kThreads + (int)threadIdx.x) * V;
      if (j < n) t[i] = load_vec(x, j, n);
    }
  };
  load(0);
  const Row w = load_row(R, r);
  const int label = labels[r] >= 0 && labels[r] < n ? (int)labels[r] : INT32_MIN;  // or no answer
  const Tables tab = tables_of(R, w, smem, log_s);
  const bool touch = tab.hist || tab.bias;
  if (threadIdx.x == 0) label_l = -INFINITY;
  sync_all(cl);  // the label's bound is written to the first CTA below
  Best best{-INFINITY, kNone};
  // allowed answer j of upper bound `bound` with what touches it
  auto answer = [&](int j, float bound, uint32_t c, uint32_t p) {
    if (j == label) {
      float v = l[r * l_rs + label];
      if (c | p) v = edit(v, c, p, w, R.bias_values_dev);
      *cl.map_shared_rank(&label_l, 0) = v != v ? -INFINITY : v;  // a bound that is no number bounds nothing
    } else {
      const float v = c | p ? edit(bound, c, p, w, R.bias_values_dev) : bound;
      take(best, v != v ? INFINITY : v, j);
    }
  };
  for (int span = 0; span < spans; ++span) {
    Span s;
    s.lo = ((span * nc) << log_s) - mis;
    s.n = n;
    const int mine = first(span);
    for (s.side = 0; s.side < (tab.wide ? 2 : 1); ++s.side) {
      if (touch) {
        if (span + s.side > 0) sync_all(cl);  // the tables are filled anew
        fill(R, w, tab, s, cl);
      }
      // what nothing touches
#pragma unroll
      for (int i = 0; i < kVpt; ++i) {
        const uint32_t at = (i * kThreads + threadIdx.x) * V;
        const int j = mine + (int)at;
        if (j >= n || (tab.wide && (int)(at >> (log_s - 1)) != s.side)) continue;
        uint32_t bits = open_bits<V>(w.allowed, j, n);
        if (touch) bits &= ~touched4(tab, at);
        const uint32_t own = (uint32_t)label - (uint32_t)j;
        if (own < V && (bits >> own & 1u)) {
          answer(label, 0.0f, 0u, 0u);
          bits &= ~(1u << own);
        }
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float v = t[i].v[e] != t[i].v[e] ? INFINITY : t[i].v[e];
          if ((bits >> e & 1u) && v > best.v) best = Best{v, j + e};  // ascending: the lowest of equal ones
        }
      }
      if (!touch) continue;
      const uint32_t listed = *tab.listed;
      uint32_t i, c, p;
      if (listed <= kList) {
        for (uint32_t k = threadIdx.x; k < listed; k += kThreads) {
          if (!listed_entry(tab, k, i, c, p)) continue;
          const int j = mine + (int)i;
          if (allowed_bits<1>(w.allowed, j) & 1u) answer(j, x[j], c, p);
        }
      } else {  // many: entry by entry
        for (i = threadIdx.x; i < 1u << log_s; i += kThreads) {
          const int j = mine + (int)i;
          if (j < 0 || j >= n || (tab.wide && (int)(i >> (log_s - 1)) != s.side)) continue;
          look(tab, i, c, p);
          if ((c | p) && (allowed_bits<1>(w.allowed, j) & 1u)) answer(j, x[j], c, p);
        }
      }
    }
    if (span + 1 < spans) load(span + 1);
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    const float v = __shfl_xor_sync(0xffffffffu, best.v, off);
    const int32_t j = __shfl_xor_sync(0xffffffffu, best.j, off);
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
    rival[r] = any ? best.j : -1;
  }
}

struct Shape {
  int vpt, cluster, log_s, spans;
  size_t smem;
};

// How a row's n answers are dealt out to slices of 256 vpt vectors of V answers.  A slice is as
// large (up to 8192 answers) as still makes four CTAs an SM; `mis` answers of slack cover a row that
// starts off a 16-byte boundary.  one_cluster: the whole row stays with one cluster (its results
// are joined there).  Else a cluster shares the walk through histories that are long on average.
constexpr int64_t kLongHistory = 1024;
Shape shape_for(const cf_answer_rules& R, int V, int64_t mis, bool one_cluster) {
  const int kMaxVpt = 32 / V;  // 8192 answers
  Shape s;
  const int64_t n = R.n + mis;
  const bool hist = R.tokens_dev && R.n_tokens > 0, bias = R.bias_ids_dev && R.n_biases > 0;
  s.vpt = 1;
  while (s.vpt < kMaxVpt && ceil_div(n, (int64_t)kThreads * V * s.vpt * 2) * R.rows >= 148 * 4) s.vpt *= 2;
  const int64_t slice = (int64_t)kThreads * V * s.vpt, slices = ceil_div(n, slice);
  s.log_s = 0;
  while (((int64_t)1 << s.log_s) < slice) ++s.log_s;
  s.cluster = 1;
  if (one_cluster || (hist && R.n_tokens / R.rows > kLongHistory))
    while (s.cluster < kMaxCluster && s.cluster < slices) s.cluster *= 2;
  s.spans = (int)ceil_div(slices, s.cluster);
  s.smem = (hist || bias) ? (size_t)slice * (R.bias_ids_dev ? 4 : 2) + 16 + kList * 2 : 0;
  return s;
}

template <typename F, typename... Args>
cf_status launch(const char* what, F* kern, const Shape& s, int64_t clusters, cudaStream_t st, Args... args) {
  const int64_t blocks = clusters * s.cluster;
  CF_REQUIRE(blocks <= 0x7fffffff, CF_ERR_SHAPE, "%s: too many rows", what);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(kThreads);
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
  CF_REQUIRE(R->n <= 1 << 30 && R->n_tokens <= 1 << 30 && R->n_biases <= 1 << 30, CF_ERR_SHAPE,
             "%s: at most 2^30 answers, tokens and biases", what);
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
  const Shape s = shape_for(R, Vec<T>::N, flat ? 0 : Vec<T>::N - 1, false);
  auto* kern = s.vpt == 1   ? k_edit_logits<T, 1>
               : s.vpt == 2 ? k_edit_logits<T, 2>
               : s.vpt == 4 ? k_edit_logits<T, 4>
                            : k_edit_logits<T, 32 / Vec<T>::N>;
  return launch("k_edit_logits", kern, s, R.rows * s.spans, st, R, (const T*)in, in_rs, (T*)out, out_rs, s.log_s,
                s.spans);
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
  const Shape s = shape_for(*R, 4, flat ? 0 : 3, true);
  auto* kern = s.vpt == 1   ? k_answer_margin<1>
               : s.vpt == 2 ? k_answer_margin<2>
               : s.vpt == 4 ? k_answer_margin<4>
                            : k_answer_margin<8>;
  return launch("k_answer_margin", kern, s, R->rows, as_stream(stream), *R, l, l_rs, u, u_rs, labels, margin, rival,
                s.log_s, s.spans);
}
