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
// What the history and the biases touch is little and is put right from their side, in the result
// that the stream has left in the cache.  For 256 x 131072 bfloat16 and 1024 tokens a row: a lookup
// for every answer on the way 228 us (some lane of nearly every warp edits), edits of each slice in
// shared memory on its way 50, the stream 21 (134 MB: 0.98 of a copy's rate, partly from the cache; 26
// with a cold one) and behind it the edits 12: random reads and writes of single answers, each waiting on the
// last for its address.
//
// Short histories go into a hash table of the answers they touch, one CTA a row, whatever the row's
// length.  Long ones are counted slice by slice in tables of all answers: 16 bits an answer, seen
// and 15 bits of times, and a bit for its having a bias; what bounds them is the walk over the history, once a
// slice, and its atomics on the answers that come again and again (33 rows of 100003, up to 32768
// tokens, the first slice 0.55 of them: 35 us, 6 of them the stream; smaller slices walk more
// often: 45 us in twice as many).
// Which of the (few) biases of one answer is the last is found by comparing them.  A row with more
// than kMaxBiases biases, or one answer more than kTimes times, is done in quarters of a
// slice, with 32 bits for the times and 32 for the place of the last bias.  Counts are integers
// and "the last entry" is a maximum, so the order of the atomics changes nothing.
#include <cooperative_groups.h>

#include "cf_common.cuh"
#include "cf_elem.cuh"

namespace cg = cooperative_groups;

namespace cf {
namespace {

// of a table's entry, 16 bits (wide: the highest of 32)
constexpr uint32_t kSeen = 0x8000u, kTimes = 0x7fffu, kWideTimes = 0x7fffffffu;
constexpr uint32_t kMaxBiases = 1024;
// Touched answers of a slice are edited from a list where a row has at most kListed tokens; a longer
// row's would wait for one another at the list's counter, and are many anyhow.
constexpr uint32_t kList = 1024, kListed = 4096;

struct Row {
  uint32_t h0, h1, answered;  // history, and where its answered part begins
  uint32_t b0, b1;            // biases
  float rep, freq, pres;
  const uint32_t* allowed;  // nullptr: everything
};

// x within 0 .. n
__device__ __forceinline__ uint32_t clamp_to(int64_t x, int64_t n) { return (uint32_t)(x < 0 ? 0 : (x > n ? n : x)); }

__device__ __forceinline__ const uint32_t* mask_of(const cf_answer_rules& R, int64_t r) {
  if (!R.allowed_dev) return nullptr;
  const int64_t m = R.allowed_row_dev ? (int64_t)R.allowed_row_dev[r] : r;
  return m >= 0 && m < R.n_masks ? (const uint32_t*)R.allowed_dev + m * R.allowed_words : nullptr;
}

__device__ __forceinline__ Row load_row(const cf_answer_rules& R, int64_t r) {
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
  w.allowed = mask_of(R, r);
  return w;
}

__device__ __forceinline__ bool is_allowed(const uint32_t* allowed, int j) {
  return !allowed || (allowed[j >> 5] >> (j & 31) & 1u);
}

// The bits of `allowed` for answers j .. j+N-1, 0 for those outside 0 .. n-1.
template <int N>
__device__ __forceinline__ uint32_t open_bits(const uint32_t* allowed, int j, int n) {
  uint32_t bits = 0;
  if (j >= 0 && j + N <= n) {
    if (!allowed) return (1u << N) - 1;
    const int sh = j & 31;
    bits = allowed[j >> 5] >> sh;
    if (sh + N > 32) bits |= allowed[(j >> 5) + 1] << (32 - sh);
    return bits & ((1u << N) - 1);
  }
  for (int e = 0; e < N; ++e)
    if (j + e >= 0 && j + e < n && is_allowed(allowed, j + e)) bits |= 1u << e;
  return bits;
}

// c: times, kSeen (in the history, the given part included)
__device__ __noinline__ float edit(float v, bool seen, uint32_t times, float rep, float freq, float pres) {
  if (seen) {
    v = v > 0.0f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
    if (times) v = __fsub_rn(__fsub_rn(v, __fmul_rn(freq, (float)times)), pres);
  }
  return v;
}

// ------------------------------------------------------------------ what a row touches
// Shared memory of a CTA that edits a slice of 1 << log_s answers.
struct Tables {
  uint32_t* words;   // 16-bit entries of a slice; wide: 32-bit counts, then places, of a quarter
  uint32_t* biased;  // a bit for each answer
  uint32_t* over;    // an answer has more than kTimes
  uint32_t* listed;  // touched answers, the list holds the first kList
  uint16_t* list;    // places in the slice (quarter)
  int32_t* ids;      // the row's biases (not wide)
  int log_s;
  bool wide, listing;
};

constexpr int kMostSmem = (2 << 15) + (1 << 12) + 16 + kList * 2 + kMaxBiases * 4;  // of slices of 32768

size_t tables_bytes(int log_s) {
  return ((size_t)2 << log_s) + ((size_t)1 << (log_s - 3)) + 16 + kList * 2 + kMaxBiases * 4;
}

__device__ __forceinline__ Tables tables_of(const Row& w, uint32_t* smem, int log_s) {
  Tables t;
  t.words = smem;
  t.biased = smem + (1u << (log_s - 1));
  t.over = t.biased + (1u << (log_s - 5));
  t.listed = t.over + 1;
  t.list = (uint16_t*)(t.over + 4);
  t.ids = (int32_t*)(t.list + kList);
  t.listing = w.h1 - w.h0 <= kListed;
  t.log_s = log_s;
  t.wide = w.b1 - w.b0 > kMaxBiases;
  return t;
}

// f(list[i], i) over [from, end) by the CTA, kBatch loads in flight a thread.
template <int kBatch, typename F>
__device__ __forceinline__ void walk(const int32_t* list, uint32_t from, uint32_t end, F&& f) {
  const uint32_t step = blockDim.x;
  for (uint32_t i = from + threadIdx.x; i < end; i += kBatch * step) {
    int32_t j[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) j[b] = i + b * step < end ? list[i + b * step] : -1;
#pragma unroll
    for (int b = 0; b < kBatch; ++b)
      if (j[b] >= 0) f(j[b], i + b * step);
  }
}

// The counts of answers [lo, lo + size) from the row's history.
// False: to be done wide.
__device__ __forceinline__ bool count(const cf_answer_rules& R, const Row& w, const Tables& t, int lo, uint32_t size) {
  const uint32_t words = t.wide ? size : (size + 1) / 2;
  for (uint32_t i = threadIdx.x * 4; i < words; i += blockDim.x * 4) {
    *(uint4*)(t.words + i) = make_uint4(0, 0, 0, 0);
    if (t.wide) *(uint4*)(t.words + (1u << (t.log_s - 2)) + i) = make_uint4(0, 0, 0, 0);
  }
  if (w.b1 > w.b0)
    for (uint32_t i = threadIdx.x; i < (size + 31) / 32; i += blockDim.x) t.biased[i] = 0;
  if (threadIdx.x == 0) *t.over = *t.listed = 0;
  if (!t.wide)
    for (uint32_t i = w.b0 + threadIdx.x; i < w.b1; i += blockDim.x) t.ids[i - w.b0] = R.bias_ids_dev[i];
  __syncthreads();
  if (!t.wide && !t.listing && w.h1 - min(w.h1, w.answered) <= kTimes) {  // nothing to be told by the old count
    walk<8>(R.tokens_dev, w.h0, w.h1, [&](int32_t j, uint32_t h) {
      const uint32_t k = (uint32_t)(j - lo), sh = (k & 1) * 16;
      if (k >= size) return;
      if (h >= w.answered)
        atomicAdd(t.words + (k >> 1), 1u << sh);
      else
        atomicOr(t.words + (k >> 1), kSeen << sh);
    });
    __syncthreads();
    return true;
  }
  walk<8>(R.tokens_dev, w.h0, w.h1, [&](int32_t j, uint32_t h) {
    const uint32_t k = (uint32_t)(j - lo);
    if (k >= size) return;
    const bool answered = h >= w.answered;
    uint32_t old;
    if (t.wide) {
      old = answered ? atomicAdd(t.words + k, 1u) : atomicOr(t.words + k, kSeen << 16);
    } else {
      const uint32_t sh = (k & 1) * 16;
      old = answered ? atomicAdd(t.words + (k >> 1), 1u << sh) : atomicOr(t.words + (k >> 1), kSeen << sh);
      old = old >> sh & 0xffffu;
      if (answered && (old & kTimes) == kTimes) *(volatile uint32_t*)t.over = 1;
    }
    if (t.listing && old == 0) {
      const uint32_t at = atomicAdd(t.listed, 1u);
      if (at < kList) t.list[at] = (uint16_t)k;
    }
  });
  if (t.wide)
    walk<4>(R.bias_ids_dev, w.b0, w.b1, [&](int32_t j, uint32_t b) {
      const uint32_t k = (uint32_t)(j - lo);
      if (k < size) atomicMax(t.words + (1u << (t.log_s - 2)) + k, b - w.b0 + 1u);
    });
  __syncthreads();
  return t.wide || *t.over == 0;
}

// Entry k: 0 if the history does not hold it, else kSeen or its times, in 32 bits.
__device__ __forceinline__ uint32_t entry(const Tables& t, uint32_t k) {
  return t.wide ? t.words[k] : t.words[k >> 1] >> (k & 1) * 16 & 0xffffu;
}
__device__ __forceinline__ uint32_t times(const Tables& t, uint32_t entry) {
  return entry & (t.wide ? kWideTimes : kTimes);
}
__device__ __forceinline__ bool is_biased(const Row& w, const Tables& t, uint32_t k) {
  return w.b1 > w.b0 && (t.biased[k >> 5] >> (k & 31) & 1u);
}

// f(answer, seen, times, bias) for each answer of the slice that has a bias; it is marked.
template <typename F>
__device__ __forceinline__ void for_biased(const cf_answer_rules& R, const Row& w, const Tables& t, int lo,
                                           uint32_t size, F&& f) {
  for (uint32_t b = w.b0 + threadIdx.x; b < w.b1; b += blockDim.x) {
    const int j = t.wide ? R.bias_ids_dev[b] : t.ids[b - w.b0];
    const uint32_t k = (uint32_t)(j - lo);
    if (k >= size) continue;
    bool last = true;
    if (t.wide) {
      last = t.words[(1u << (t.log_s - 2)) + k] == b - w.b0 + 1u;
    } else {
      const uint32_t n = w.b1 - w.b0;
#pragma unroll 4
      for (uint32_t i = b - w.b0 + 1; i < n; ++i) last &= t.ids[i] != j;
    }
    if (!last) continue;
    atomicOr(t.biased + (k >> 5), 1u << (k & 31));
    const uint32_t c = entry(t, k);
    f(j, c != 0, times(t, c), R.bias_values_dev[b]);
  }
}

// f(answer, times, x[answer]) for each allowed answer of the slice that the history holds and
// that has no bias; several a thread at a time, their loads of x in flight together.
template <typename T, typename F>
__device__ __forceinline__ void for_seen(const Row& w, const Tables& t, int lo, uint32_t size, const T* x, F&& f) {
  if (t.listing && *t.listed <= kList) {
    constexpr int kBatch = 4;
    const uint32_t n = *t.listed;
    for (uint32_t i = threadIdx.x; i < n; i += kBatch * blockDim.x) {
      uint32_t k[kBatch], c[kBatch];
      T v[kBatch];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const bool ok = i + b * blockDim.x < n;
        k[b] = ok ? t.list[i + b * blockDim.x] : 0u;
        c[b] = ok && !is_biased(w, t, k[b]) && is_allowed(w.allowed, lo + (int)k[b]) ? entry(t, k[b]) : 0u;
        v[b] = c[b] ? x[lo + (int)k[b]] : from_f32<T>(0.0f);
      }
#pragma unroll
      for (int b = 0; b < kBatch; ++b)
        if (c[b]) f(lo + (int)k[b], times(t, c[b]), to_f32(v[b]));
    }
    return;
  }
  for (uint32_t k0 = threadIdx.x * 8; k0 < size; k0 += blockDim.x * 8) {
    uint32_t c[8];
    if (t.wide) {
      *(uint4*)c = *(const uint4*)(t.words + k0);
      *(uint4*)(c + 4) = *(const uint4*)(t.words + k0 + 4);
    } else {
      const uint4 d = *(const uint4*)(t.words + k0 / 2);
      if (!(d.x | d.y | d.z | d.w)) continue;
      const uint32_t h[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
      for (int b = 0; b < 8; ++b) c[b] = h[b / 2] >> (b & 1) * 16 & 0xffffu;
    }
    T v[8];
#pragma unroll
    for (int b = 0; b < 8; ++b) {
      const int j = lo + (int)k0 + b;
      if (k0 + b >= size || (c[b] && (is_biased(w, t, k0 + b) || !is_allowed(w.allowed, j)))) c[b] = 0;
      v[b] = c[b] ? x[j] : from_f32<T>(0.0f);
    }
#pragma unroll
    for (int b = 0; b < 8; ++b)
      if (c[b]) f(lo + (int)k0 + b, times(t, c[b]), to_f32(v[b]));
  }
}

// What a short row touches: open addressing over the answers.
// kShort tokens and biases of a row at most, kMarginShort for its margin (whose CTAs, four an SM, all run at
// once, and read through what the tables leave of the L1 cache).
constexpr uint32_t kSlots = 4096, kShort = 2800, kMarginSlots = 2048, kMarginShort = 1536;

struct Hash {
  int log_n;  // 1 << log_n slots, twice a row's tokens and biases where there are that many
  uint32_t *key, *cnt, *pos;  // answer + 1 (0: free); times and, highest bit, seen; place of the last bias
  uint32_t* listed;
  uint16_t* list;  // slots in use
};

constexpr size_t hash_bytes(uint32_t slots, uint32_t most) { return slots * 12 + 16 + most * 2; }

template <uint32_t kMost>
__device__ __forceinline__ bool is_short(const Row& w) {
  return w.h1 - w.h0 + (w.b1 - w.b0) <= kMost;
}

__device__ __forceinline__ Hash hash_of(const Row& w, uint32_t* smem, uint32_t slots) {
  Hash h;
  h.log_n = min(max(33 - __clz((int)(w.h1 - w.h0 + (w.b1 - w.b0))), 6), 31 - __clz((int)slots));
  h.key = smem;
  h.cnt = smem + (1u << h.log_n);
  h.pos = smem + (2u << h.log_n);
  h.listed = smem + (3u << h.log_n);
  h.list = (uint16_t*)(h.listed + 4);
  return h;
}

// The slot of answer j; the first to come to it lists it.
__device__ __forceinline__ uint32_t slot_of(const Hash& h, uint32_t j) {
  uint32_t s = j * 2654435761u >> (32 - h.log_n);  // by the golden ratio
  for (;;) {
    const uint32_t old = atomicCAS(h.key + s, 0u, j + 1u);
    if (old == 0u) {
      h.list[atomicAdd(h.listed, 1u)] = (uint16_t)s;
      return s;
    }
    if (old == j + 1u) return s;
    s = (s + 1) & ((1u << h.log_n) - 1);
  }
}

// Whether the table holds answer j.
__device__ __forceinline__ bool holds(const Hash& h, uint32_t j) {
  for (uint32_t s = j * 2654435761u >> (32 - h.log_n);; s = (s + 1) & ((1u << h.log_n) - 1)) {
    const uint32_t key = h.key[s];
    if (key == 0u || key == j + 1u) return key != 0u;
  }
}

__device__ __forceinline__ void fill(const cf_answer_rules& R, const Row& w, const Hash& h) {
  for (uint32_t i = threadIdx.x * 4; i < 3u << h.log_n; i += blockDim.x * 4) *(uint4*)(h.key + i) = make_uint4(0, 0, 0, 0);
  if (threadIdx.x == 0) *h.listed = 0;
  __syncthreads();
  const int32_t n = (int32_t)R.n;
  walk<4>(R.tokens_dev, w.h0, w.h1, [&](int32_t j, uint32_t at) {
    if (j >= n) return;
    const uint32_t s = slot_of(h, (uint32_t)j);
    if (at >= w.answered)
      atomicAdd(h.cnt + s, 1u);
    else
      atomicOr(h.cnt + s, kSeen << 16);
  });
  walk<4>(R.bias_ids_dev, w.b0, w.b1, [&](int32_t j, uint32_t at) {
    if (j < n) atomicMax(h.pos + slot_of(h, (uint32_t)j), at - w.b0 + 1u);
  });
  __syncthreads();
}

// 16 bytes of a row, moved whole.  Rows are read once, past the cache; what is written stays there
// for the edits behind.
template <typename T>
struct alignas(16) Vec {
  static constexpr int N = 16 / sizeof(T);
  T v[N];
  __device__ __forceinline__ void load(const T* p) { *(uint4*)v = __ldcs((const uint4*)p); }
  __device__ __forceinline__ void store(T* p) const { *(uint4*)p = *(const uint4*)v; }
};

// ---------------------------------------------------------------------- edit_logits
// out = allowed ? in : -inf, by a grid that is resident all at once; chunks of 256 x kUnroll
// vectors.  Where out is in, only vectors that hold something not allowed are written.
constexpr int kStreamThreads = 256, kUnroll = 4;

template <typename T>
__global__ void __launch_bounds__(kStreamThreads)
    k_answer_stream(const cf_answer_rules R, const T* in, int64_t in_rs, T* out, int64_t out_rs, int chunks,
                    int64_t units) {
  constexpr int V = Vec<T>::N, kChunk = kStreamThreads * kUnroll * V;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int n = (int)R.n;
  const bool in_place = in == out && in_rs == out_rs;
  int64_t r = blockIdx.x / chunks;
  int c = (int)(blockIdx.x - r * chunks);
  const int64_t step_r = gridDim.x / chunks;
  const int step_c = (int)(gridDim.x - step_r * chunks);
  for (int64_t unit = blockIdx.x; unit < units; unit += gridDim.x) {
    const T* x = in + r * in_rs;
    T* y = out + r * out_rs;
    // vectors start at 16-byte boundaries of the row's memory
    const int mis = (int)(((uintptr_t)x & 15) / sizeof(T));
    const bool aligned = (((uintptr_t)y - (uintptr_t)mis * sizeof(T)) & 15) == 0;
    const uint32_t* allowed = mask_of(R, r);
    const int j0 = c * kChunk - mis + (int)threadIdx.x * V;
    if (!in_place || allowed) {
      Vec<T> t[kUnroll];
#pragma unroll
      for (int i = 0; i < kUnroll; ++i) {
        const int j = j0 + i * kStreamThreads * V;
        if (j >= 0 && j + V <= n) {
          t[i].load(x + j);
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e)
            if (j + e >= 0 && j + e < n) t[i].v[e] = x[j + e];
        }
      }
#pragma unroll
      for (int i = 0; i < kUnroll; ++i) {
        const int j = j0 + i * kStreamThreads * V;
        if (j >= n) break;
        const uint32_t bits = open_bits<V>(allowed, j, n);
        if (in_place && bits == (1u << V) - 1) continue;
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (!(bits >> e & 1u)) t[i].v[e] = from_f32<T>(-INFINITY);
        if (aligned && j >= 0 && j + V <= n) {
          t[i].store(y + j);
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e)
            if (j + e >= 0 && j + e < n) y[j + e] = t[i].v[e];
        }
      }
    }
    r += step_r;
    c += step_c;
    if (c >= chunks) {
      c -= chunks;
      ++r;
    }
  }
}

// The answers that the history and the biases touch, in the result, after the stream: what is not
// allowed stays -inf there, the others are their logits.  `ctas` a row: a short row is the first
// one's, the slices of a long one are dealt out.
template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads)
    k_answer_edits(const cf_answer_rules R, T* out, int64_t out_rs, int log_s, int slices, int ctas) {
  extern __shared__ __align__(16) uint32_t smem[];
  const int64_t r = blockIdx.x / ctas;
  const int cta = (int)(blockIdx.x - r * ctas);
  const Row w = load_row(R, r);
  const bool brief = is_short<kShort>(w);
  if ((w.h0 == w.h1 && w.b0 == w.b1) || (brief && cta != 0)) {
    asm volatile("griddepcontrol.wait;" ::: "memory");  // this grid's end must not come before the stream's
    return;
  }
  T* y = out + r * out_rs;
  if (brief) {
    const Hash h = hash_of(w, smem, kSlots);
    fill(R, w, h);
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the stream is done
    constexpr int kBatch = 4;
    const uint32_t listed = *h.listed;
    for (uint32_t i = threadIdx.x; i < listed; i += kBatch * blockDim.x) {
      int j[kBatch];
      uint32_t c[kBatch], p[kBatch];
      float bias[kBatch];
      T v[kBatch];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const bool ok = i + b * blockDim.x < listed;
        const uint32_t s = ok ? h.list[i + b * blockDim.x] : 0u;
        j[b] = ok ? (int)h.key[s] - 1 : -1;
        c[b] = h.cnt[s];
        p[b] = h.pos[s];
      }
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        v[b] = j[b] >= 0 ? y[j[b]] : from_f32<T>(0.0f);
        bias[b] = j[b] >= 0 && p[b] ? R.bias_values_dev[w.b0 + p[b] - 1u] : 0.0f;
        if (j[b] >= 0 && !is_allowed(w.allowed, j[b])) j[b] = -1;
      }
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        if (j[b] < 0) continue;
        float e = edit(to_f32(v[b]), c[b] != 0, c[b] & kWideTimes, w.rep, w.freq, w.pres);
        if (p[b]) e = __fadd_rn(e, bias[b]);
        y[j[b]] = from_f32<T>(e);
      }
    }
    return;
  }
  Tables t = tables_of(w, smem, log_s);
  const int n = (int)R.n;
  bool waited = false;
  for (int slice = cta; slice < slices; slice += ctas) {
    const int end = (int)min((int64_t)n, (int64_t)(slice + 1) << log_s);
    uint32_t size;
    for (int lo = slice << log_s; lo < end; lo += (int)size) {
      size = (uint32_t)min(1 << (t.wide ? log_s - 2 : log_s), end - lo);
      if (waited) __syncthreads();  // the tables are filled anew
      const bool done = count(R, w, t, lo, size);
      if (!waited) asm volatile("griddepcontrol.wait;" ::: "memory");  // the stream is done
      waited = true;
      if (!done) {
        t.wide = true;
        size = 0;
        continue;
      }
      if (w.b1 > w.b0) {
        for_biased(R, w, t, lo, size, [&](int j, bool seen, uint32_t times, float bias) {
          if (is_allowed(w.allowed, j))
            y[j] = from_f32<T>(__fadd_rn(edit(to_f32(y[j]), seen, times, w.rep, w.freq, w.pres), bias));
        });
        __syncthreads();  // the marks
      }
      for_seen(w, t, lo, size, y, [&](int j, uint32_t times, float v) {
        y[j] = from_f32<T>(edit(v, true, times, w.rep, w.freq, w.pres));
      });
    }
  }
}

// --------------------------------------------------------------------- answer_margin
struct Best {
  float v;
  int32_t j;
};

// the larger value; the lower answer on equal ones
__device__ __forceinline__ bool beats(float v, int32_t j, const Best& a) { return v > a.v || (v == a.v && j < a.j); }

__device__ __forceinline__ void take(Best& a, float v, int32_t j) {
  if (beats(v, j, a)) {
    a.v = v;
    a.j = j;
  }
}

constexpr int32_t kNone = INT32_MAX;
constexpr int kMarginThreads = 256, kMaxCluster = 8;

// floats as integers of the same order, and back
__device__ __forceinline__ int to_ordered(float v) {
  const int i = __float_as_int(v);
  return i ^ ((i >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float from_ordered(int i) { return __int_as_float(i ^ ((i >> 31) & 0x7fffffff)); }

// the larger, NaN if one is
__device__ __forceinline__ float max_nan(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}

// One cluster per row: the label's edited lower bound less the best edited upper bound among the
// other answers.  Each CTA has a share of the answers (of a row with a long history, slices); what
// is touched has its own pass, and on the way over the bounds a vector is looked into only where it
// holds something above the best that the CTA's warps have told one another of.  128 rows of 131072, 67 MB:
// 14 us without edits (from the L2 cache; 21 when each warp only knew its own best), 25 with up to 1024
// tokens a row: the table has to be there before the first bound can be passed over.
__global__ void __launch_bounds__(kMarginThreads, 4)
    k_answer_margin(const cf_answer_rules R, const float* __restrict__ l, int64_t l_rs, const float* __restrict__ u,
                    int64_t u_rs, const int64_t* __restrict__ labels, float* margin, int32_t* rival, int log_s,
                    int slices) {
  extern __shared__ __align__(16) uint32_t smem[];
  __shared__ Best part_best[kMarginThreads / 32];
  __shared__ Best joined[kMaxCluster];
  __shared__ float joined_l[kMaxCluster];
  __shared__ float label_l;
  __shared__ int heard;  // the best of the CTA's warps, as far as told
  constexpr int V = 4, kVpt = 4, kChunk = kMarginThreads * V * kVpt;
  cg::cluster_group cl = cg::this_cluster();
  const int nc = (int)cl.num_blocks(), rank = (int)cl.block_rank(), n = (int)R.n;
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // this CTA runs; awaited at the end
  const int64_t r = blockIdx.x / nc;
  const float* x = u + r * u_rs;
  const int mis = (int)(((uintptr_t)x & 15) / 4);
  Vec<float> t[kVpt];
  // vector i of this thread of the chunk at j0 (j0 + mis a multiple of 4)
  auto load = [&](int i, int j0, int end) {
    const int j = j0 + (i * kMarginThreads + (int)threadIdx.x) * V;
    if (j >= end) return;
    if (j >= 0 && j + V <= n) {
      *(float4*)t[i].v = *(const float4*)(x + j);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) t[i].v[e] = j + e >= 0 && j + e < n ? x[j + e] : 0.0f;
    }
  };
  auto load_all = [&](int j0, int end) {
#pragma unroll
    for (int i = 0; i < kVpt; ++i) load(i, j0, end);
  };
  // of answers [lo, end), the first vector's place
  auto first = [&](int lo) { return ((lo + mis) & ~3) - mis; };
  const Row w = load_row(R, r);
  const bool touch = w.h1 > w.h0 || w.b1 > w.b0, brief = is_short<kMarginShort>(w);
  // this CTA's share of a row without a long history
  const int share = (int)(((n + nc - 1) / nc + 3) & ~3), lo0 = min(rank * share, n), end0 = min(lo0 + share, n);
  if (brief && lo0 < end0) load_all(first(lo0), end0);
  const int label = labels[r] >= 0 && labels[r] < n ? (int)labels[r] : INT32_MIN;  // or no answer
  const float label_x = label >= 0 ? l[r * l_rs + label] : 0.0f;
  if (threadIdx.x == 0) {
    label_l = -INFINITY;
    heard = to_ordered(-INFINITY);
  }
  __syncthreads();
  Best best{-INFINITY, kNone};
  // the edited bound v of allowed answer j
  auto bound = [&](int j, float v) { take(best, v != v ? INFINITY : v, j); };
  auto own = [&](float v) { label_l = v != v ? -INFINITY : v; };  // a bound that is no number bounds nothing
  // the bounds of answers [lo, stop) that are not touched; their first chunk is loaded
  auto pass = [&](int lo, int stop, auto&& touched) {
    if (lo >= stop) return;
    if (label >= lo && label < stop && threadIdx.x == 0 && is_allowed(w.allowed, label) && !touched(label)) own(label_x);
    __syncwarp();
    float floor = best.v;  // what the warp, and as far as it has heard the CTA, has found
    for (int j0 = first(lo); j0 < stop; j0 += kChunk) {
      floor = fmaxf(floor, from_ordered(*(volatile int*)&heard));
#pragma unroll
      for (int i = 0; i < kVpt; ++i) {
        const int j = j0 + (i * kMarginThreads + (int)threadIdx.x) * V;
        const Vec<float> a = t[i];
        load(i, j0 + kChunk, stop);
        const float top = max_nan(max_nan(a.v[0], a.v[1]), max_nan(a.v[2], a.v[3]));
        const bool look = j < stop && !(top < floor);
        if (__any_sync(0xffffffffu, look)) {
          if (look) {
            const uint32_t bits = open_bits<V>(w.allowed, j, n);
#pragma unroll
            for (int e = 0; e < V; ++e) {
              const float v = a.v[e] != a.v[e] ? INFINITY : a.v[e];
              if (v >= floor && beats(v, j + e, best) && (bits >> e & 1u) && j + e >= lo && j + e < stop &&
                  j + e != label && !touched(j + e))
                best = {v, j + e};
            }
          }
          float top_found = best.v;
#pragma unroll
          for (int off = 16; off > 0; off >>= 1)
            top_found = fmaxf(top_found, __shfl_xor_sync(0xffffffffu, top_found, off));
          if (top_found > floor) {
            floor = top_found;
            if ((threadIdx.x & 31) == 0) atomicMax(&heard, to_ordered(floor));
          }
        }
      }
    }
  };
  if (!touch) {
    pass(lo0, end0, [](int) { return false; });
  } else if (brief) {
    const Hash h = hash_of(w, smem, kMarginSlots);
    fill(R, w, h);
    const uint32_t listed = *h.listed;
    for (uint32_t i = threadIdx.x; i < listed; i += kMarginThreads) {
      const uint32_t s = h.list[i], c = h.cnt[s], at = h.pos[s];
      const int j = (int)h.key[s] - 1;
      if (j < lo0 || j >= end0 || !is_allowed(w.allowed, j)) continue;
      float v = edit(j == label ? label_x : x[j], c != 0, c & kWideTimes, w.rep, w.freq, w.pres);
      if (at) v = __fadd_rn(v, R.bias_values_dev[w.b0 + at - 1u]);
      if (j == label)
        own(v);
      else
        bound(j, v);
    }
    __syncwarp();
    pass(lo0, end0, [&](int j) { return holds(h, (uint32_t)j); });
  } else {
    Tables tab = tables_of(w, smem, log_s);
    bool counted = false;
    for (int slice = rank; slice < slices; slice += nc) {
      const int end = (int)min((int64_t)n, (int64_t)(slice + 1) << log_s);
      uint32_t size;
      for (int lo = slice << log_s; lo < end; lo += (int)size) {
        const int stop = min(lo + (1 << (tab.wide ? log_s - 2 : log_s)), end);
        size = (uint32_t)(stop - lo);
        load_all(first(lo), stop);
        if (counted) __syncthreads();  // the tables are filled anew
        counted = true;
        if (!count(R, w, tab, lo, size)) {
          tab.wide = true;
          size = 0;
          continue;
        }
        for_biased(R, w, tab, lo, size, [&](int j, bool seen, uint32_t times, float bias) {
          if (!is_allowed(w.allowed, j)) return;
          const float v = __fadd_rn(edit(j == label ? label_x : x[j], seen, times, w.rep, w.freq, w.pres), bias);
          if (j == label)
            own(v);
          else
            bound(j, v);
        });
        if (w.b1 > w.b0) __syncthreads();  // the marks
        for_seen(w, tab, lo, size, x, [&](int j, uint32_t times, float v) {
          v = edit(j == label ? label_x : v, true, times, w.rep, w.freq, w.pres);
          if (j == label)
            own(v);
          else
            bound(j, v);
        });
        __syncwarp();
        pass(lo, stop, [&](int j) {
          const uint32_t k = (uint32_t)(j - lo);
          return entry(tab, k) != 0 || is_biased(w, tab, k);
        });
      }
    }
  }
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
    const float v = __shfl_xor_sync(0xffffffffu, best.v, off);
    const int32_t j = __shfl_xor_sync(0xffffffffu, best.j, off);
    take(best, v, j);
  }
  if ((threadIdx.x & 31) == 0) part_best[threadIdx.x >> 5] = best;
  __syncthreads();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // all of the cluster's CTAs run
  if (threadIdx.x == 0) {
    for (int i = 1; i < kMarginThreads / 32; ++i) take(best, part_best[i].v, part_best[i].j);
    cl.map_shared_rank(joined, 0)[rank] = best;
    cl.map_shared_rank(joined_l, 0)[rank] = label_l;
  }
  cl.sync();
  if (rank == 0 && threadIdx.x == 0) {
    float mine = label_l;  // one CTA has the label, the others' is -inf
    for (int i = 0; i < nc; ++i) {
      take(best, joined[i].v, joined[i].j);
      mine = fmaxf(mine, joined_l[i]);
    }
    const bool any = best.v > -INFINITY;
    const float m = mine - best.v;
    margin[r] = m != m ? -INFINITY : m;  // an infinite bound less itself says nothing
    rival[r] = any ? best.j : -1;
  }
}

// ------------------------------------------------------------------------------ host
size_t smem_bytes(int log_s, size_t hash) {
  const size_t tables = tables_bytes(log_s);
  return tables > hash ? tables : hash;
}

bool has_edits(const cf_answer_rules& R) {
  return (R.tokens_dev && R.n_tokens > 0) || (R.bias_ids_dev && R.n_biases > 0);
}

// `allowed`: the devices on which the kernel may have kMostSmem bytes (nullptr: it needs no more than 48 KB)
template <typename F, typename... Args>
cf_status launch(const char* what, F* kern, std::atomic<uint64_t>* allowed, int64_t blocks, int threads, size_t smem,
                 int cluster, bool dependent, cudaStream_t st, Args... args) {
  CF_REQUIRE(blocks <= 0x7fffffff, CF_ERR_SHAPE, "%s: too many rows", what);
  if (smem > 48 * 1024) CF_TRY(allow_smem(kern, kMostSmem, *allowed, what));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  int n = 0;
  if (cluster > 0) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = (unsigned)cluster;
    at[n].val.clusterDim.y = at[n].val.clusterDim.z = 1;
    ++n;
  }
  if (dependent) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = at;
  cfg.numAttrs = n;
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
  CF_REQUIRE(R->n < 1 << 30 && R->n_tokens < 1 << 30 && R->n_biases < 1 << 30, CF_ERR_SHAPE,
             "%s: fewer than 2^30 answers, tokens and biases", what);
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
  CF_REQUIRE(((uintptr_t)R->token_offsets_dev | (uintptr_t)R->bias_offsets_dev) % 8 == 0 &&
                 ((uintptr_t)R->tokens_dev | (uintptr_t)R->prompt_len_dev | (uintptr_t)R->repetition_dev |
                  (uintptr_t)R->frequency_dev | (uintptr_t)R->presence_dev | (uintptr_t)R->bias_ids_dev |
                  (uintptr_t)R->bias_values_dev | (uintptr_t)R->allowed_dev | (uintptr_t)R->allowed_row_dev) % 4 == 0,
             CF_ERR_SHAPE, "%s: unaligned rules", what);
  return CF_OK;
}

template <typename T>
cf_status edit_logits(const cf_answer_rules& R, const void* in, int64_t in_rs, void* out, int64_t out_rs,
                      cudaStream_t st) {
  constexpr int V = Vec<T>::N, kChunk = kStreamThreads * kUnroll * V;
  CF_REQUIRE(((uintptr_t)in | (uintptr_t)out) % sizeof(T) == 0, CF_ERR_SHAPE, "edit_logits: unaligned rows");
  if (R.rows == 1) in_rs = out_rs;
  const bool stream = in != out || in_rs != out_rs || R.allowed_dev;
  if (stream) {
    const int chunks = (int)ceil_div(R.n + V - 1, kChunk);
    const int64_t units = R.rows * chunks, most = 148 * 4;  // four CTAs an SM
    CF_TRY(launch("k_answer_stream", k_answer_stream<T>, nullptr, units < most ? units : most, kStreamThreads, 0, 0, false, st,
                  R, (const T*)in, in_rs, (T*)out, out_rs, chunks, units));
  }
  if (!has_edits(R)) return CF_OK;
  // Rows of up to 2048 tokens on average: one small CTA a row, which counts while the stream's last CTAs
  // run (four of them leave an SM a quarter of its registers, half of what the smaller CTA takes).
  // Longer ones: 32768 answers a slice (64 KB of tables; 1024 threads of 64 registers are an SM's), fewer
  // where that leaves SMs idle.  The mean decides for all rows: 256 rows of 131072 bfloat16 take 29 us
  // with 1000 tokens each and 204 if one of them has 32768, whose slices then go through one CTA (191
  // if all have).
  const bool brief = R.n_tokens <= R.rows * 2048;
  int log_s = brief ? 14 : 15;
  if (!brief)
    while (log_s > 11 && R.rows * ceil_div(R.n, (int64_t)1 << log_s) < 148) --log_s;
  while (log_s > 11 && (int64_t)1 << (log_s - 1) >= R.n) --log_s;
  const int slices = (int)ceil_div(R.n, (int64_t)1 << log_s), ctas = brief ? 1 : slices;
  const size_t smem = smem_bytes(log_s, hash_bytes(kSlots, kShort));
  static std::atomic<uint64_t> allowed[2];
  // More short rows than SMs: two CTAs of 512 an SM (256 rows of 131072 bfloat16, up to 2048 tokens: 34.3 us, 36.7 with
  // 1024); else 1024 (64 rows, up to 1000 tokens: 12.4 us, 13.6 with 512).
  if (brief && R.rows > 148)
    return launch("k_answer_edits", k_answer_edits<T, 512>, &allowed[0], R.rows * ctas, 512, smem, 0, stream, st, R,
                  (T*)out, out_rs, log_s, slices, ctas);
  return launch("k_answer_edits", k_answer_edits<T, 1024>, &allowed[1], R.rows * ctas, 1024, smem, 0, stream, st, R,
                (T*)out, out_rs, log_s, slices, ctas);
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
  CF_REQUIRE(in != out || R->rows <= 1 || in_rs == out_rs, CF_ERR_SHAPE, "edit_logits: rows change places");
  CF_REQUIRE(dtype == CF_F32 || dtype == CF_BF16 || dtype == CF_F16, CF_ERR_UNSUPPORTED, "edit_logits: dtype %d",
             dtype);
  if (R->rows * R->n == 0) return CF_OK;
  CF_REQUIRE(in && out, CF_ERR_NULL, "edit_logits: NULL argument");
  CF_REQUIRE((in == out && (R->rows == 1 || in_rs == out_rs)) ||
                 !rows_overlap(in, in_rs, R->n, out, out_rs, R->n, R->rows, dtype == CF_F32 ? 4 : 2),
             CF_ERR_SHAPE, "edit_logits: the logits and the result overlap");
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
  CF_REQUIRE((uintptr_t)labels % 8 == 0 && ((uintptr_t)margin | (uintptr_t)rival) % 4 == 0, CF_ERR_SHAPE,
             "answer_margin: unaligned labels or results");
  // 8192 answers a slice, 16384 where rows are long on average, fewer for few answers or few rows; a cluster of up
  // to eight for a row, as far as all rows' fit the GPU at once
  int log_s = R->n_tokens > R->rows * kMarginShort ? 14 : 13;
  while (log_s > 11 && ((int64_t)1 << (log_s - 1) >= R->n ||
                        (R->rows * ceil_div(R->n, (int64_t)1 << log_s) < 148 && (int64_t)8 << (log_s - 1) >= R->n)))
    --log_s;
  const int slices = (int)ceil_div(R->n, (int64_t)1 << log_s);
  int cluster = 1;
  while (cluster < kMaxCluster && cluster < slices && R->rows * cluster * 2 <= 148 * 4) cluster *= 2;
  static std::atomic<uint64_t> allowed{0};
  return launch("k_answer_margin", k_answer_margin, &allowed, R->rows * cluster, kMarginThreads,
                has_edits(*R) ? smem_bytes(log_s, hash_bytes(kMarginSlots, kMarginShort)) : 0, cluster, false, as_stream(stream), *R, l, l_rs, u, u_rs,
                labels, margin, rival, log_s, slices);
}
