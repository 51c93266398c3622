// What the tensor-core kernels of the adapter product share: operand images, stores, the
// row-by-row low-rank part.
#pragma once

#include "cf_adapter.cuh"
#include "cf_tc.cuh"

namespace cf {
namespace adapter {

// Instruction descriptor: float32 accumulator, A and B of type ab (0 f16, 1 bf16, 2 tf32), A
// K-major, B K-major or (bit 16) MN-major, 128 x n.
__device__ __forceinline__ uint32_t idesc(uint32_t ab, uint32_t n, bool mn_major) {
  return (1u << 4) | (ab << 7) | (ab << 10) | ((uint32_t)mn_major << 16) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}

template <typename T>
struct Kind;  // of a type: elements in 128 bytes, descriptor type
template <>
struct Kind<float> {
  static constexpr int kStep = 32, kAb = 2;
};
template <>
struct Kind<__nv_bfloat16> {
  static constexpr int kStep = 64, kAb = 1;
};
template <>
struct Kind<__half> {
  static constexpr int kStep = 64, kAb = 0;
};

// Loads that stay where they are written, zeros where not `ok`: a thread has two steps' loads in
// flight, and neither a move of them to their uses nor a selection behind them may wait for one.
__device__ __forceinline__ uint4 ldg16_if(const void* p, bool ok) {
  uint4 v;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
      "@p ld.global.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
      : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w)
      : "l"(p), "r"((int)ok));
  return v;
}
__device__ __forceinline__ uint32_t ldg4_if(const void* p, bool ok) {
  uint32_t v;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %2, 0;\n\t"
      "mov.b32 %0, 0;\n\t"
      "@p ld.global.u32 %0, [%1];\n\t}"
      : "=&r"(v)
      : "l"(p), "r"((int)ok));
  return v;
}

// 16 bytes of row `row` (elements k .. of n_k), zero beyond
template <typename T>
__device__ __forceinline__ uint4 load16(const T* row, int64_t k, int64_t n_k, bool vec) {
  constexpr int E = 16 / sizeof(T);
  if (vec && k + E <= n_k) return *(const uint4*)(row + k);
  alignas(16) T t[E];
#pragma unroll
  for (int i = 0; i < E; ++i) t[i] = k + i < n_k ? row[k + i] : from_f32<T>(0.0f);
  return *(const uint4*)t;
}

// a 16-byte chunk of one float32 operand row into its planes hi and lo
__device__ __forceinline__ void put(uint32_t plane, uint32_t plane_bytes, uint32_t row, uint32_t chunk, uint4 d) {
  const uint32_t at = plane + row * 128u + ((chunk ^ (row & 7u)) << 4);
  float hi[4], lo[4];
  tc::split_tf32(__uint_as_float(d.x), hi[0], lo[0]);
  tc::split_tf32(__uint_as_float(d.y), hi[1], lo[1]);
  tc::split_tf32(__uint_as_float(d.z), hi[2], lo[2]);
  tc::split_tf32(__uint_as_float(d.w), hi[3], lo[3]);
  asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at), "f"(hi[0]), "f"(hi[1]), "f"(hi[2]), "f"(hi[3])
               : "memory");
  asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at + plane_bytes), "f"(lo[0]), "f"(lo[1]), "f"(lo[2]),
               "f"(lo[3])
               : "memory");
}

// y columns n .. n+3 of row t
template <typename T>
__device__ __forceinline__ void store4(const Problem& p, int64_t t, int64_t n, const float (&a)[4]) {
  T* y = (T*)p.y + t * p.y_rs + n;
  if (p.y_vec && n + 4 <= p.N) {
    alignas(16) T o[4] = {from_f32<T>(a[0]), from_f32<T>(a[1]), from_f32<T>(a[2]), from_f32<T>(a[3])};
    if constexpr (sizeof(T) == 4)
      *(uint4*)y = *(const uint4*)o;
    else
      *(uint2*)y = *(const uint2*)o;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < p.N) y[i] = from_f32<T>(a[i]);
  }
}

// a += v[t] Q_e at columns n .. n+3 (columns beyond N are not read)
template <typename T, bool kSub>
__device__ __forceinline__ void add_lowrank(const Problem& p, int64_t t, int e, int rank, int64_t n, float (&a)[4]) {
  const float* v = p.v + t * p.v_rs;
  const T* Q = (const T*)p.Qm + e * p.q_es;
  if constexpr (kSub) {  // rows of n
    const bool full = n + 4 <= p.N;
#pragma unroll 4
    for (int r = 0; r < rank; ++r) {
      const T* q = Q + r * p.q_rs + n;
      const float w = v[r];
      if (full && p.q_vec) {
        alignas(16) T d[4];
        if constexpr (sizeof(T) == 4)
          *(uint4*)d = *(const uint4*)q;
        else
          *(uint2*)d = *(const uint2*)q;
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = fmaf(w, to_f32(d[i]), a[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (n + i < p.N) a[i] = fmaf(w, to_f32(q[i]), a[i]);
      }
    }
  } else {  // rows of r
    constexpr int E = 16 / sizeof(T);
    int r = 0;
    if (p.q_vec) {
#pragma unroll 2
      for (; r + E <= rank; r += E) {
        float w[E];
        uint4 d[4];
#pragma unroll
        for (int i = 0; i < E; i += 4) *(float4*)(w + i) = *(const float4*)(v + r + i);  // rows of v are aligned
#pragma unroll
        for (int c = 0; c < 4; ++c)
          d[c] = n + c < p.N ? *(const uint4*)(Q + (n + c) * p.q_ns + r) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int i = 0; i < E; ++i) a[c] = fmaf(w[i], to_f32(((const T*)&d[c])[i]), a[c]);
      }
    }
    for (; r < rank; ++r)
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (n + c < p.N) a[c] = fmaf(v[r], to_f32(Q[(n + c) * p.q_ns + r]), a[c]);
  }
}

// The same for the 16 columns n .. n+15 of one thread's row.
template <typename T, bool kSub>
__device__ __forceinline__ void add_lowrank16(const Problem& p, int64_t t, int e, int rank, int64_t n,
                                              float (&a)[16]) {
  const float* v = p.v + t * p.v_rs;
  const T* Q = (const T*)p.Qm + e * p.q_es;
  constexpr int E = 16 / sizeof(T);
  const bool vec = p.q_vec && n + 16 <= p.N;
  if constexpr (kSub) {
    if (vec) {
#pragma unroll 4
      for (int r = 0; r < rank; ++r) {
        const T* q = Q + r * p.q_rs + n;
        const float w = v[r];
#pragma unroll
        for (int c = 0; c < 16; c += E) {
          alignas(16) T d[E];
          *(uint4*)d = *(const uint4*)(q + c);
#pragma unroll
          for (int i = 0; i < E; ++i) a[c + i] = fmaf(w, to_f32(d[i]), a[c + i]);
        }
      }
    } else {
      for (int r = 0; r < rank; ++r) {
        const T* q = Q + r * p.q_rs + n;
        const float w = v[r];
#pragma unroll
        for (int c = 0; c < 16; ++c)
          if (n + c < p.N) a[c] = fmaf(w, to_f32(q[c]), a[c]);
      }
    }
  } else {
    int r = 0;
    if (vec) {
      for (; r + E <= rank; r += E) {
        float w[E];
#pragma unroll
        for (int i = 0; i < E; ++i) w[i] = v[r + i];
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          alignas(16) T d[E];
          *(uint4*)d = *(const uint4*)(Q + (n + c) * p.q_ns + r);
#pragma unroll
          for (int i = 0; i < E; ++i) a[c] = fmaf(w[i], to_f32(d[i]), a[c]);
        }
      }
    }
    for (; r < rank; ++r) {
      const float w = v[r];
#pragma unroll
      for (int c = 0; c < 16; ++c)
        if (n + c < p.N) a[c] = fmaf(w, to_f32(Q[(n + c) * p.q_ns + r]), a[c]);
    }
  }
}

// A CTA's error word, by one warp at its end, into its kernel file's.
__device__ __forceinline__ void report(int err, int* site) {
  if (err != 0 && (threadIdx.x & 31) == 0) atomicCAS(site, 0, err);
}

// Read and clear a kernel file's error word.
inline cf_status take_site(int* symbol, int* site, cudaStream_t st) {
  void* at = nullptr;
  *site = 0;
  cudaError_t e = cudaGetSymbolAddress(&at, (const void*)symbol);
  if (e == cudaSuccess) e = cudaMemcpyAsync(site, at, sizeof(int), cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e == cudaSuccess && *site != 0) {
    e = cudaMemsetAsync(at, 0, sizeof(int), st);
    if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  }
  CF_REQUIRE(e == cudaSuccess, CF_ERR_CUDA, "adapter_check: %s", cudaGetErrorString(e));
  return CF_OK;
}

// CTAs of a cluster that share a tile's contraction, at least four steps each: as many as still
// have an SM to themselves.  Clusters do not pack the GPU's processor clusters fully, so 128 CTAs
// count as full and 64 in clusters of eight (4096 x 4096 for one token, 32 tiles: 11.1 us with 4,
// 12.9 with 3, 15.5 with 5, 17.0 with 8; 16 tiles: 10.5 with 6, 13.7 with 8).
inline int split_for(int64_t tiles, int64_t steps) {
  for (int s : {8, 6, 4, 3, 2})
    if (tiles * s <= (s == 8 ? 64 : 128) && steps >= s * 4) return s;
  return 1;
}

}  // namespace adapter
}  // namespace cf
