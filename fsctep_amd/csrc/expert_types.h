// Element types and vector accesses shared by the expert readout's kernels (norm, router, products).
#pragma once

#include <hip/hip_runtime.h>
#include <cstdint>

namespace fsc {

typedef unsigned u1v;
typedef unsigned u2v __attribute__((ext_vector_type(2)));
typedef unsigned u4v __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__bf16 v) { return (float)v; }
template <typename T>
__device__ __forceinline__ T from_f(float v) { return (T)v; }
// the value as an array of type T holds it
template <typename T>
__device__ __forceinline__ float held(float v) { return to_f(from_f<T>(v)); }

// LDS that one wave writes and reads: what its lanes wrote before is what they read after.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Larger of two values, NaN if either is one (a row with a NaN shows it).
__device__ __forceinline__ float max_nan(float a, float b) { return (a > b || a != a) ? a : b; }

// V values widened to 32 bits by one load (V * sizeof(T) of 16 bytes, aligned to that; V 1: any alignment).
template <int V>
__device__ __forceinline__ void load_vec(const float* p, float (&v)[V]) {
  if constexpr (V % 4 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      const f4 t = ld4(p + i);
      v[i] = t.x; v[i + 1] = t.y; v[i + 2] = t.z; v[i + 3] = t.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = p[i];
  }
}
template <int V>
__device__ __forceinline__ void load_vec(const __bf16* p, float (&v)[V]) {
  if constexpr (V % 8 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 8) {
      const bf8 t = *reinterpret_cast<const bf8*>(p + i);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i + j] = (float)t[j];
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = (float)p[i];
  }
}
template <int V>
__device__ __forceinline__ void store_vec(float* p, const float (&v)[V]) {
  if constexpr (V % 4 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 4) st4(p + i, f4{v[i], v[i + 1], v[i + 2], v[i + 3]});
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) p[i] = v[i];
  }
}
template <int V>
__device__ __forceinline__ void store_vec(__bf16* p, const float (&v)[V]) {
  if constexpr (V % 8 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 8) {
      bf8 t;
#pragma unroll
      for (int j = 0; j < 8; ++j) t[j] = (__bf16)v[i + j];
      *reinterpret_cast<bf8*>(p + i) = t;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) p[i] = (__bf16)v[i];
  }
}
// V bytes (V 8 or 4: aligned to V)
template <int V>
__device__ __forceinline__ void store_bytes(int8_t* p, const int8_t (&b)[V]) {
  if constexpr (V % 4 == 0) {
    unsigned w[V / 4];
#pragma unroll
    for (int i = 0; i < V / 4; ++i)
      w[i] = (uint8_t)b[4 * i] | (unsigned)(uint8_t)b[4 * i + 1] << 8 | (unsigned)(uint8_t)b[4 * i + 2] << 16 |
             (unsigned)(uint8_t)b[4 * i + 3] << 24;
    if constexpr (V == 4) *reinterpret_cast<unsigned*>(p) = w[0];
    else *reinterpret_cast<u2v*>(p) = u2v{w[0], w[1]};
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) p[i] = b[i];
  }
}

}  // namespace fsc
