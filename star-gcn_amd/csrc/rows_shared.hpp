// rows_shared.hpp -- what the row kernels of the catalogue head share: the three float types, 16-byte vectors at any element
// alignment, workgroup reductions.
#pragma once
#include "common.hpp"

namespace sg {

using f16 = _Float16;
struct bf16 {
  uint16_t bits;
};

inline bool valid_dtype(int d) { return d == SG_DTYPE_F32 || d == SG_DTYPE_F16 || d == SG_DTYPE_BF16; }

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(f16 v) { return static_cast<float>(v); }
__device__ __forceinline__ float to_f32(bf16 v) { return __uint_as_float(static_cast<unsigned>(v.bits) << 16); }

template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ f16 from_f32<f16>(float v) { return static_cast<f16>(v); }
template <> __device__ __forceinline__ bf16 from_f32<bf16>(float v) {      // to nearest, ties to even; NaN stays NaN
  const unsigned u = __float_as_uint(v);
  const unsigned r = (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
  return bf16{static_cast<uint16_t>(v != v ? 0x7fc0u : r)};
}
template <typename T> __device__ __forceinline__ float round_to(float v) { return to_f32(from_f32<T>(v)); }

// V elements as one vector access.  The hardware takes vector accesses at any byte address; rows of odd length start where
// they start.
template <typename T, int V>
struct __attribute__((packed, aligned(sizeof(T)))) vec_any {
  T v[V];
};

// n = V: one vector load; 0 < n < V: element loads, zeros behind them; n <= 0: zeros, nothing is read
template <typename T, int V>
__device__ __forceinline__ void load_vec(float* out, const T* p, int n) {
  if (n >= V) {
    vec_any<T, V> a;
    __builtin_memcpy(&a, p, sizeof(a));
#pragma unroll
    for (int j = 0; j < V; ++j) out[j] = to_f32(a.v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) out[j] = j < n ? to_f32(p[j]) : 0.f;
  }
}

template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const float* in, int n) {
  if (n >= V) {
    vec_any<T, V> a;
#pragma unroll
    for (int j = 0; j < V; ++j) a.v[j] = from_f32<T>(in[j]);
    __builtin_memcpy(p, &a, sizeof(a));
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j < n) p[j] = from_f32<T>(in[j]);
  }
}

template <int V>
__device__ __forceinline__ void store_codes(int8_t* p, const int* q, int n) {
  if (n >= V) {
    vec_any<int8_t, V> a;
#pragma unroll
    for (int j = 0; j < V; ++j) a.v[j] = static_cast<int8_t>(q[j]);
    __builtin_memcpy(p, &a, sizeof(a));
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j < n) p[j] = static_cast<int8_t>(q[j]);
  }
}

}  // namespace sg
