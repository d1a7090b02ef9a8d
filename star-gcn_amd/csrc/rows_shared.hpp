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
template <> __device__ __forceinline__ bf16 from_f32<bf16>(float v) {      // v_cvt_pk_bf16_f32: to nearest, ties to even
  return __builtin_bit_cast(bf16, static_cast<__bf16>(v));
}
template <typename T> __device__ __forceinline__ float round_to(float v) { return to_f32(from_f32<T>(v)); }

// V elements as one access of 1, 2, 4, 8 or 16 bytes (loads: or several of 16).  The hardware takes vector accesses at any byte address; rows of odd
// length start where they start.  The vector types keep the compiler from taking the access apart to share its first element's
// store with the tail's.
template <typename T, int V>
struct alignas(sizeof(T) * V) pack {
  T v[V];
};
typedef int vec16 __attribute__((ext_vector_type(4)));
typedef vec16 vec16_any __attribute__((aligned(1)));
typedef int vec8 __attribute__((ext_vector_type(2)));
typedef vec8 vec8_any __attribute__((aligned(1)));
typedef int vec4_any __attribute__((aligned(1)));
typedef short vec2_any __attribute__((aligned(1)));

template <typename T, int V>
__device__ __forceinline__ pack<T, V> load_pack(const T* p) {
  constexpr int B = sizeof(T) * V;
  if constexpr (V == 1) {
    return pack<T, V>{{*p}};
  } else if constexpr (B == 4) {
    return __builtin_bit_cast(pack<T, V>, *reinterpret_cast<const vec4_any*>(p));
  } else if constexpr (B == 8) {
    return __builtin_bit_cast(pack<T, V>, *reinterpret_cast<const vec8_any*>(p));
  } else {
    static_assert(B % 16 == 0, "4, 8 or a multiple of 16 bytes");
    struct alignas(B) { vec16 q[B / 16]; } a;
#pragma unroll
    for (int i = 0; i < B / 16; ++i) a.q[i] = reinterpret_cast<const vec16_any*>(p)[i];
    return __builtin_bit_cast(pack<T, V>, a);
  }
}

template <typename T, int V>
__device__ __forceinline__ void store_pack(T* p, const pack<T, V>& a) {
  constexpr int B = sizeof(T) * V;
  if constexpr (V == 1) {
    *p = a.v[0];
  } else if constexpr (B == 2) {
    *reinterpret_cast<vec2_any*>(p) = __builtin_bit_cast(short, a);
  } else if constexpr (B == 4) {
    *reinterpret_cast<vec4_any*>(p) = __builtin_bit_cast(int, a);
  } else if constexpr (B == 8) {
    *reinterpret_cast<vec8_any*>(p) = __builtin_bit_cast(vec8, a);
  } else {
    static_assert(B == 16, "4, 8 or 16 bytes");
    *reinterpret_cast<vec16_any*>(p) = __builtin_bit_cast(vec16, a);
  }
}

// n = V: one vector load; 0 < n < V: element loads, zeros behind them; n <= 0: zeros, nothing is read
template <typename T, int V>
__device__ __forceinline__ void load_vec(float* out, const T* p, int n) {
  if (n >= V) {
    const pack<T, V> a = load_pack<T, V>(p);
#pragma unroll
    for (int j = 0; j < V; ++j) out[j] = to_f32(a.v[j]);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) out[j] = j < n ? to_f32(p[j]) : 0.f;
  }
}

template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const float* in, int n) {
  pack<T, V> a;
#pragma unroll
  for (int j = 0; j < V; ++j) a.v[j] = from_f32<T>(in[j]);
  if (n >= V) {
    store_pack<T, V>(p, a);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j < n) p[j] = a.v[j];
  }
}

// 16 aligned bytes past the caches: for what nothing reads soon
template <typename T, int V>
__device__ __forceinline__ void store_vec_nt(T* p, const float* in) {
  pack<T, V> a;
#pragma unroll
  for (int j = 0; j < V; ++j) a.v[j] = from_f32<T>(in[j]);
  __builtin_nontemporal_store(__builtin_bit_cast(vec16, a), reinterpret_cast<vec16*>(p));
}

template <int V>
__device__ __forceinline__ void store_codes(int8_t* p, const int* q) {
  pack<int8_t, V> a;
#pragma unroll
  for (int j = 0; j < V; ++j) a.v[j] = static_cast<int8_t>(q[j]);
  store_pack<int8_t, V>(p, a);
}

// ---- reductions over a wave on the vector ALU --------------------------------------------------------------------------------
// v of the lane that CTRL names, `rest` where there is none or where the row of 16 lanes is not in ROWS
template <int CTRL, int ROWS, typename T>
__device__ __forceinline__ T dpp(T v, T rest) {
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, rest), __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false));
  } else if constexpr (sizeof(T) == 16) {
    const unsigned long long lo = dpp<CTRL, ROWS>(static_cast<unsigned long long>(v), static_cast<unsigned long long>(rest));
    return static_cast<T>(dpp<CTRL, ROWS>(static_cast<unsigned long long>(v >> 64), static_cast<unsigned long long>(rest >> 64))) << 64 | lo;
  } else {
    const long long a = __builtin_bit_cast(long long, v), r = __builtin_bit_cast(long long, rest);
    const unsigned lo = __builtin_amdgcn_update_dpp(static_cast<int>(r), static_cast<int>(a), CTRL, ROWS, 0xf, false);
    const unsigned hi = __builtin_amdgcn_update_dpp(static_cast<int>(r >> 32), static_cast<int>(a >> 32), CTRL, ROWS, 0xf, false);
    return __builtin_bit_cast(T, static_cast<long long>(static_cast<unsigned long long>(hi) << 32 | lo));
  }
}

// op over the lanes up to this one, `rest` its neutral element: shifts by 1, 2, 4, 8 inside rows of 16 lanes, then lanes 15 and
// 31 into the rows behind them.  (A shuffle through LDS costs a hundred cycles a step.)
template <typename T, typename F>
__device__ __forceinline__ T wave_scan(T v, T rest, F op) {
  v = op(v, dpp<0x111, 0xf>(v, rest));
  v = op(v, dpp<0x112, 0xf>(v, rest));
  v = op(v, dpp<0x114, 0xf>(v, rest));
  v = op(v, dpp<0x118, 0xf>(v, rest));
  v = op(v, dpp<0x142, 0xa>(v, rest));
  v = op(v, dpp<0x143, 0xc>(v, rest));
  return v;
}
template <typename T>
__device__ __forceinline__ T from_lane(T v, int lane) {
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
  } else if constexpr (sizeof(T) == 16) {
    return static_cast<T>(from_lane(static_cast<unsigned long long>(v >> 64), lane)) << 64 | from_lane(static_cast<unsigned long long>(v), lane);
  } else {
    const long long a = __builtin_bit_cast(long long, v);
    const unsigned lo = __builtin_amdgcn_readlane(static_cast<int>(a), lane), hi = __builtin_amdgcn_readlane(static_cast<int>(a >> 32), lane);
    return __builtin_bit_cast(T, static_cast<long long>(static_cast<unsigned long long>(hi) << 32 | lo));
  }
}
template <typename T>
__device__ __forceinline__ T wave_sum(T v) {
  return from_lane(wave_scan(v, T{0}, [](T a, T b) { return a + b; }), kWave - 1);
}
__device__ __forceinline__ float wave_max(float v) {
  return from_lane(wave_scan(v, -__builtin_inff(), [](float a, float b) { return fmaxf(a, b); }), kWave - 1);
}
__device__ __forceinline__ double wave_max(double v) {
  return from_lane(wave_scan(v, -__builtin_inf(), [](double a, double b) { return fmax(a, b); }), kWave - 1);
}

}  // namespace sg
