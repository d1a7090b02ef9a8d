// gemm_i8.hip -- product of 8-bit codes with a scale for each row of either operand:
//
//   C[m, n] = act( sa[m] * sb[n] * sum_k A[m, k] B[n, k] + bias[n] ),   A (M, K), B (N, K) row-major codes
//
// B holds one output channel a row (an item's row, a dense layer's weight as it is stored).  The sums are exact in 32-bit
// integers (K < 2^17), so every kernel and every split of K gives the same bits; the epilogue rounds the sum to fp32, then
// once for each of its two products, once for the bias and once to C's type.
//
// Tile kernel.  v_mfma_i32_32x32x32_i8: a lane feeds 16 consecutive k of one row of A and one of B, so both operands are used
// exactly as they lie in memory.  A K step is 64 bytes of each of the tile's rows.  In LDS a row's four 16-byte chunks sit at
// slot = chunk ^ ((row >> 1) & 3): the eight rows that a b128 read touches at once then fall on eight different 16-byte bank
// groups.
//   * Aligned operands (base and pitch multiples of 16): LDS-DMA, NST stages, one barrier a K step, NST - 1 steps in flight.
//   * Otherwise, and for the last K step where K % 64 != 0: through registers, out-of-range k as zeros.
// Rows past M or N are read as the last row; nothing is stored for them.
#include "rows_shared.hpp"

#include <algorithm>
#include <type_traits>

#include "gemm_x3_shared.hpp"

namespace sg {
namespace i8 {

using i32x4 = __attribute__((ext_vector_type(4))) int;
using i32x16 = __attribute__((ext_vector_type(16))) int;
using f16x3::act_fn;
using f16x3::glb_void;
using f16x3::lds_void;

constexpr int BK = 64;      // bytes of a row in a K step

struct Args {
  void* C;
  const int8_t* A;
  const int8_t* B;
  const float* sa;
  const float* sb;
  const float* bias;
  int* ws;                 // split K: [splits][M][N] sums
  long long lda, ldb, ldc;
  int M, N, K, act, splits, steps_per_split, tiles_m, tiles_n;
  float slope;
};

template <typename T>
__device__ __forceinline__ void finish(const Args& g, T* c, int sum, float sa, float sb, float bias) {
  *c = from_f32<T>(act_fn(fmaf(static_cast<float>(sum) * sa, sb, bias), g.act, g.slope));
}

// 16 codes of a row from k on, zeros past K; any alignment
__device__ __forceinline__ i32x4 load_codes(const int8_t* row, int k, int K) {
  i32x4 v = {0, 0, 0, 0};
  if (k + 16 <= K) {
    __builtin_memcpy(&v, row + k, 16);
  } else if (k < K) {
    int8_t b[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) b[j] = k + j < K ? row[k + j] : static_cast<int8_t>(0);
    __builtin_memcpy(&v, b, 16);
  }
  return v;
}

template <int N>
__device__ __forceinline__ void wait_dma() {
  static_assert(N >= 0 && N < 64, "vmcnt has six bits");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));      // vmcnt(N); expcnt, lgkmcnt as they are
  asm volatile("" ::: "memory");
}

// tile TM x TN, waves of WM x WN; NST LDS stages; DMA: operands are 16-byte aligned
template <typename T, int TM, int TN, int WM, int WN, int NST, bool DMA>
__global__ __launch_bounds__(TM / WM * (TN / WN) * 64) void gemm_i8_kernel(const Args g) {
  constexpr int NWN = TN / WN, NW = TM / WM * NWN, IM = WM / 32, IN = WN / 32;
  constexpr int ROWS = TM + TN, STAGE = ROWS * BK, PIECES = ROWS / 16 / NW;      // a piece: 16 rows x 64 bytes, one wave access
  static_assert(ROWS % (16 * NW) == 0, "pieces divide over the waves");
  __shared__ __attribute__((aligned(16))) char smem[NST * STAGE];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int wm = wave / NWN, wn = wave % NWN;
  // workgroup b runs on XCD b % 8: give each XCD consecutive tiles, so that those that share rows of A share an L2
  const int nt = g.tiles_m * g.tiles_n, z = blockIdx.x / nt, lin = blockIdx.x - z * nt;
  const int q8 = nt >> 3, r8 = nt & 7, x8 = lin & 7;
  const int tile = (x8 < r8 ? x8 * (q8 + 1) : r8 * (q8 + 1) + (x8 - r8) * q8) + (lin >> 3);
  const int m0 = tile / g.tiles_n * TM, n0 = tile % g.tiles_n * TN;
  const int s0 = z * g.steps_per_split, s1 = min((g.K + BK - 1) / BK, s0 + g.steps_per_split);
  const int full = DMA ? min(s1, g.K / BK) : s0;       // steps [s0, full) by DMA, [full, s1) through registers

  // this wave's pieces: lane l moves chunk (l & 3) ^ ((row >> 1) & 3) of row l >> 2 to the piece's byte 16 l
  const int prow = lane >> 2, pchunk = (lane & 3) ^ ((prow >> 1) & 3);
  const int8_t* src[PIECES];
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const int r = (wave * PIECES + i) * 16 + prow;
    src[i] = r < TM ? g.A + static_cast<long long>(min(m0 + r, g.M - 1)) * g.lda
                    : g.B + static_cast<long long>(min(n0 + r - TM, g.N - 1)) * g.ldb;
  }
  auto issue = [&](int s) {
    char* st = smem + (s % NST) * STAGE + wave * PIECES * 1024;
#pragma unroll
    for (int i = 0; i < PIECES; ++i)
      __builtin_amdgcn_global_load_lds((glb_void*)(src[i] + s * BK + pchunk * 16), (lds_void*)(st + i * 1024), 16, 0, 0);
  };

  i32x16 acc[IM][IN];
#pragma unroll
  for (int i = 0; i < IM; ++i)
#pragma unroll
    for (int j = 0; j < IN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;
  const int l31 = lane & 31, kh = lane >> 5, sw = (l31 >> 1) & 3;      // a fragment row's swizzle: its block starts at a multiple of 32
  auto multiply = [&](int s) {
    const char* st = smem + (s % NST) * STAGE;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const int slot = ((ks * 2 + kh) ^ sw) * 16;
      i32x4 a[IM], b[IN];
#pragma unroll
      for (int i = 0; i < IM; ++i) a[i] = *reinterpret_cast<const i32x4*>(st + (wm * WM + i * 32 + l31) * BK + slot);
#pragma unroll
      for (int j = 0; j < IN; ++j) b[j] = *reinterpret_cast<const i32x4*>(st + (TM + wn * WN + j * 32 + l31) * BK + slot);
#pragma unroll
      for (int i = 0; i < IM; ++i)
#pragma unroll
        for (int j = 0; j < IN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[i], b[j], acc[i][j], 0, 0, 0);
    }
  };

  if constexpr (DMA) {
#pragma unroll
    for (int i = 0; i < NST - 1; ++i)
      if (s0 + i < full) issue(s0 + i);
    for (int s = s0; s < full; ++s) {
      if (s + NST - 2 < full) wait_dma<PIECES * (NST - 2)>();      // the pieces of step s have landed
      else wait_dma<0>();
      __builtin_amdgcn_s_barrier();                                // ... for every wave, and step s - 1 has been multiplied
      asm volatile("" ::: "memory");
      if (s + NST - 1 < full) issue(s + NST - 1);
      multiply(s);
    }
  }
  if (full < s1) {
    i32x4 v[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) v[i] = load_codes(src[i], full * BK + pchunk * 16, g.K);
    for (int s = full; s < s1; ++s) {
      __syncthreads();                                             // the stage's last readers are done
      char* st = smem + (s % NST) * STAGE + wave * PIECES * 1024 + lane * 16;
#pragma unroll
      for (int i = 0; i < PIECES; ++i) *reinterpret_cast<i32x4*>(st + i * 1024) = v[i];
      if (s + 1 < s1) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) v[i] = load_codes(src[i], (s + 1) * BK + pchunk * 16, g.K);
      }
      __syncthreads();
      multiply(s);
    }
  }

  // epilogue: a lane holds column l31 and rows (e & 3) + 8 (e >> 2) + 4 kh of each 32 x 32 block
#pragma unroll
  for (int j = 0; j < IN; ++j) {
    const int n = n0 + wn * WN + j * 32 + l31;
    if (n >= g.N) continue;
    const float sb = g.splits == 1 ? g.sb[n] : 0.f, bias = g.splits == 1 && g.bias ? g.bias[n] : 0.f;
#pragma unroll
    for (int i = 0; i < IM; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int m = m0 + wm * WM + i * 32 + (e & 3) + 8 * (e >> 2) + 4 * kh;
        if (m >= g.M) continue;
        if (g.splits == 1) finish(g, static_cast<T*>(g.C) + m * g.ldc + n, acc[i][j][e], g.sa[m], sb, bias);
        else g.ws[(static_cast<long long>(z) * g.M + m) * g.N + n] = acc[i][j][e];
      }
  }
}

// the splits' sums of one C element, and its epilogue
template <typename T>
__global__ __launch_bounds__(256) void gemm_i8_join_kernel(const Args g) {
  const long long mn = static_cast<long long>(g.M) * g.N;
  for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < mn; i += static_cast<long long>(gridDim.x) * 256) {
    int sum = 0;
    for (int z = 0; z < g.splits; ++z) sum += g.ws[z * mn + i];
    const int m = static_cast<int>(i / g.N), n = static_cast<int>(i - static_cast<long long>(m) * g.N);
    finish(g, static_cast<T*>(g.C) + m * g.ldc + n, sum, g.sa[m], g.sb[n], g.bias ? g.bias[n] : 0.f);
  }
}

struct Shape {
  int tm, tn, splits, steps_per_split;
};

// tile and split of K.  Small products are spread over the chip by splitting K while fewer than 256 tiles are at hand and a
// split keeps at least four steps.
inline Shape shape_of(int64_t M, int64_t N, int64_t K) {
  Shape s;
  s.tm = M <= 32 ? 32 : 128;
  s.tn = 128;
  const int64_t tiles = (M + s.tm - 1) / s.tm * ((N + s.tn - 1) / s.tn), steps = std::max<int64_t>(1, (K + BK - 1) / BK);
  int64_t splits = tiles >= 256 ? 1 : std::min<int64_t>(256 / tiles, steps / 4);
  splits = std::max<int64_t>(1, splits);
  s.steps_per_split = static_cast<int>((steps + splits - 1) / splits);
  s.splits = static_cast<int>((steps + s.steps_per_split - 1) / s.steps_per_split);
  return s;
}

template <typename T>
void launch(const Args& g, const Shape& s, bool dma, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(g.tiles_m * g.tiles_n * g.splits));
  if (s.tm == 32) {
    if (dma) hipLaunchKernelGGL((gemm_i8_kernel<T, 32, 128, 32, 64, 4, true>), grid, dim3(128), 0, st, g);
    else hipLaunchKernelGGL((gemm_i8_kernel<T, 32, 128, 32, 64, 2, false>), grid, dim3(128), 0, st, g);
  } else {
    if (dma) hipLaunchKernelGGL((gemm_i8_kernel<T, 128, 128, 64, 64, 3, true>), grid, dim3(256), 0, st, g);
    else hipLaunchKernelGGL((gemm_i8_kernel<T, 128, 128, 64, 64, 2, false>), grid, dim3(256), 0, st, g);
  }
  if (g.splits > 1) {
    const int64_t blocks = std::min<int64_t>(2048, (static_cast<int64_t>(g.M) * g.N + 255) / 256);
    hipLaunchKernelGGL(gemm_i8_join_kernel<T>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, st, g);
  }
}

}  // namespace i8
}  // namespace sg

using namespace sg;

SG_API size_t sg_gemm_i8_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  const i8::Shape s = i8::shape_of(M, N, K);
  return s.splits > 1 ? static_cast<size_t>(s.splits) * M * N * sizeof(int) : 0;
}

SG_API int sg_gemm_i8_hip(void* C, int64_t ldc, int dtype, const int8_t* A, int64_t lda, const float* sa, const int8_t* B,
                          int64_t ldb, const float* sb, const float* bias, int64_t M, int64_t N, int64_t K, int act, float slope,
                          void* workspace, size_t workspace_bytes, void* stream) {
  if (!valid_dtype(dtype)) return fail(SG_ERR_INVALID, "gemm_i8: unknown dtype %d", dtype);
  if (act < SG_ACT_NONE || act > SG_ACT_TANH) return fail(SG_ERR_INVALID, "gemm_i8: unknown activation %d", act);
  if (M < 0 || N < 0 || K < 0) return fail(SG_ERR_INVALID, "gemm_i8: negative size");
  if (K >= SG_GEMM_I8_MAX_K) return fail(SG_ERR_UNSUPPORTED, "gemm_i8: K must be below %d (32-bit sums)", SG_GEMM_I8_MAX_K);
  if (M >= (1ll << 30) || N >= (1ll << 30)) return fail(SG_ERR_UNSUPPORTED, "gemm_i8: M and N must be below 2^30");
  if (M == 0 || N == 0) return SG_OK;
  if (!C || !sa || !sb || (K > 0 && (!A || !B))) return fail(SG_ERR_INVALID, "gemm_i8: null pointer argument");
  if (lda < K || ldb < K || ldc < N) return fail(SG_ERR_INVALID, "gemm_i8: rows overlap");
  const i8::Shape s = i8::shape_of(M, N, K);
  i8::Args g{C, A, B, sa, sb, bias, static_cast<int*>(workspace), lda, ldb, ldc, static_cast<int>(M), static_cast<int>(N),
             static_cast<int>(K), act, s.splits, s.steps_per_split, static_cast<int>((M + s.tm - 1) / s.tm),
             static_cast<int>((N + s.tn - 1) / s.tn), slope};
  if (static_cast<int64_t>(g.tiles_m) * g.tiles_n * s.splits >= (1ll << 31)) return fail(SG_ERR_UNSUPPORTED, "gemm_i8: too many tiles");
  if (s.splits > 1 && (!workspace || workspace_bytes < sg_gemm_i8_workspace_bytes(M, N, K)))
    return fail(SG_ERR_WORKSPACE, "gemm_i8 workspace too small");
  const bool dma = aligned(A, 16) && aligned(B, 16) && lda % 16 == 0 && ldb % 16 == 0 && K >= i8::BK;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == SG_DTYPE_F32) i8::launch<float>(g, s, dma, st);
  else if (dtype == SG_DTYPE_F16) i8::launch<f16>(g, s, dma, st);
  else i8::launch<bf16>(g, s, dma, st);
  return check_launch("gemm_i8");
}
