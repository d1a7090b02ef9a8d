// gemm_i8.hip -- product of 8-bit codes with a scale for each row of either operand:
//
//   C[m, n] = act( sa[m] * sb[n] * sum_k A[m, k] B[n, k] + bias[n] ),   A (M, K), B (N, K) row-major codes
//
// B holds one output channel a row (an item's row, a dense layer's weight as it is stored).  The sums are exact in 32-bit
// integers (K < 2^17), so every kernel and every split of K gives the same bits; the epilogue rounds the sum to fp32, its product
// with sa, the fused product with sb and bias, and the result to C's type.  The product of the three is right over fp32's whole
// range: waves in which some sa is 2^97 or more, or below the normal numbers, take a path of their own.
//
// Tile kernel.  v_mfma_i32_32x32x32_i8: a lane feeds 16 consecutive k of one row of A and one of B, so both operands are used
// exactly as they lie in memory.  A K step is 64 or 128 bytes of each of the tile's rows.  In LDS a row's 16-byte chunks sit at
// slot = chunk ^ swizzle(row), chosen so that the 16 rows that a b128 read touches at once fall on 16 different 16-byte groups
// of the 64 banks (SQ_LDS_BANK_CONFLICT 0 in the steps; the first choice, for eight rows at once, cost half of the LDS cycles).
//   * Aligned operands (base and pitch multiples of 16): LDS-DMA by buffer loads, whose addresses are one register a piece and
//     a scalar step; one barrier a step, the next step's pieces are issued between the last matrix instructions of a step.
//   * Otherwise, and for the last step where K is no multiple of it: through registers, out-of-range k as zeros.
// Rows past M or N are read as the last row; nothing is stored for them.
//
// What bounds it, measured on an MI355X.  8192 x 8192 x 4096 into bf16: 229 us, 2.4 POP/s, for quantised normal rows, 281 us for
// uniformly random codes, 181 us for zeros: the chip's power sets the clock (1.7 GHz in the counters' runs), the matrix units are
// busy 72 % of the cycles.  A K-short product (10000 x 10677 x 256 into fp32) is bound by its stores: 106 to 112 us, 4 TB/s
// against 6.6 TB/s of a fill of the same buffer; K = 250, through registers, takes 115 to 118.  One row against 10677: 4.5 us of a call of 12.
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

constexpr int GROUP = 8;                   // columns of tiles in a band; 4 and 16 run from 1 % faster to 4 % slower

// slot of 16-byte chunk c of a row in LDS: c ^ swizzle(row)
template <int BK>
__device__ __forceinline__ int swizzle(int row) {
  static_assert(BK == 64 || BK == 128, "rows of 64 or 128 bytes");
  return BK == 64 ? (row >> 2) & 3 : (row >> 1) & 7;
}

struct Args {
  void* C;
  const int8_t* A;
  const int8_t* B;
  const float* sa;
  const float* sb;
  const float* bias;
  int* ws;                 // split K: [splits][M][N] sums
  long long lda, ldb, ldc;
  int M, N, K, act, splits, k_per_split, tiles_m, tiles_n;
  float slope;
  int nt;                  // store past the caches: C's rows are 16-byte aligned, and C is larger than the Infinity Cache
};

// Whether sum * sa can leave fp32's range, or its normal numbers, where the product with sb need not: sums are below 2^31.
__device__ __forceinline__ bool far_scale(float sa) {
  const float a = fabsf(sa);
  return (a >= 0x1p97f && a <= 3.402823466e38f) || (a < 0x1p-126f && a > 0.f);
}
// sum * sa * sb + bias for any scales: a far sa takes 2^64 from sb or gives it 2^64.  Where sb leaves the range by that the product
// does too (above, a sum of 1 times 2^97 times 2^64), or is nothing (below 2^31 2^-62 2^-126).
__device__ __forceinline__ float scaled(int sum, float sa, float sb, float bias) {
  if (far_scale(sa)) {
    const bool large = fabsf(sa) >= 1.f;
    sa *= large ? 0x1p-64f : 0x1p64f;
    const float far = sb * (large ? 0x1p64f : 0x1p-64f);
    sb = fabsf(sb) <= 3.402823466e38f ? fminf(fmaxf(far, -3.402823466e38f), 3.402823466e38f) : far;
  }
  return fmaf(static_cast<float>(sum) * sa, sb, bias);
}

template <typename T>
__device__ __forceinline__ void finish(const Args& g, T* c, int sum, float sa, float sb, float bias) {
  *c = from_f32<T>(act_fn(scaled(sum, sa, sb, bias), g.act, g.slope));
}

// 16 codes of a row from k on, zeros past K; any alignment.  Where they end past K the row's last 16 are loaded and moved down, so
// that no load hangs on a condition.
__device__ __forceinline__ i32x4 load_codes(const int8_t* row, int k, int K) {
  if (K >= 16) {
    typedef unsigned long long u64x2 __attribute__((ext_vector_type(2)));
    const int at = min(k, K - 16), gone = (k - at) * 8;      // bits to move down
    const u64x2 v = __builtin_bit_cast(u64x2, static_cast<vec16>(*reinterpret_cast<const vec16_any*>(row + at)));
    const unsigned long long far = v[1] >> (gone & 63), near = (v[0] >> (gone & 63)) | (gone & 63 ? v[1] << (64 - (gone & 63)) : 0);
    u64x2 r;
    r[0] = gone < 64 ? near : gone < 128 ? far : 0;
    r[1] = gone < 64 ? far : 0;
    return __builtin_bit_cast(i32x4, r);
  }
  int8_t b[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) b[j] = k + j < K ? row[k + j] : static_cast<int8_t>(0);
  return __builtin_bit_cast(i32x4, b);
}

template <int N>
__device__ __forceinline__ void wait_dma() {
  static_assert(N >= 0 && N < 64, "vmcnt has six bits");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));      // vmcnt(N); expcnt, lgkmcnt as they are
  asm volatile("" ::: "memory");
}

// Waves a SIMD that the registers have to leave room for: 128 of them let two workgroups of 128 x 256 into a compute unit, of which
// one stores while the other multiplies (10000 x 10677 x 250 into fp32: 126 us a call, with 130 registers 138).  The 16-bit types
// and the DMA forms of this tile need 132 and more, and spill if held to 128.
template <typename T, int TM, int TN, bool DMA>
constexpr int kWavesPerSimd = sizeof(T) == 4 && TM == 128 && TN == 256 && !DMA ? 4 : 1;

// tile TM x TN, waves of WM x WN, K steps of BK bytes, NST LDS stages; DMA: operands are 16-byte aligned
template <typename T, int TM, int TN, int WM, int WN, int BK, int NST, bool DMA, bool ACT>
__global__ __launch_bounds__(TM / WM * (TN / WN) * 64, (kWavesPerSimd<T, TM, TN, DMA>)) void gemm_i8_kernel(const Args g) {
  constexpr int NWN = TN / WN, NW = TM / WM * NWN, IM = WM / 32, IN = WN / 32, H = BK / 32;
  constexpr int CPR = BK / 16, RP = 64 / CPR;                           // 16-byte chunks a row; a piece: RP rows x BK bytes, one wave access
  constexpr int PA = TM / RP / NW, PB = TN / RP / NW, PIECES = PA + PB, STAGE = (TM + TN) * BK;
  constexpr int V = 16 / sizeof(T), LPR = WN / V, RPP = 64 / LPR;       // epilogue: lanes a row, rows a pass
  constexpr int CP = WN + 4, CST = 32 * CP;                             // a wave's part of LDS: 32 rows, padded
  static_assert(TM % (RP * NW) == 0 && TN % (RP * NW) == 0, "pieces divide over the waves");
  constexpr int SMEM = NST * STAGE > NW * CST * 4 ? NST * STAGE : NW * CST * 4;
  __shared__ __attribute__((aligned(16))) char smem[SMEM];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int wm = wave / NWN, wn = wave % NWN;
  // workgroup b runs on XCD b % 8: give each XCD consecutive tiles, so that those that share rows share an L2
  const int nt = g.tiles_m * g.tiles_n, z = blockIdx.x / nt, lin = blockIdx.x - z * nt;
  const int q8 = nt >> 3, r8 = nt & 7, x8 = lin & 7;
  const int tile = (x8 < r8 ? x8 * (q8 + 1) : r8 * (q8 + 1) + (x8 - r8) * q8) + (lin >> 3);
  // tiles in bands of GROUP columns, by rows inside a band: the tiles of an XCD at one time share rows of A and of B
  const int band = tile / (GROUP * g.tiles_m), in_band = tile - band * GROUP * g.tiles_m, width = min(GROUP, g.tiles_n - band * GROUP);
  const int m0 = in_band / width * TM, n0 = (band * GROUP + in_band % width) * TN;
  const int k0 = z * g.k_per_split, k1 = min(g.K, k0 + g.k_per_split);  // this split's k; k0 is a multiple of every BK
  const int steps = (k1 - k0 + BK - 1) / BK, full = DMA ? (k1 - k0) / BK : 0;      // steps [0, full) by DMA, [full, steps) through registers

  // this wave's pieces: lane l moves chunk (l % CPR) ^ swizzle(row) of row l / CPR to the piece's byte 16 l
  const int prow = lane / CPR;
  const int8_t* pa = g.A + m0 * g.lda + k0;
  const int8_t* pb = g.B + n0 * g.ldb + k0;
  const auto ra = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(pa), 0, 0xffffffffu, 0x00027000);
  const auto rb = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(pb), 0, 0xffffffffu, 0x00027000);
  typename std::conditional<DMA, unsigned, long long>::type off[PIECES];      // by DMA the pitch is bounded
  auto chunk = [&](int i) { return ((lane % CPR) ^ swizzle<BK>((i < PA ? wave * PA + i : wave * PB + i - PA) * RP + prow)) * 16; };
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const int r = (i < PA ? wave * PA + i : wave * PB + i - PA) * RP + prow;
    off[i] = (i < PA ? min(r, g.M - 1 - m0) * g.lda : min(r, g.N - 1 - n0) * g.ldb) + (DMA ? chunk(i) : 0);
  }
  auto piece = [&](int s, int i) { return smem + (s % NST) * STAGE + (i < PA ? wave * PA + i : TM / RP + wave * PB + i - PA) * 1024; };
  auto issue = [&](int s, int i) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(i < PA ? ra : rb, (lds_void*)piece(s, i), 16, static_cast<int>(off[i]), s * BK, 0, 0);
  };

  // what the epilogue scales with, loaded ahead of the steps
  const bool whole = g.splits == 1;
  const int col = lane % LPR * V, n = n0 + wn * WN + col, room = g.N - n, mw = m0 + wm * WM;
  float sb[V], bias[V], sa[IM];                        // sa: row lane % 32 of each 32-row block
#pragma unroll
  for (int q = 0; q < V; ++q) {
    sb[q] = whole ? g.sb[min(n + q, g.N - 1)] : 0.f;
    bias[q] = whole && g.bias ? g.bias[min(n + q, g.N - 1)] : 0.f;
  }
#pragma unroll
  for (int i = 0; i < IM; ++i) sa[i] = whole ? g.sa[min(mw + i * 32 + (lane & 31), g.M - 1)] : 0.f;

  i32x16 acc[IM][IN];
#pragma unroll
  for (int i = 0; i < IM; ++i)
#pragma unroll
    for (int j = 0; j < IN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;
  const int l31 = lane & 31, kh = lane >> 5, sw = swizzle<BK>(l31);     // a fragment's rows start at a multiple of 32
  const int a_row = (wm * WM + l31) * BK, b_row = (TM + wn * WN + l31) * BK;
  i32x4 a[2][IM], b[2][IN];                            // fragments of 32 k: one set multiplied, one being read
  auto read_one = [&](int s, int ks, int f) {
    const char* st = smem + (s % NST) * STAGE + ((ks * 2 + kh) ^ sw) * 16;
    if (f < IM) a[ks & 1][f] = *reinterpret_cast<const i32x4*>(st + a_row + f * 32 * BK);
    else b[ks & 1][f - IM] = *reinterpret_cast<const i32x4*>(st + b_row + (f - IM) * 32 * BK);
  };
  auto read = [&](int s, int ks) {
#pragma unroll
    for (int f = 0; f < IM + IN; ++f) read_one(s, ks, f);
  };
  // between(q) goes before matrix instruction q and stays there: left alone, the compiler moves the reads of the next fragments
  // down to their use and the matrix units wait for them
  auto multiply = [&](int ks, auto between) {
#pragma unroll
    for (int i = 0; i < IM; ++i)
#pragma unroll
      for (int j = 0; j < IN; ++j) {
        between(i * IN + j);
        acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(a[ks & 1][i], b[ks & 1][j], acc[i][j], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
  };
  auto read_next = [&](int q, int s, int ks) {         // a fragment's share of the reads, in the first half of the matrix instructions
#pragma unroll
    for (int f = 0; f < IM + IN; ++f)
      if (f * IM * IN / (2 * (IM + IN)) == q) read_one(s, ks, f);
  };
  auto nothing = [](int) {};

  if constexpr (DMA) {
    // While 32 k are multiplied the next 32 are read.  The barrier before the last 32 k of step s says that step s + 1 has landed
    // for every wave and that step s has been read out, whose stage then receives step s + NST.
    if (full > 0) {
#pragma unroll
      for (int p = 0; p < NST; ++p)
        if (p < full)
#pragma unroll
          for (int i = 0; i < PIECES; ++i) issue(p, i);
      if (NST - 1 < full) wait_dma<PIECES * (NST - 1)>();
      else wait_dma<0>();
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      read(0, 0);
    }
    auto step = [&](int s, auto more) {                // more: step s + NST exists
#pragma unroll
      for (int ks = 0; ks < H - 1; ++ks) {
        multiply(ks, [&](int q) { read_next(q, s, ks + 1); });
      }
      if (more.value || s + 1 < full) {
        if (more.value || s + NST - 1 < full) wait_dma<PIECES * (NST - 2)>();
        else wait_dma<0>();
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
      }
      multiply(H - 1, [&](int q) {
        if (more.value || s + 1 < full) read_next(q, s + 1, 0);
        if constexpr (more.value) {
#pragma unroll
          for (int i = 0; i < PIECES; ++i)
            if (i * IM * IN / PIECES == q) issue(s + NST, i);
        }
      });
    };
    int s = 0;
    for (; s + NST < full; ++s) step(s, std::true_type{});
    for (; s < full; ++s) step(s, std::false_type{});
  }
  if (full < steps) {
    i32x4 v[PIECES];
    auto load = [&](int s) {
      if ((s + 1) * BK <= k1 - k0) {                               // a whole step: nothing to look at
#pragma unroll
        for (int i = 0; i < PIECES; ++i)
          v[i] = *reinterpret_cast<const vec16_any*>((i < PA ? pa : pb) + (off[i] - (DMA ? chunk(i) : 0)) + s * BK + chunk(i));
      } else {
#pragma unroll
        for (int i = 0; i < PIECES; ++i)
          v[i] = load_codes((i < PA ? pa : pb) + (off[i] - (DMA ? chunk(i) : 0)), s * BK + chunk(i), k1 - k0);
      }
    };
    load(full);
    for (int s = full; s < steps; ++s) {
      __syncthreads();                                             // the stage's last readers are done
#pragma unroll
      for (int i = 0; i < PIECES; ++i) *reinterpret_cast<i32x4*>(piece(s, i) + lane * 16) = v[i];
      if (s + 1 < steps) load(s + 1);
      __syncthreads();
#pragma unroll
      for (int ks = 0; ks < H; ++ks) {
        read(s, ks);
        multiply(ks, nothing);
      }
    }
  }

  // epilogue: 32 rows at a time through the wave's own part of LDS, where a lane's column of sums (column l31, rows
  // (e & 3) + 8 (e >> 2) + 4 kh of each 32 x 32 block) becomes 16 bytes of a row of C
  __syncthreads();
  int* cst = reinterpret_cast<int*>(smem) + wave * CST;
  const int first = lane / LPR, rows = g.M - mw - first;
  const auto block = [&](int i, auto rolled, auto use) {      // use(r, sums): row r of the 32, V sums from column `col` on
#pragma unroll
    for (int j = 0; j < IN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) cst[((e & 3) + 8 * (e >> 2) + 4 * kh) * CP + j * 32 + l31] = acc[i][j][e];
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    constexpr int UN = ACT || rolled.value ? 1 : 32 / RPP;      // unrolled, the activations' code overflows the instruction cache
#pragma unroll UN
    for (int it = 0; it < 32 / RPP; ++it) {
      int v[V];
#pragma unroll
      for (int q = 0; q < V; q += 4) {
        const i32x4 t4 = *reinterpret_cast<const i32x4*>(cst + (it * RPP + first) * CP + col + q);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[q + e] = t4[e];
      }
      use(it * RPP + first, v);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  };
  const auto finish_all = [&](auto far, auto store) {  // far: some row's scale is, see far_scale
    T* o = static_cast<T*>(g.C) + (mw + first) * g.ldc + n;
    const long long stride = RPP * g.ldc;
#pragma unroll
    for (int i = 0; i < IM; ++i)
      block(i, far, [&](int r, const int* v) {
        const float sa_r = __shfl(sa[i], r);
        float f[V];
#pragma unroll
        for (int q = 0; q < V; ++q) {
          f[q] = far.value ? scaled(v[q], sa_r, sb[q], bias[q]) : fmaf(static_cast<float>(v[q]) * sa_r, sb[q], bias[q]);
          if (ACT) f[q] = act_fn(f[q], g.act, g.slope);
        }
        store(o, f, i * 32 + r - first);
        o += stride;
      });
  };
  if (!whole) {
    int* w = g.ws + (static_cast<long long>(z) * g.M + mw + first) * g.N + n;
#pragma unroll
    for (int i = 0; i < IM; ++i)
      block(i, std::false_type{}, [&](int r, const int* v) {
        if (i * 32 + r - first < rows) {
#pragma unroll
          for (int q = 0; q < V; ++q)
            if (q < room) w[q] = v[q];
        }
        w += RPP * g.N;
      });
    return;
  }
  bool far = false;
#pragma unroll
  for (int i = 0; i < IM; ++i) far = far || far_scale(sa[i]);
  const auto store_checked = [&](T* o, const float* f, int r) {
    if (r < rows && room > 0) store_vec<T, V>(o, f, room);
  };
  if (__ballot(far) != 0) finish_all(std::true_type{}, store_checked);
  else if (m0 + TM > g.M || n0 + TN > g.N) finish_all(std::false_type{}, store_checked);
  else if (g.nt) finish_all(std::false_type{}, [](T* o, const float* f, int) { store_vec_nt<T, V>(o, f); });
  else finish_all(std::false_type{}, [](T* o, const float* f, int) { store_vec<T, V>(o, f, V); });
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
  int tm, tn, splits, k_per_split;
};

// The largest tile of which there are enough for all 256 compute units: it moves the fewest operand bytes a product.  Measured
// (us, tiles of 256 x 256 / 128 x 256 / 128 x 128): 8192 x 8192 x 2048 162 / 185 / 175, 8192 x 8192 x 512 60 / 70 / 69; for K
// below 512 the epilogue is all, and more and smaller workgroups hide it: 8192 x 8192 x 256 59 / 52 / 54.  Where not even 128 x
// 128 gives 256 tiles, 32 x 128 (200 x 4096 x 4096: 16 against 27), and K is split while a split keeps 256 k.
inline Shape shape_of(int64_t M, int64_t N, int64_t K) {
  auto tiles = [&](int tm, int tn) { return (M + tm - 1) / tm * ((N + tn - 1) / tn); };
  Shape s;
  if (K >= 512 && tiles(256, 256) >= 256) s.tm = 256, s.tn = 256;
  else if (tiles(128, 256) >= 256) s.tm = 128, s.tn = 256;
  else if (tiles(128, 128) >= 256) s.tm = 128, s.tn = 128;
  else s.tm = 32, s.tn = 128;
  const int64_t n = tiles(s.tm, s.tn), steps = std::max<int64_t>(1, (K + 127) / 128);
  const int64_t splits = n >= 256 ? 1 : std::max<int64_t>(1, std::min<int64_t>(256 / n, steps / 2));
  s.k_per_split = static_cast<int>((steps + splits - 1) / splits * 128);
  s.splits = static_cast<int>(std::max<int64_t>(1, (K + s.k_per_split - 1) / s.k_per_split));
  return s;
}

template <typename T, int TM, int TN, int WM, int WN, int BK, int NST, bool DMA>
void go(const Args& g, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(g.tiles_m * g.tiles_n * g.splits)), block(TM / WM * (TN / WN) * 64);
  if (g.act == SG_ACT_NONE) hipLaunchKernelGGL((gemm_i8_kernel<T, TM, TN, WM, WN, BK, NST, DMA, false>), grid, block, 0, st, g);
  else hipLaunchKernelGGL((gemm_i8_kernel<T, TM, TN, WM, WN, BK, NST, DMA, true>), grid, block, 0, st, g);
}

template <typename T>
void launch(const Args& g, const Shape& s, bool dma, hipStream_t st) {
  if (s.tm == 256) {
    if (dma) go<T, 256, 256, 128, 64, 128, 2, true>(g, st);
    else go<T, 256, 256, 128, 64, 64, 2, false>(g, st);
  } else if (s.tm == 128 && s.tn == 256) {
    if (dma && g.K >= 512) go<T, 128, 256, 64, 64, 128, 2, true>(g, st);
    else if (dma) go<T, 128, 256, 64, 64, 64, 2, true>(g, st);
    else go<T, 128, 256, 64, 64, 64, 2, false>(g, st);
  } else if (s.tm == 128) {
    if (dma) go<T, 128, 128, 64, 64, 128, 2, true>(g, st);
    else go<T, 128, 128, 64, 64, 64, 2, false>(g, st);
  } else {
    if (dma) go<T, 32, 128, 32, 64, 64, 4, true>(g, st);
    else go<T, 32, 128, 32, 64, 64, 2, false>(g, st);
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
             static_cast<int>(K), act, s.splits, s.k_per_split, static_cast<int>((M + s.tm - 1) / s.tm),
             static_cast<int>((N + s.tn - 1) / s.tn), slope, 0};
  const int size = dtype == SG_DTYPE_F32 ? 4 : 2;
  // measured at 10000 x 10752 into fp32: 93 us past the caches, 99 through them
  g.nt = aligned(C, 16) && ldc * size % 16 == 0 && M * N * size > (256ll << 20);
  if (static_cast<int64_t>(g.tiles_m) * g.tiles_n * s.splits >= (1ll << 23)) return fail(SG_ERR_UNSUPPORTED, "gemm_i8: too many tiles");
  if (s.splits > 1 && (!workspace || workspace_bytes < sg_gemm_i8_workspace_bytes(M, N, K)))
    return fail(SG_ERR_WORKSPACE, "gemm_i8 workspace too small");
  const bool dma = aligned(A, 16) && aligned(B, 16) && lda % 16 == 0 && ldb % 16 == 0 && lda <= SG_GEMM_I8_MAX_K * 64 && ldb <= SG_GEMM_I8_MAX_K * 64;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == SG_DTYPE_F32) i8::launch<float>(g, s, dma, st);
  else if (dtype == SG_DTYPE_F16) i8::launch<f16>(g, s, dma, st);
  else i8::launch<bf16>(g, s, dma, st);
  return check_launch("gemm_i8");
}
