// quant_rows.hip -- rows to 8-bit codes with one scale a row, optionally behind a root-mean-square norm with the residual's
// addition: what feeds the 8-bit product (gemm_i8.hip).
//
//   h = rnd(x + residual)      rounded to the type of x: the stored sum, and what everything below reads
//   y = h / sqrt(mean(h^2) + eps) * w              (norm)          y = h           (no norm)
//   scale = fl32(max|y| / 127),   code = rint(y / scale) in [-127, 127], ties to even
//
// A code is a decision at the border between two whole numbers, so everything up to it is held in 64 bits: the sum of
// squares, y (an fp32 h times an fp32 w is exact in 64 bits) and the quotient.  The card's 64-bit vector rate makes that
// cheap: ~10 operations an element against 7..13 bytes of memory traffic.  A row with an infinity or a NaN in it, or whose
// scale overflows 32 bits, has no codes: scale NaN, codes 0, so that a product with it is NaN (0 behind relu, as the
// library has it).  A row of zeros has scale 0.
//
// Memory bound: x and the residual are read once, codes and the sum written once; a row stays in the registers of its
// threads between its reduction and its codes.  69878 x 256 fp32 with a residual: 43 us, 5.4 TB/s; 8192 x 4096 bf16: 50 us, 4.7
// TB/s (a copy reaches 5.3).
#include "common.hpp"
#include "rows_shared.hpp"

#include <algorithm>

namespace sg {
namespace {

struct QuantArgs {
  int8_t* codes;
  float* scale;
  void* sum;
  const void* x;
  const void* res;
  const void* w;
  long long ldx, ldr;
  long long rows;
  int dim, norm, w_f32;
  double eps;
};

// TPR threads a row, NV vectors of V elements a thread; V divides the row's length, so a vector is whole or not there.  All of a
// thread's loads are issued before the first is used.
template <typename T, int TPR, int V, int NV>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void quant_rows_kernel(const QuantArgs g) {
  constexpr int THREADS = TPR < 256 ? 256 : TPR, RPB = THREADS / TPR, WPR = TPR / kWave;
  __shared__ double red[2][THREADS / kWave];
  const int t = threadIdx.x % TPR;
  const long long mine = static_cast<long long>(blockIdx.x) * RPB + threadIdx.x / TPR, row = min(mine, g.rows - 1);
  const bool live = mine < g.rows;
  const T* x = static_cast<const T*>(g.x) + row * g.ldx;
  const T* res = static_cast<const T*>(g.res) + row * g.ldr;
  pack<T, V> xs[NV], rs[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + t) * V, at = c < g.dim ? c : 0;       // past the row: its first elements, not used
    xs[i] = load_pack<T, V>(x + at);
    if (g.res) rs[i] = load_pack<T, V>(res + at);
  }
  double p[NV][V];                                       // h * w, exact
  double ss = 0.0, top = 0.0, bad = 0.0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + t) * V;
    const bool in = live && c < g.dim;
    float h[V], w[V];
#pragma unroll
    for (int j = 0; j < V; ++j) h[j] = to_f32(xs[i].v[j]), w[j] = 1.f;
    if (g.res) {
#pragma unroll
      for (int j = 0; j < V; ++j) h[j] = round_to<T>(h[j] + to_f32(rs[i].v[j]));
    }
    if (g.sum && in) {
#pragma unroll
      for (int j = 0; j < V; ++j) xs[i].v[j] = from_f32<T>(h[j]);
      store_pack<T, V>(static_cast<T*>(g.sum) + row * g.dim + c, xs[i]);
    }
    if (g.w) {
      const int at = c < g.dim ? c : 0;
      if (g.w_f32) {
        const pack<float, V> a = load_pack<float, V>(static_cast<const float*>(g.w) + at);
#pragma unroll
        for (int j = 0; j < V; ++j) w[j] = a.v[j];
      } else {
        const pack<T, V> a = load_pack<T, V>(static_cast<const T*>(g.w) + at);
#pragma unroll
        for (int j = 0; j < V; ++j) w[j] = to_f32(a.v[j]);
      }
    }
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (!in) h[j] = 0.f, w[j] = 0.f;
      const double hd = h[j];
      p[i][j] = hd * static_cast<double>(w[j]);
      if (g.norm) ss = fma(hd, hd, ss);
      top = fmax(top, fabs(p[i][j]));
      bad = fma(p[i][j], 0.0, bad);                      // NaN once a value is not finite (fmax drops NaNs)
    }
  }
  ss += bad;
  ss = wave_sum(ss), top = wave_max(top);
  if (WPR > 1) {
    const int wave = threadIdx.x / kWave;
    if (threadIdx.x % kWave == 0) red[0][wave] = ss, red[1][wave] = top;
    __syncthreads();
    ss = 0.0, top = 0.0;
#pragma unroll
    for (int i = 0; i < WPR; ++i) ss += red[0][i], top = fmax(top, red[1][i]);
  }
  if (!live) return;
  const double rstd = !g.norm ? 1.0 : top == 0.0 ? 0.0 : 1.0 / sqrt(ss / g.dim + g.eps);      // zeros stay zeros, whatever eps
  float scale = static_cast<float>(top * rstd / 127.0);
  const bool none = ss != ss || !(scale <= 3.402823466e38f);        // NaN and infinities
  if (none) scale = __builtin_nanf("");
  if (t == 0) g.scale[row] = scale;
  const double s = scale, inv = (none || scale == 0.f) ? 0.0 : 1.0 / s;
  int8_t* codes = g.codes + row * g.dim;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (i * TPR + t) * V;
    int q[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const double y = none ? 0.0 : p[i][j] * rstd, a = y * inv;
      double k = rint(a);
      if (fabs(fabs(a - k) - 0.5) < 1e-6) {              // near a tie: decide by the exact remainder, not the reciprocal
        const double r = fma(-k, s, y), far = 2.0 * fabs(r) - s;
        const bool odd = (static_cast<int>(k) & 1) != 0;
        if (far > 0.0 || (far == 0.0 && odd)) k += copysign(1.0, r);
      }
      q[j] = static_cast<int>(fmin(fmax(k, -127.0), 127.0));
    }
    if (c < g.dim) store_codes<V>(codes + c, q);
  }
}

template <typename T, int TPR, int V, int E>
void launch(const QuantArgs& g, hipStream_t st) {
  constexpr int THREADS = TPR < 256 ? 256 : TPR, RPB = THREADS / TPR;
  hipLaunchKernelGGL((quant_rows_kernel<T, TPR, V, E / V>), dim3(static_cast<unsigned>((g.rows + RPB - 1) / RPB)), dim3(THREADS), 0, st, g);
}

// the narrowest form that holds a row: a wave for short rows (no barrier, four rows a workgroup), else a workgroup
template <typename T, int V>
void dispatch(const QuantArgs& g, hipStream_t st) {
  constexpr int E = 16 / sizeof(T);                      // elements of 16 bytes
  if (g.dim <= 64 * E) launch<T, 64, V, E>(g, st);
  else if (g.dim <= 128 * E) launch<T, 64, V, 2 * E>(g, st);
  else if (g.dim <= 256 * E) launch<T, 256, V, E>(g, st);
  else if (g.dim <= 512 * E) launch<T, 256, V, 2 * E>(g, st);
  else if (g.dim <= 1024 * E) launch<T, 256, V, 4 * E>(g, st);
  else if (g.dim <= 2048 * E) launch<T, 1024, V, 2 * E>(g, st);
  else if constexpr (sizeof(T) == 4) launch<T, 1024, V, 4 * E>(g, st);
}

// vectors as wide as the row's length allows
template <typename T>
void dispatch(const QuantArgs& g, hipStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (g.dim % 8 == 0) return dispatch<T, 8>(g, st);
  }
  if (g.dim % 4 == 0) return dispatch<T, 4>(g, st);
  if (g.dim % 2 == 0) return dispatch<T, 2>(g, st);
  return dispatch<T, 1>(g, st);
}

}  // namespace
}  // namespace sg

using namespace sg;

SG_API int sg_quant_rows_i8_hip(int8_t* codes, float* scale, void* sum, const void* x, int64_t ldx, const void* residual,
                                int64_t ldr, const void* weight, int weight_f32, int64_t rows, int64_t dim, int dtype, int norm,
                                double eps, void* stream) {
  if (!valid_dtype(dtype)) return fail(SG_ERR_INVALID, "quant_rows: unknown dtype %d", dtype);
  if (rows < 0 || dim < 1 || rows >= (1ll << 31)) return fail(SG_ERR_INVALID, "quant_rows: bad shape");
  if (dim > SG_QUANT_ROWS_MAX_DIM) return fail(SG_ERR_UNSUPPORTED, "quant_rows: rows of at most %d elements", SG_QUANT_ROWS_MAX_DIM);
  if (norm && !(eps >= 0.0)) return fail(SG_ERR_INVALID, "quant_rows: eps must not be negative");
  if (rows == 0) return SG_OK;
  if (!codes || !scale || !x) return fail(SG_ERR_INVALID, "quant_rows: null pointer argument");
  if (ldx < dim || (residual && ldr < dim)) return fail(SG_ERR_INVALID, "quant_rows: rows overlap");
  if (sum && rows > 1 && ((sum == x && ldx != dim) || (sum == residual && ldr != dim)))
    return fail(SG_ERR_INVALID, "quant_rows: a sum in place needs rows without gaps");
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int64_t size = dtype == SG_DTYPE_F32 ? 4 : 2, most = int64_t{1} << 21;      // a launch has to stay below 2^32 threads
  for (int64_t r = 0; r < rows; r += most) {
    auto of = [&](auto* p, int64_t ld) { return p ? reinterpret_cast<decltype(p)>(reinterpret_cast<uintptr_t>(p) + r * ld * size) : p; };
    const QuantArgs g{codes + r * dim, scale + r, of(sum, dim), of(x, ldx), of(residual, ldr), weight, ldx, ldr, std::min(most, rows - r),
                      static_cast<int>(dim), norm, weight_f32, eps};
    if (dtype == SG_DTYPE_F32) dispatch<float>(g, st);
    else if (dtype == SG_DTYPE_F16) dispatch<f16>(g, st);
    else dispatch<bf16>(g, st);
  }
  return check_launch("quant_rows");
}
