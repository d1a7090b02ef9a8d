// distill.hip -- a student's scores fitted to a teacher's top scores: forward and backward.
//
//   q = softmax(s / T) over a row's N items,  p = softmax(t / T) over the teacher's K entries of the row
//   loss = scale * T^2 * sum_rows sum_k p_k (log p_k - log q_{id_k}),        d loss / d s_j = scale * T * (q_j - sum_{id_k = j} p_k)
//
// An entry whose id lies outside [0, N) or whose score is -inf is no entry.  A row without an entry, or whose student scores
// are all -inf, has nothing to fit: it adds no loss and its gradient is zero.  An item that is named twice takes both shares.
//
// Bound by memory: the forward reads the scores once (running maximum and sum, one exp an element), the backward reads them
// again and writes the gradient; the K entries of a row are noise next to its N scores.  Long rows of small batches are split
// over workgroups and joined.  Exponents are taken of differences from the row's largest score, so T scales exact differences;
// the K terms of the loss, which cancel where the student is close, are formed in 64 bits.
#include "rows_shared.hpp"

#include <algorithm>

namespace sg {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / kWave;

struct DistillArgs {
  const void* s;
  const float* t;
  const int32_t* ids;
  float* stats;            // (rows, 2): largest score, 1 / sum exp (0: the row has nothing to fit)
  float* p;                // (rows, K)
  float* part;             // (rows, splits, 2): running maximum and sum of a piece
  float* row_loss;         // (rows)
  void* grad;
  const float* gout;
  long long ld;
  int rows, n, k, splits, piece;
  float temperature, scale;
};

constexpr float kLowest = -3.402823466e38f, kLog2e = 1.442695040888963f;

// v_exp_f32 itself: results below 2^-126 come out as 0, which neither a sum of at least 1 nor a gradient misses
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// (m, s) <- the maximum and sum of both; s counts exp((x - m) / T)
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2, float c) {
  const float top = fmaxf(m, m2);
  s = s * exp2_fast((m - top) * c) + s2 * exp2_fast((m2 - top) * c);
  m = top;
}

template <typename T>
__device__ __forceinline__ void piece_max_sum(const DistillArgs& g, const T* row, int lo, int hi, float c, float& m, float& s) {
  constexpr int V = 16 / sizeof(T), U = 4, STEP = kThreads * V;
  m = kLowest, s = 0.f;
  for (int base = lo + threadIdx.x * V; base < hi; base += U * STEP) {
    float x[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int n = hi - (base + u * STEP);
      load_vec<T, V>(x[u], row + base + u * STEP, n);
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (j >= n) x[u][j] = -__builtin_inff();
    }
    float top = x[0][0];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < V; ++j) top = fmaxf(top, x[u][j]);
    if (top > m) {
      s *= exp2_fast((m - top) * c);
      m = top;
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < V; ++j) s += exp2_fast((x[u][j] - m) * c);
  }
  __shared__ float red[kWaves][2];
  for (int off = 32; off > 0; off >>= 1) join(m, s, __shfl_xor(m, off), __shfl_xor(s, off), c);
  if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave][0] = m, red[threadIdx.x / kWave][1] = s;
  __syncthreads();
  m = red[0][0], s = red[0][1];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) join(m, s, red[i][0], red[i][1], c);
}

// sum (or maximum) over the workgroup, the same on every thread
template <typename F>
__device__ __forceinline__ double over_group(double v, F f) {
  __shared__ double red[kWaves];
  for (int off = 32; off > 0; off >>= 1) v = f(v, __shfl_xor(v, off));
  __syncthreads();
  if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) v = f(v, red[i]);
  return v;
}

// the row's largest score and sum are known: its entries, statistics and loss
template <typename T>
__device__ __forceinline__ void finish_row(const DistillArgs& g, int row, float m, float s) {
  const T* sc = static_cast<const T*>(g.s) + static_cast<long long>(row) * g.ld;
  const float* t = g.t + static_cast<long long>(row) * g.k;
  const int32_t* ids = g.ids + static_cast<long long>(row) * g.k;
  float* p = g.p + static_cast<long long>(row) * g.k;
  const double inv_t = 1.0 / g.temperature;
  auto sum = [](double a, double b) { return a + b; };
  auto entry = [&](int i) { return static_cast<unsigned>(ids[i]) < static_cast<unsigned>(g.n) && !(t[i] == -__builtin_inff()); };
  double top = -__builtin_inf();
  for (int i = threadIdx.x; i < g.k; i += kThreads)
    if (entry(i)) top = fmax(top, static_cast<double>(t[i]));
  top = over_group(top, [](double a, double b) { return fmax(a, b); });
  double total = 0.0, count = 0.0;
  for (int i = threadIdx.x; i < g.k; i += kThreads)
    if (entry(i)) total += static_cast<double>(expf(static_cast<float>((t[i] - top) * inv_t))), count += 1.0;
  total = over_group(total, sum);
  count = over_group(count, sum);
  const bool none = count == 0.0 || s == 0.f;
  const double log_total = none ? 0.0 : log(total), log_s = none ? 0.0 : log(static_cast<double>(s));
  double loss = 0.0;
  for (int i = threadIdx.x; i < g.k; i += kThreads) {
    double pi = 0.0;
    if (!none && entry(i)) {
      const double a = (t[i] - top) * inv_t;
      pi = static_cast<double>(expf(static_cast<float>(a))) / total;
      if (!(pi == 0.0)) loss += pi * ((a - log_total) - ((static_cast<double>(to_f32(sc[ids[i]])) - m) * inv_t - log_s));
    }
    p[i] = static_cast<float>(pi);
  }
  loss = over_group(loss, sum);
  if (threadIdx.x == 0) {
    g.stats[2 * row] = m;
    g.stats[2 * row + 1] = none ? 0.f : 1.f / s;
    g.row_loss[row] = static_cast<float>(loss);
  }
}

// one workgroup a piece of a row; a row of one piece is finished at once
template <typename T>
__global__ __launch_bounds__(kThreads) void distill_pieces_kernel(const DistillArgs g) {
  const int row = blockIdx.x / g.splits, z = blockIdx.x % g.splits;
  const int lo = z * g.piece, hi = min(g.n, lo + g.piece);
  float m, s;
  piece_max_sum<T>(g, static_cast<const T*>(g.s) + static_cast<long long>(row) * g.ld, lo, hi, kLog2e / g.temperature, m, s);
  if (g.splits == 1) {
    finish_row<T>(g, row, m, s);
  } else if (threadIdx.x == 0) {
    float* part = g.part + (static_cast<long long>(row) * g.splits + z) * 2;
    part[0] = m, part[1] = s;
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void distill_join_kernel(const DistillArgs g) {
  const int row = blockIdx.x;
  const float* part = g.part + static_cast<long long>(row) * g.splits * 2;
  float m = part[0], s = part[1];
  for (int z = 1; z < g.splits; ++z) join(m, s, part[2 * z], part[2 * z + 1], kLog2e / g.temperature);
  finish_row<T>(g, row, m, s);
}

__global__ __launch_bounds__(kThreads) void distill_sum_kernel(float* loss, const float* row_loss, int rows, double scale) {
  double v = 0.0;
  for (int i = threadIdx.x; i < rows; i += kThreads) v += row_loss[i];
  v = over_group(v, [](double a, double b) { return a + b; });
  if (threadIdx.x == 0) *loss = static_cast<float>(scale * v);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void distill_bwd_kernel(const DistillArgs g) {
  constexpr int V = 16 / sizeof(T), U = 4, STEP = kThreads * V;
  const int row = blockIdx.x / g.splits, z = blockIdx.x % g.splits;
  const int lo = z * g.piece, hi = min(g.n, lo + g.piece);
  const T* sc = static_cast<const T*>(g.s) + static_cast<long long>(row) * g.ld;
  T* grad = static_cast<T*>(g.grad) + static_cast<long long>(row) * g.n;
  const float m = g.stats[2 * row], inv = g.stats[2 * row + 1], c = kLog2e / g.temperature;
  const bool none = inv == 0.f;
  const float f = g.scale * g.temperature * *g.gout, fq = f * inv;
  for (int base = lo + threadIdx.x * V; base < hi; base += U * STEP) {
    float x[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u) load_vec<T, V>(x[u], sc + base + u * STEP, hi - (base + u * STEP));
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int j = 0; j < V; ++j) x[u][j] = none ? 0.f : fq * exp2_fast((x[u][j] - m) * c);
      store_vec<T, V>(grad + base + u * STEP, x[u], hi - (base + u * STEP));
    }
  }
  if (none) return;
  // the teacher's items of this piece: the first entry that names an item writes it whole, the others' shares in entry order
  extern __shared__ int32_t ids[];
  for (int i = threadIdx.x; i < g.k; i += kThreads) ids[i] = g.ids[static_cast<long long>(row) * g.k + i];
  __syncthreads();                                       // also orders these stores behind the loop's
  const float* p = g.p + static_cast<long long>(row) * g.k;
  for (int i = threadIdx.x; i < g.k; i += kThreads) {
    const int id = ids[i];
    if (id < lo || id >= hi) continue;
    bool first = true;
    float share = 0.f;
    for (int j = 0; j < g.k; ++j)
      if (ids[j] == id) {
        first = first && j >= i;
        share += p[j];
      }
    if (first) grad[id] = from_f32<T>(f * (inv * exp2_fast((to_f32(sc[id]) - m) * c) - share));
  }
}

// pieces of at least 8192 scores, enough for four workgroups a compute unit
inline void split_rows(int64_t rows, int64_t n, int* splits, int* piece) {
  const int64_t want = std::max<int64_t>(1, 1024 / std::max<int64_t>(1, rows));
  const int64_t s = std::max<int64_t>(1, std::min<int64_t>(want, n / 8192));
  *piece = static_cast<int>(((n + s - 1) / s + 7) & ~int64_t{7});
  *splits = static_cast<int>((n + *piece - 1) / *piece);
}

inline int check_args(const char* what, int dtype, int64_t ld, int64_t rows, int64_t n, int64_t k, float temperature) {
  if (!valid_dtype(dtype)) return fail(SG_ERR_INVALID, "%s: unknown dtype %d", what, dtype);
  if (rows < 0 || n < 1 || k < 0) return fail(SG_ERR_INVALID, "%s: bad shape", what);
  if (n >= (1ll << 30) || rows >= (1ll << 30) || k > SG_DISTILL_MAX_K)
    return fail(SG_ERR_UNSUPPORTED, "%s: at most %d teacher entries a row, fewer than 2^30 rows and items", what, SG_DISTILL_MAX_K);
  if (ld < n) return fail(SG_ERR_INVALID, "%s: rows overlap", what);
  if (!(temperature > 0.f) || !(temperature <= 3.402823466e38f)) return fail(SG_ERR_INVALID, "%s: temperature must be positive", what);
  return SG_OK;
}

}  // namespace
}  // namespace sg

using namespace sg;

SG_API size_t sg_distill_workspace_bytes(int64_t rows, int64_t n) {
  if (rows <= 0 || n <= 0) return 0;
  int splits, piece;
  split_rows(rows, n, &splits, &piece);
  return static_cast<size_t>(rows) * (1 + (splits > 1 ? 2 * splits : 0)) * sizeof(float);
}

SG_API int sg_distill_hip(float* loss, float* stats, float* p, const void* student, int64_t ld, int dtype, const float* teacher,
                          const int32_t* ids, int64_t rows, int64_t n, int64_t k, float temperature, float scale, void* workspace,
                          size_t workspace_bytes, void* stream) {
  if (int rc = check_args("distill", dtype, ld, rows, n, k, temperature)) return rc;
  if (!loss || (rows > 0 && (!stats || !student)) || (rows > 0 && k > 0 && (!p || !teacher || !ids)))
    return fail(SG_ERR_INVALID, "distill: null pointer argument");
  if (rows > 0 && (!workspace || workspace_bytes < sg_distill_workspace_bytes(rows, n)))
    return fail(SG_ERR_WORKSPACE, "distill workspace too small");
  hipStream_t st = static_cast<hipStream_t>(stream);
  float* row_loss = static_cast<float*>(workspace);
  if (rows > 0) {
    DistillArgs g{student, teacher, ids, stats, p, row_loss + rows, row_loss, nullptr, nullptr, ld, static_cast<int>(rows),
                  static_cast<int>(n), static_cast<int>(k), 0, 0, temperature, scale};
    split_rows(rows, n, &g.splits, &g.piece);
    auto run = [&](auto tag) {
      using T = decltype(tag);
      hipLaunchKernelGGL(distill_pieces_kernel<T>, dim3(static_cast<unsigned>(rows) * g.splits), dim3(kThreads), 0, st, g);
      if (g.splits > 1) hipLaunchKernelGGL(distill_join_kernel<T>, dim3(static_cast<unsigned>(rows)), dim3(kThreads), 0, st, g);
    };
    if (dtype == SG_DTYPE_F32) run(float{});
    else if (dtype == SG_DTYPE_F16) run(f16{});
    else run(bf16{});
  }
  hipLaunchKernelGGL(distill_sum_kernel, dim3(1), dim3(kThreads), 0, st, loss, row_loss, static_cast<int>(rows),
                     static_cast<double>(scale) * temperature * temperature);
  return check_launch("distill");
}

SG_API int sg_distill_bwd_hip(void* grad, const void* student, int64_t ld, int dtype, const float* stats, const float* p,
                              const int32_t* ids, int64_t rows, int64_t n, int64_t k, float temperature, float scale,
                              const float* grad_loss, void* stream) {
  if (int rc = check_args("distill_bwd", dtype, ld, rows, n, k, temperature)) return rc;
  if (rows == 0) return SG_OK;
  if (!grad || !student || !stats || !grad_loss || (k > 0 && (!p || !ids))) return fail(SG_ERR_INVALID, "distill_bwd: null pointer argument");
  DistillArgs g{student, nullptr, ids, const_cast<float*>(stats), const_cast<float*>(p), nullptr, nullptr, grad, grad_loss, ld,
                static_cast<int>(rows), static_cast<int>(n), static_cast<int>(k), 0, 0, temperature, scale};
  split_rows(rows, n, &g.splits, &g.piece);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(rows) * g.splits);
  const size_t lds = static_cast<size_t>(k) * sizeof(int32_t);
  if (dtype == SG_DTYPE_F32) hipLaunchKernelGGL(distill_bwd_kernel<float>, grid, dim3(kThreads), lds, st, g);
  else if (dtype == SG_DTYPE_F16) hipLaunchKernelGGL(distill_bwd_kernel<f16>, grid, dim3(kThreads), lds, st, g);
  else hipLaunchKernelGGL(distill_bwd_kernel<bf16>, grid, dim3(kThreads), lds, st, g);
  return check_launch("distill_bwd");
}
