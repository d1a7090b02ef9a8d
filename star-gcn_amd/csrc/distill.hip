// distill.hip -- a student's scores fitted to a teacher's top scores: forward and backward.
//
//   q = softmax(s / T) over a row's N items,  p = softmax(t / T) over the teacher's K entries of the row
//   loss = scale * T^2 * sum_rows sum_k p_k (log p_k - log q_{id_k}),        d loss / d s_j = scale * T * (q_j - sum_{id_k = j} p_k)
//
// An entry whose id lies outside [0, N) or whose score is -inf is no entry.  A row without an entry, or whose student scores
// are all -inf, has nothing to fit: it adds no loss and its gradient is zero.  An item that is named twice takes both shares.
//
// 10000 rows of 10677 bf16 scores: forward 49 us (4.4 TB/s; the chain of one row's entries shows), backward 85 us (5.0 TB/s, a
// copy of that size reaches 5.3); 64 rows of 1,000,000 fp32: 38 and 87 us (6.8 and 5.9 TB/s).
//
// Bound by memory: the forward reads the scores once (running maximum and sum, one exp an element), the backward reads them
// again and writes the gradient; the K entries of a row are noise next to its N scores.  Long rows of small batches are split
// over workgroups and joined.  Exponents are taken of differences from a score near the row's largest, so T scales exact differences;
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
  float* stats;            // (rows, 2): a score near the largest, 1 / sum of exp over it (0: the row has nothing to fit)
  float* p;                // (rows, K)
  float* part;             // (rows, splits, 2): the same of a piece, with the sum itself
  float* row_loss;         // (rows): in the scores' unit, T sum p (log p - log q), which is about as large as the scores' differences
  void* grad;
  const float* gout;
  long long ld;
  int rows, n, k, splits, piece;
  float temperature, scale;
  // Store the gradient past the caches: from 128 MB on scores and gradient together exceed the Infinity Cache, so a reader that
  // starts at its beginning would not find it there, and writing it back delays whatever runs next.  64 x 1,000,000 fp32:
  // backward 87 us instead of 91, the step 142 instead of 178; 10000 x 10677 bf16: 86 and 91, 145 and 164.
  int past;
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

// The elements [lo, hi) of a row: one(index) for the fewer than 2 V at its ends, at most one a thread, then vectors from aligned
// addresses on (rows of odd length start anywhere): many(vectors, first index) for U of them at a time while a thread has as
// many left, else for one.  Nothing of a load hangs on a condition of its own, so U loads are under way at once.
template <int U, typename T, typename One, typename Many>
__device__ __forceinline__ void walk(const T* row, int lo, int hi, One one, Many many) {
  constexpr int V = 16 / sizeof(T);
  const int skew = static_cast<int>((reinterpret_cast<uintptr_t>(row + lo) / sizeof(T)) % V);
  const int b0 = min(hi, lo + (V - skew) % V), vecs = (hi - b0) / V, b1 = b0 + vecs * V, t = threadIdx.x;
  const int head = b0 - lo;
  if (t < head) one(lo + t);
  else if (t < head + hi - b1) one(b1 + t - head);
  int v = t;
  for (; v + (U - 1) * kThreads < vecs; v += U * kThreads) {
    pack<T, V> a[U];
#pragma unroll
    for (int u = 0; u < U; ++u) a[u] = load_pack<T, V>(row + b0 + (v + u * kThreads) * V);
#pragma unroll
    for (int u = 0; u < U; ++u) many(a[u], b0 + (v + u * kThreads) * V);
  }
  for (; v < vecs; v += kThreads) many(load_pack<T, V>(row + b0 + v * V), b0 + v * V);
}

// The wave's running maximum and sum over the piece's elements of its lanes.  A thread of a long row adds hundreds of vectors, and
// equal terms are rounded the same way each time: in 32 bits 1.6e-5 of the sum for 1,000,000 scores of 0 and 1.  So a vector is
// summed pairwise and the vectors in 64 bits.  The maximum is followed in steps of at least a factor of 16 of the terms (a term is
// then at most 16, and what the sum was scaled by before is forgotten as fast as its rounding adds up): followed at once, scores
// that rise a little with every vector cost 1e-5 of the sum.
template <typename T>
__device__ __forceinline__ void piece_max_sum(const T* row, int lo, int hi, float c, float& m, float& s) {
  constexpr int V = 16 / sizeof(T);
  const float step = 4.f / c;
  double sum = 0.0;
  m = kLowest;
  walk<4>(row, lo, hi,
           [&](int i) {
             const float x = to_f32(row[i]);
             m = fmaxf(m, x);                            // the thread's first element; NaN and -inf leave the lowest value
             sum = exp2_fast((x - m) * c);
           },
           [&](const pack<T, V>& a, int) {
             float x[V], top = m;
#pragma unroll
             for (int j = 0; j < V; ++j) x[j] = to_f32(a.v[j]), top = fmaxf(top, x[j]);
             if (top > m + step) {
               sum *= exp2_fast((m - top) * c);
               m = top;
             }
#pragma unroll
             for (int j = 0; j < V; ++j) x[j] = exp2_fast((x[j] - m) * c);
#pragma unroll
             for (int half = V / 2; half > 0; half /= 2)
#pragma unroll
               for (int j = 0; j < half; ++j) x[j] += x[j + half];
             sum += x[0];
           });
  const float top = wave_max(m);
  s = static_cast<float>(wave_sum(sum * exp2_fast((m - top) * c)));
  m = top;
}

// A row's teacher entries: a thread takes up to four, their scores and items while the row is still being read, the student's
// scores of the items after it; one wave uses them at the end.
constexpr int kTake = SG_DISTILL_MAX_K / kThreads;
struct Taken {
  float t[kTake], x[kTake];        // -inf in t: no entry
  int id[kTake];
};
struct Entries {
  float t[SG_DISTILL_MAX_K], x[SG_DISTILL_MAX_K];
  float part[kWaves][3];           // a wave's largest score, its sum, its largest teacher score
};

__device__ __forceinline__ void take_entries(const DistillArgs& g, int row, Taken& e) {
#pragma unroll
  for (int j = 0; j < kTake; ++j) {
    const int i = j * kThreads + threadIdx.x;
    if (i < g.k) e.t[j] = g.t[static_cast<long long>(row) * g.k + i], e.id[j] = g.ids[static_cast<long long>(row) * g.k + i];
  }
}

template <typename T>
__device__ __forceinline__ void put_entries(const DistillArgs& g, int row, Taken& e, Entries& lds) {
  const T* sc = static_cast<const T*>(g.s) + static_cast<long long>(row) * g.ld;
#pragma unroll
  for (int j = 0; j < kTake; ++j) {
    const int i = j * kThreads + threadIdx.x;
    if (i < g.k) {
      const bool entry = static_cast<unsigned>(e.id[j]) < static_cast<unsigned>(g.n);
      e.x[j] = entry ? to_f32(sc[e.id[j]]) : 0.f;
      if (!entry) e.t[j] = -__builtin_inff();
    }
  }
  float top = -__builtin_inff();
#pragma unroll
  for (int j = 0; j < kTake; ++j) {
    const int i = j * kThreads + threadIdx.x;
    if (i < g.k) {
      lds.t[i] = e.t[j], lds.x[i] = e.x[j];
      top = fmaxf(top, e.t[j] != e.t[j] ? __builtin_inff() : e.t[j]);        // a maximum drops NaN, and NaN is to come out
    }
  }
  top = wave_max(top);
  if (threadIdx.x % kWave == 0) lds.part[threadIdx.x / kWave][2] = top;
}

// one wave: the row's sum s over exp((score - m) / T) is known -> its shares, statistics and loss
__device__ __forceinline__ void finish_row(const DistillArgs& g, int row, float m, float s, const Entries& e) {
  const int lane = threadIdx.x;
  const double inv_t = 1.0 / g.temperature;
  float top = e.part[0][2];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) top = fmaxf(top, e.part[i][2]);
  const bool none = top == -__builtin_inff() || s == 0.f;
  auto below = [&](int i) { return (e.t[i] - static_cast<double>(top)) * inv_t; };
  double total = 0.0;
  for (int i = lane; i < g.k; i += kWave)
    if (!none && e.t[i] != -__builtin_inff()) total += static_cast<double>(expf(static_cast<float>(below(i))));
  total = wave_sum(total);
  // log p - log q = (t - top) / T - (x - m) / T + log(s / total)
  const double log_ratio = none ? 0.0 : log(static_cast<double>(s) / total);
  float* p = g.p + static_cast<long long>(row) * g.k;
  double loss = 0.0;
  for (int i = lane; i < g.k; i += kWave) {
    double pi = 0.0;
    if (!none && e.t[i] != -__builtin_inff()) {
      const double a = below(i);
      pi = static_cast<double>(expf(static_cast<float>(a))) / total;
      if (!(pi == 0.0)) loss += pi * ((a - (static_cast<double>(e.x[i]) - m) * inv_t) + log_ratio);
    }
    p[i] = static_cast<float>(pi);
  }
  loss = wave_sum(loss);
  if (lane == 0) {
    g.stats[2 * row] = m;
    g.stats[2 * row + 1] = none ? 0.f : 1.f / s;
    g.row_loss[row] = static_cast<float>(loss * g.temperature);
  }
}

// one workgroup a piece of a row; a row of one piece is finished at once
template <typename T>
__global__ __launch_bounds__(kThreads) void distill_pieces_kernel(const DistillArgs g) {
  __shared__ Entries e;
  const int row = blockIdx.x / g.splits, z = blockIdx.x % g.splits, wave = threadIdx.x / kWave;
  const int lo = z * g.piece, hi = min(g.n, lo + g.piece);
  const float c = kLog2e / g.temperature;
  Taken mine;
  if (g.splits == 1) take_entries(g, row, mine);
  float m, s;
  piece_max_sum<T>(static_cast<const T*>(g.s) + static_cast<long long>(row) * g.ld, lo, hi, c, m, s);
  if (threadIdx.x % kWave == 0) e.part[wave][0] = m, e.part[wave][1] = s;
  if (g.splits == 1) put_entries<T>(g, row, mine, e);
  __syncthreads();
  if (wave != 0) return;
  m = e.part[0][0], s = e.part[0][1];
#pragma unroll
  for (int i = 1; i < kWaves; ++i) join(m, s, e.part[i][0], e.part[i][1], c);
  if (g.splits == 1) {
    finish_row(g, row, m, s, e);
  } else if (threadIdx.x == 0) {
    float* part = g.part + (static_cast<long long>(row) * g.splits + z) * 2;
    part[0] = m, part[1] = s;
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void distill_join_kernel(const DistillArgs g) {
  __shared__ Entries e;
  const int row = blockIdx.x;
  const float c = kLog2e / g.temperature;
  Taken mine;
  take_entries(g, row, mine);
  put_entries<T>(g, row, mine, e);
  __syncthreads();
  if (threadIdx.x >= kWave) return;
  const float* part = g.part + static_cast<long long>(row) * g.splits * 2;
  float m = kLowest, s = 0.f;
  for (int z = threadIdx.x; z < g.splits; z += kWave) join(m, s, part[2 * z], part[2 * z + 1], c);
  const float top = wave_max(m);
  s = wave_sum(s * exp2_fast((m - top) * c));
  finish_row(g, row, top, s, e);
}

constexpr int kSumThreads = 1024;
__global__ __launch_bounds__(kSumThreads) void distill_sum_kernel(float* loss, const float* row_loss, int rows, double scale) {
  __shared__ double red[kSumThreads / kWave];
  double v = 0.0;
#pragma unroll 8
  for (int i = threadIdx.x; i < rows; i += kSumThreads) v += row_loss[i];
  v = wave_sum(v);
  if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = v;
  __syncthreads();
  v = 0.0;
#pragma unroll
  for (int i = 0; i < kSumThreads / kWave; ++i) v += red[i];
  if (threadIdx.x == 0) *loss = static_cast<float>(scale * v);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void distill_bwd_kernel(const DistillArgs g) {
  constexpr int V = 16 / sizeof(T);
  __shared__ int32_t ids[SG_DISTILL_MAX_K];
  __shared__ float share[SG_DISTILL_MAX_K];
  const int row = blockIdx.x / g.splits, z = blockIdx.x % g.splits;
  const int lo = z * g.piece, hi = min(g.n, lo + g.piece);
  const T* sc = static_cast<const T*>(g.s) + static_cast<long long>(row) * g.ld;
  T* grad = static_cast<T*>(g.grad) + static_cast<long long>(row) * g.n;
  int my_id[kTake];
  float my_p[kTake];
#pragma unroll
  for (int j = 0; j < kTake; ++j) {
    const int i = j * kThreads + threadIdx.x;
    if (i < g.k) my_id[j] = g.ids[static_cast<long long>(row) * g.k + i], my_p[j] = g.p[static_cast<long long>(row) * g.k + i];
  }
  const float m = g.stats[2 * row], inv = g.stats[2 * row + 1], c = kLog2e / g.temperature;
  const bool none = inv == 0.f;
  const float f = g.scale * g.temperature * *g.gout, fq = f * inv;
  const bool past = g.past && ((reinterpret_cast<uintptr_t>(grad) ^ reinterpret_cast<uintptr_t>(sc)) & 15) == 0;
  auto slope = [&](T x) { return none ? 0.f : fq * exp2_fast((to_f32(x) - m) * c); };
  walk<4>(sc, lo, hi, [&](int i) { grad[i] = from_f32<T>(slope(sc[i])); },
           [&](pack<T, V> a, int at) {
#pragma unroll
             for (int j = 0; j < V; ++j) a.v[j] = from_f32<T>(slope(a.v[j]));
             if (past) __builtin_nontemporal_store(__builtin_bit_cast(vec16, a), reinterpret_cast<vec16*>(grad + at));
             else store_pack<T, V>(grad + at, a);
           });
  if (none) return;
  // the teacher's items of this piece: the first entry that names an item writes it whole, the others' shares in entry order
#pragma unroll
  for (int j = 0; j < kTake; ++j) {
    const int i = j * kThreads + threadIdx.x;
    if (i < g.k) ids[i] = my_id[j], share[i] = my_p[j];
  }
  __syncthreads();                                       // also orders these stores behind the loop's
#pragma unroll
  for (int j = 0; j < kTake; ++j) {
    const int i = j * kThreads + threadIdx.x;
    if (i >= g.k || my_id[j] < lo || my_id[j] >= hi) continue;
    const int id = my_id[j];
    const float x = to_f32(sc[id]);
    bool first = true;
    float sum = 0.f;
    for (int o = 0; o < g.k; ++o)
      if (ids[o] == id) {
        first = first && o >= i;
        sum += share[o];
      }
    if (first) grad[id] = from_f32<T>(f * (inv * exp2_fast((x - m) * c) - sum));
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
  if (n >= (1ll << 30) || rows >= (1ll << 24) || k > SG_DISTILL_MAX_K)      // 2^32 threads a launch
    return fail(SG_ERR_UNSUPPORTED, "%s: at most %d teacher entries a row, fewer than 2^24 rows and 2^30 items", what, SG_DISTILL_MAX_K);
  if (ld < n) return fail(SG_ERR_INVALID, "%s: rows overlap", what);
  // beyond, its square leaves 32 bits: the loss's factor, and at the lower end the exponents' too
  if (!(temperature >= 0x1p-63f) || !(temperature <= 0x1p63f)) return fail(SG_ERR_INVALID, "%s: temperature must lie between 2^-63 and 2^63", what);
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
                  static_cast<int>(n), static_cast<int>(k), 0, 0, temperature, scale, 0};
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
  hipLaunchKernelGGL(distill_sum_kernel, dim3(1), dim3(kSumThreads), 0, st, loss, row_loss, static_cast<int>(rows),
                     static_cast<double>(scale) * temperature);
  return check_launch("distill");
}

SG_API int sg_distill_bwd_hip(void* grad, const void* student, int64_t ld, int dtype, const float* stats, const float* p,
                              const int32_t* ids, int64_t rows, int64_t n, int64_t k, float temperature, float scale,
                              const float* grad_loss, void* stream) {
  if (int rc = check_args("distill_bwd", dtype, ld, rows, n, k, temperature)) return rc;
  if (rows == 0) return SG_OK;
  if (!grad || !student || !stats || !grad_loss || (k > 0 && (!p || !ids))) return fail(SG_ERR_INVALID, "distill_bwd: null pointer argument");
  DistillArgs g{student, nullptr, ids, const_cast<float*>(stats), const_cast<float*>(p), nullptr, nullptr, grad, grad_loss, ld,
                static_cast<int>(rows), static_cast<int>(n), static_cast<int>(k), 0, 0, temperature, scale,
                rows * n * (dtype == SG_DTYPE_F32 ? 4 : 2) >= (int64_t{128} << 20)};
  split_rows(rows, n, &g.splits, &g.piece);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(rows) * g.splits);
  if (dtype == SG_DTYPE_F32) hipLaunchKernelGGL(distill_bwd_kernel<float>, grid, dim3(kThreads), 0, st, g);
  else if (dtype == SG_DTYPE_F16) hipLaunchKernelGGL(distill_bwd_kernel<f16>, grid, dim3(kThreads), 0, st, g);
  else hipLaunchKernelGGL(distill_bwd_kernel<bf16>, grid, dim3(kThreads), 0, st, g);
  return check_launch("distill_bwd");
}
