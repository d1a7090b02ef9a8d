// sample.hip -- one item a row, drawn from the row's scores with temperature, top-k, top-p and min-p, from given random numbers.
//
//   w_i = exp((l_i - max l) / T);  order: larger score first, the lower index first among equals;  the kept items are the
//   shortest prefix of the order that top-k (k items), top-p (the first items that hold the share p of the top-k items' weight)
//   and min-p (w_i >= m) leave, and at least the first item.
//   drawn: the first item, by index, at which the kept weight summed up to it exceeds u times the kept weight
//
// Which item is drawn is a decision at the border of two sums over the catalogue, so a weight is a whole number: w * 2^s, s = min(51, 62 - log2 N), from a 64-bit polynomial.  Sums of whole numbers are exact in any order: the
// result does not depend on how the row is spread over threads, on the order of the atomic additions, or on the run.  Weights
// below 2^-(s+1) of the largest are 0 and cannot be drawn.
//
// The order is never formed.  A histogram of (max l - l) / T, count and weight, shows in which bin a limit falls; the limit's
// own element is then found among that bin's elements, digit by digit of the score's ordered bits, and among equal scores by
// index.  -inf and NaN are scores of items that are never drawn; a row without any other draws -1.
#include "rows_shared.hpp"

#include <algorithm>

namespace sg {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / kWave;
constexpr int kBins = 2048;        // of the histogram, and of an 11-bit digit
constexpr int kChunks = 4096;      // partial weights by index

typedef unsigned long long u64;

struct SampleArgs {
  int32_t* ids;
  float* prob;
  const void* l;
  const float* u;
  const float* temperature;        // per row, or null: the scalars below
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  double t0, p0, m0;
  long long ld, k0;
  int rows, n, bits;               // bits: s above
};

struct Row {                       // a row's settings, the same on every thread
  double c;                        // log2(e) / T
  double p, m;                     // m as a scaled weight
  long long k;                     // 0: none
  bool by_p;
};

__device__ __forceinline__ Row row_settings(const SampleArgs& g, int row) {
  Row r;
  const double t = g.temperature ? g.temperature[row] : g.t0;
  r.k = g.top_k ? g.top_k[row] : g.k0;
  r.p = g.top_p ? g.top_p[row] : g.p0;
  double m = g.min_p ? g.min_p[row] : g.m0;
  if (r.k < 0 || r.k >= g.n) r.k = 0;
  r.by_p = !(r.p >= 1.0);
  if (!(t > 0.0) || !(r.p > 0.0) || !(m <= 1.0)) r.k = 1;      // nothing but the first item
  if (r.k == 1) r.by_p = false, m = 0.0;
  r.c = t > 0.0 ? 1.4426950408889634074 / t : 1.0;
  r.m = m > 0.0 ? ldexp(m, g.bits) : 0.0;
  return r;
}

// scores as whole numbers in the scores' order (both zeros are the same score; NaN is dealt with before)
__device__ __forceinline__ unsigned ordered(float l) {
  const unsigned b = __float_as_uint(l + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// d = (max - l) log2(e) / T, >= 0; NaN and -inf: beyond every weight
__device__ __forceinline__ double below_top(float l, float top, double c) {
  if (l == top) return 0.0;
  const double d = (static_cast<double>(top) - static_cast<double>(l)) * c;
  return d >= 0.0 ? d : __builtin_inf();
}

// 2^(bits - d), rounded to a whole number by the caller (Taylor series of 2^f, |f| <= 1/2: the first term left out is 6e-15)
__device__ __forceinline__ double scaled_weight(double d, int bits) {
  if (!(d < bits + 1.0)) return 0.0;
  const double n = rint(d), f = n - d;
  double y = 4.44553827187081e-10;                       // (ln 2)^11 / 11!
  y = fma(y, f, 7.054911620801121e-09);
  y = fma(y, f, 1.0178086009239696e-07);
  y = fma(y, f, 1.3215486790144305e-06);
  y = fma(y, f, 1.5252733804059838e-05);
  y = fma(y, f, 0.00015403530393381606);
  y = fma(y, f, 0.0013333558146428441);
  y = fma(y, f, 0.009618129107628477);
  y = fma(y, f, 0.055504108664821576);
  y = fma(y, f, 0.2402265069591007);
  y = fma(y, f, 0.6931471805599453);
  y = fma(y, f, 1.0);
  return ldexp(y, bits - static_cast<int>(n));
}
__device__ __forceinline__ u64 whole(double w) {              // w < 2^52
  return static_cast<u64>(__double_as_longlong(w + 4503599627370496.0)) - 0x4330000000000000ull;
}

__device__ __forceinline__ int bin_of(double d, double scale) { return static_cast<int>(fmin(d * scale, kBins - 1.0)); }

// where the kept items of one limit end: scores above `key`, and those equal to it up to index `last`
struct Limit {
  unsigned key;
  int last;
};

__device__ __forceinline__ bool inside(const Limit& lim, unsigned key, int i) { return key > lim.key || (key == lim.key && i <= lim.last); }

struct Shared {
  u64 mass[kBins];
  unsigned count[kBins];
  u64 wave_mass[kWaves];
  unsigned wave_count[kWaves];
  u64 before_mass;
  unsigned before_count;
  int found;
};

__device__ __forceinline__ u64 wave_sum(u64 v) {
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
  return v;
}

// sums of all lanes below this one
__device__ __forceinline__ u64 wave_before(u64 v) {
  const int lane = threadIdx.x % kWave;
  u64 s = v;
  for (int off = 1; off < kWave; off <<= 1) {
    const u64 o = __shfl_up(s, off);
    if (lane >= off) s += o;
  }
  return s - v;
}

// The bin of sh.count / sh.mass, counted from bin 0 on, in which the sum of counts reaches `need` (by_mass: the sum of weights
// reaches `need`): its number, or kBins, with the sums of the bins before it.  Two bins a thread.
__device__ __forceinline__ int find_bin(Shared& sh, bool by_mass, u64 need, unsigned& before_count, u64& before_mass) {
  const int t = threadIdx.x, wave = t / kWave, lane = t % kWave;
  if (t == 0) sh.found = kBins;
  const u64 m0 = sh.mass[2 * t], m1 = sh.mass[2 * t + 1];
  const unsigned c0 = sh.count[2 * t], c1 = sh.count[2 * t + 1];
  u64 mb = wave_before(m0 + m1), cb = wave_before(static_cast<u64>(c0) + c1);
  if (lane == kWave - 1) sh.wave_mass[wave] = mb + m0 + m1, sh.wave_count[wave] = static_cast<unsigned>(cb) + c0 + c1;
  __syncthreads();
  for (int i = 0; i < wave; ++i) mb += sh.wave_mass[i], cb += sh.wave_count[i];
  const u64 a = by_mass ? mb : cb, v0 = by_mass ? m0 : c0, v1 = by_mass ? m1 : c1;
  if (a < need && need <= a + v0) sh.found = 2 * t, sh.before_count = static_cast<unsigned>(cb), sh.before_mass = mb;
  else if (a + v0 < need && need <= a + v0 + v1) sh.found = 2 * t + 1, sh.before_count = static_cast<unsigned>(cb) + c0, sh.before_mass = mb + m0;
  __syncthreads();
  before_count = sh.before_count, before_mass = sh.before_mass;
  const int found = sh.found;
  __syncthreads();
  return found;
}

__device__ __forceinline__ void clear_bins(Shared& sh) {
  for (int i = threadIdx.x; i < kBins; i += kThreads) sh.mass[i] = 0, sh.count[i] = 0;
  __syncthreads();
}

// f(score, index) for every element of the row, any order
template <typename T, typename F>
__device__ __forceinline__ void each(const T* row, int n, F f) {
  constexpr int V = 16 / sizeof(T);
  for (int base = threadIdx.x * V; base < n; base += kThreads * V) {
    float x[V];
    load_vec<T, V>(x, row + base, n - base);
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (base + j < n) f(x[j], base + j);
  }
}

// The limit inside bin `bin`, of which the order's items before it number `count` and weigh `mass`: by count, the item with
// which the count reaches `need`; by mass, the last item before which the weight is below `need`.  On return count and mass
// include the limit's own item.
template <typename T>
__device__ __forceinline__ Limit find_limit(Shared& sh, const T* row, const SampleArgs& g, float top, double c, double bin_scale, int bin,
                                            bool by_mass, u64 need, unsigned& count, u64& mass) {
  unsigned key = 0, here = 0;
  u64 weight = 0;
#pragma unroll
  for (int level = 0; level < 3; ++level) {              // digits of 11, 11 and 10 bits, the largest digit first
    const int shift = level == 0 ? 21 : level == 1 ? 10 : 0, width = level == 2 ? 10 : 11;
    clear_bins(sh);
    each(row, g.n, [&](float l, int) {
      const double d = below_top(l, top, c);
      const unsigned k = ordered(l);
      if (bin_of(d, bin_scale) != bin || d == __builtin_inf() || (level > 0 && (k >> (shift + width)) != (key >> (shift + width)))) return;
      const unsigned digit = ((1u << width) - 1) - ((k >> shift) & ((1u << width) - 1));
      atomicAdd(&sh.count[digit], 1u);
      atomicAdd(&sh.mass[digit], whole(scaled_weight(d, g.bits)));
    });
    __syncthreads();
    unsigned bc;
    u64 bm;
    const int digit = find_bin(sh, by_mass, need - (by_mass ? mass : count), bc, bm);
    here = sh.count[digit], weight = sh.mass[digit];
    __syncthreads();
    key |= (((1u << width) - 1) - digit) << shift;
    count += bc, mass += bm;
  }
  // `here` items share the score: equal weights, taken by index
  const u64 one = weight / here;
  const unsigned take = by_mass ? static_cast<unsigned>(one ? (need - mass + one - 1) / one : here) : static_cast<unsigned>(need - count);
  Limit lim{key, 0x7fffffff};
  count += take, mass += one * take;
  if (take >= here) return lim;
  unsigned left = take, index = 0;
#pragma unroll
  for (int level = 0; level < 3; ++level) {
    const int shift = level == 0 ? 20 : level == 1 ? 9 : 0, width = level == 2 ? 9 : 11;
    clear_bins(sh);
    each(row, g.n, [&](float l, int i) {
      if (l != l || ordered(l) != key || (level > 0 && (static_cast<unsigned>(i) >> (shift + width)) != (index >> (shift + width)))) return;
      atomicAdd(&sh.count[(static_cast<unsigned>(i) >> shift) & ((1u << width) - 1)], 1u);
    });
    __syncthreads();
    unsigned bc;
    u64 bm;
    const int digit = find_bin(sh, false, left, bc, bm);
    left -= bc;
    index |= static_cast<unsigned>(digit) << shift;
  }
  lim.last = static_cast<int>(index);
  return lim;
}

// one workgroup a row
template <typename T>
__global__ __launch_bounds__(kThreads) void sample_kernel(const SampleArgs g) {
  __shared__ Shared sh;
  __shared__ u64 chunk[kChunks];
  __shared__ float red[kWaves];
  constexpr int V = 16 / sizeof(T);
  const int row = blockIdx.x, t = threadIdx.x, wave = t / kWave, lane = t % kWave;
  const T* l = static_cast<const T*>(g.l) + row * g.ld;
  const Row r = row_settings(g, row);

  float top = -__builtin_inff();
  each(l, g.n, [&](float x, int) { top = fmaxf(top, x); });
  for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off));
  if (lane == 0) red[wave] = top;
  __syncthreads();
  top = red[0];
  for (int i = 1; i < kWaves; ++i) top = fmaxf(top, red[i]);
  if (top == -__builtin_inff()) {                        // nothing to draw from (also N = 0)
    if (t == 0) g.ids[row] = -1, g.prob[row] = 0.f;
    return;
  }

  // limits.  The last bin holds items of weight 0 only: a limit there keeps every weight.
  Limit by_k{0, 0x7fffffff}, by_p{0, 0x7fffffff};
  if (r.k > 0 || r.by_p) {
    const double bin_scale = (kBins - 1.0) / (g.bits + 1.0);
    auto histogram = [&]() {
      clear_bins(sh);
      each(l, g.n, [&](float x, int) {
        const double d = below_top(x, top, r.c);
        if (d == __builtin_inf()) return;
        const int b = bin_of(d, bin_scale);
        atomicAdd(&sh.count[b], 1u);
        const u64 w = whole(scaled_weight(d, g.bits));
        if (w) atomicAdd(&sh.mass[b], w);
      });
      __syncthreads();
    };
    histogram();
    u64 total = 0;
    for (int i = lane; i < kBins; i += kWave) total += sh.mass[i];
    total = wave_sum(total);
    __syncthreads();
    unsigned count = 0;
    u64 mass = 0;
    if (r.k > 0) {
      const int b = find_bin(sh, false, static_cast<u64>(r.k), count, mass);
      if (b < kBins - 1) {
        by_k = find_limit(sh, l, g, top, r.c, bin_scale, b, false, static_cast<u64>(r.k), count, mass);
        total = mass;
        if (r.by_p) histogram();
      }
    }
    if (r.by_p) {
      const u64 need = max(u64{1}, static_cast<u64>(ceil(r.p * static_cast<double>(total))));
      const int b = find_bin(sh, true, need, count, mass);
      if (b < kBins - 1) by_p = find_limit(sh, l, g, top, r.c, bin_scale, b, true, need, count, mass);
    }
  }

  // kept weight by index: one wave a chunk of 64 V * 2^j items
  auto weight = [&](float x, int i) -> u64 {
    const double d = below_top(x, top, r.c);
    if (!(d < g.bits + 1.0)) return 0;
    const unsigned key = ordered(x);
    if (!inside(by_k, key, i) || !inside(by_p, key, i)) return 0;
    const double w = scaled_weight(d, g.bits);
    return w >= r.m ? whole(w) : 0;
  };
  int span = kWave * V;
  while ((g.n + span - 1) / span > kChunks) span *= 2;
  const int chunks = (g.n + span - 1) / span;
  for (int ch = wave; ch < chunks; ch += kWaves) {
    u64 sum = 0;
    const int end = min(g.n, (ch + 1) * span);
    for (int base = ch * span + lane * V; base < end; base += kWave * V) {
      float x[V];
      load_vec<T, V>(x, l + base, end - base);
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (base + j < end) sum += weight(x[j], base + j);
    }
    sum = wave_sum(sum);
    if (lane == 0) chunk[ch] = sum;
  }
  __syncthreads();
  if (wave != 0) return;
  // the chunk, then the item, at which the sum passes the drawn share
  const int per = (chunks + kWave - 1) / kWave, c0 = min(chunks, lane * per), c1 = min(chunks, c0 + per);
  u64 mine = 0;
  for (int i = c0; i < c1; ++i) mine += chunk[i];
  const u64 total = wave_sum(mine);
  const double u = g.u[row];
  u64 goal = u > 0.0 ? static_cast<u64>(fmin(u, 1.0) * static_cast<double>(total)) : 0;
  goal = min(goal, total - 1);
  u64 before = wave_before(mine);
  int at = -1;
  if (before <= goal && goal < before + mine) {
    for (at = c0; before + chunk[at] <= goal; ++at) before += chunk[at];
  }
  const u64 has = __ballot(at >= 0);
  const int owner = __ffsll(has) - 1;
  at = __shfl(at, owner);
  before = __shfl(before, owner);
  const int end = min(g.n, (at + 1) * span);
  for (int base0 = at * span; base0 < end; base0 += kWave * V) {
    const int base = base0 + lane * V;
    float x[V];
    load_vec<T, V>(x, l + base, end - base);
    u64 w[V], sum = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) w[j] = base + j < end ? weight(x[j], base + j) : 0, sum += w[j];
    u64 b = before + wave_before(sum);
    const bool hit = b <= goal && goal < b + sum;
    if (hit) {
      bool done = false;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (!done && goal < b + w[j]) {
          g.ids[row] = base + j;
          g.prob[row] = static_cast<float>(static_cast<double>(w[j]) / static_cast<double>(total));
          done = true;
        }
        b += w[j];
      }
    }
    if (__ballot(hit)) return;
    before += wave_sum(sum);
  }
}

}  // namespace
}  // namespace sg

using namespace sg;

SG_API size_t sg_sample_rows_workspace_bytes(int64_t rows, int64_t n) {
  (void)rows, (void)n;
  return 0;
}

SG_API int sg_sample_rows_hip(int32_t* ids, float* prob, const void* logits, int64_t ld, int dtype, const float* u, int64_t rows,
                              int64_t n, double temperature, int64_t top_k, double top_p, double min_p, const float* temperature_rows,
                              const int32_t* top_k_rows, const float* top_p_rows, const float* min_p_rows, void* workspace,
                              size_t workspace_bytes, void* stream) {
  (void)workspace, (void)workspace_bytes;
  if (!valid_dtype(dtype)) return fail(SG_ERR_INVALID, "sample_rows: unknown dtype %d", dtype);
  if (rows < 0 || n < 0) return fail(SG_ERR_INVALID, "sample_rows: negative size");
  if (rows >= (1ll << 31) || n >= SG_SAMPLE_MAX_ITEMS) return fail(SG_ERR_UNSUPPORTED, "sample_rows: fewer than %d items", SG_SAMPLE_MAX_ITEMS);
  if (rows == 0) return SG_OK;
  if (!ids || !prob || !u || (n > 0 && !logits)) return fail(SG_ERR_INVALID, "sample_rows: null pointer argument");
  if (ld < n) return fail(SG_ERR_INVALID, "sample_rows: rows overlap");
  if (!(temperature >= 0.0) || !(top_p >= 0.0) || !(min_p >= 0.0) || top_k < 0)
    return fail(SG_ERR_INVALID, "sample_rows: temperature, top_k, top_p and min_p must not be negative");
  int log_n = 0;
  while ((1ll << log_n) < n) ++log_n;
  SampleArgs g{ids, prob, logits, u, temperature_rows, top_k_rows, top_p_rows, min_p_rows, temperature, top_p, min_p, ld, top_k,
               static_cast<int>(rows), static_cast<int>(n), std::min(51, 62 - log_n)};
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(rows));
  if (dtype == SG_DTYPE_F32) hipLaunchKernelGGL(sample_kernel<float>, grid, dim3(kThreads), 0, st, g);
  else if (dtype == SG_DTYPE_F16) hipLaunchKernelGGL(sample_kernel<f16>, grid, dim3(kThreads), 0, st, g);
  else hipLaunchKernelGGL(sample_kernel<bf16>, grid, dim3(kThreads), 0, st, g);
  return check_launch("sample_rows");
}
