// sample.hip -- one item a row, drawn from the row's scores with temperature, top-k, top-p and min-p, from given random numbers.
//
//   w_i = exp((l_i - max l) / T);  order: larger score first, the lower index first among equals;  the kept items are the
//   shortest prefix of the order that top-k (k items), top-p (the first items that hold the share p of the top-k items' weight)
//   and min-p (w_i >= m) leave, and at least the first item.
//   drawn: the first item, by index, at which the kept weight summed up to it exceeds u times the kept weight
//
// Which item is drawn is a decision at the border of two sums over the catalogue, so a weight is a whole number: w * 2^s, from a
// 64-bit polynomial.  Sums of whole numbers are exact in any order: the result does not depend on how the row is spread over
// threads and workgroups, on the order of the atomic additions, or on the run.  Weights below 2^-(s+1) of the largest are 0 and
// cannot be drawn, so N items can gain or lose N 2^-(s+1) of the largest weight together.  Rows of up to 2^20 items are summed
// in 64 bits, s = min(51, 63 - log2 N): at most 2^-24, half a step of an fp32 share.  Longer rows keep s = 51 and are summed in
// 128 bits: 2^-24 up to 2^28 items, 2^-22 at 2^30 (4 x 10,000,000 fp32, no limits: 106 us; in 64 bits 96, which lost 2e-5).
//
// The order is never formed.  A histogram of (max l - l) / T, count and weight, shows in which bin a limit falls.  The limit's
// own element is found among that bin's elements, by rank where they are few, else by subdividing the range of their place in
// the order (score and index in 64 bits, all different) until they are.  -inf and NaN are scores of items that are never drawn;
// a row without any other draws -1.
//
// Rows of up to 16384 items: one workgroup a row, the row in LDS.  Longer rows are cut into pieces, five launches: maximum;
// histogram; the limits' bins; weight by index of what is surely kept, and the list of the limits' candidates; limits and draw.
// A list of more than 8192 candidates (many equal scores, or a spread that is small beside T) is replaced by passes of one workgroup
// over the row: 64 rows of 1,000,000 scores of deviation 0.5 T then take 1.6 ms.  64 rows of 1,000,000 fp32 scores,
// top-p: 37 us for the maximum (6.9 TB/s), 61 for the histogram (bound by the 64-bit arithmetic: 24 operations an item), 10, 52 and
// 12 for the rest.
#include "rows_shared.hpp"

#include <algorithm>
#include <type_traits>

namespace sg {
namespace {

// 512 threads and up to 128 registers: two workgroups a compute unit (512 rows of 10677: 28 us; of 1024 threads, one at a time: 43)
constexpr int kThreads = 512, kWaves = kThreads / kWave;
constexpr int kBins = 2048;        // of the histogram and of a subdivision
constexpr int kPer = kBins / kThreads;
constexpr int kFew = 512;          // candidates that are ranked against each other
constexpr int kChunks = 4096;      // partial weights by index of a long row
constexpr int kListed = 8192;      // candidates of a long row's limits
constexpr int kMaxPieces = 32, kMaxParts = 128;
constexpr int kLevels = 4096 / kThreads;      // groups of four that a thread holds of a short row

typedef unsigned long long u64;
typedef unsigned __int128 u128;
constexpr int kNarrowItems = 1 << 20;          // rows summed in 64 bits

// sums of weights, at most 2^52 each, from many threads at once: S is u64 or u128 (two atomic additions, the second only where
// the first has passed 2^64)
template <typename S, int N>
struct Sums {
  u64 v[N];
  __device__ __forceinline__ u64 get(int i) const { return v[i]; }
  __device__ __forceinline__ void set(int i, u64 x) { v[i] = x; }
  __device__ __forceinline__ void add(int i, u64 w) { atomicAdd(&v[i], w); }
};
template <int N>
struct Sums<u128, N> {
  u64 lo[N];
  unsigned hi[N];                              // a sum is below 2^82
  __device__ __forceinline__ u128 get(int i) const { return static_cast<u128>(hi[i]) << 64 | lo[i]; }
  __device__ __forceinline__ void set(int i, u128 x) { lo[i] = static_cast<u64>(x), hi[i] = static_cast<unsigned>(x >> 64); }
  __device__ __forceinline__ void add(int i, u64 w) {
    if (atomicAdd(&lo[i], w) > ~w) atomicAdd(&hi[i], 1u);
  }
};
__device__ __forceinline__ double as_double(u64 v) { return static_cast<double>(v); }
__device__ __forceinline__ double as_double(u128 v) {
  return fma(static_cast<double>(static_cast<u64>(v >> 64)), 18446744073709551616.0, static_cast<double>(static_cast<u64>(v)));
}
// a whole number that S holds
template <typename S>
__device__ __forceinline__ S as_sum(double x) {
  if constexpr (sizeof(S) == 8) {
    return static_cast<u64>(x);
  } else {
    const u64 hi = static_cast<u64>(x * 5.421010862427522e-20);      // 2^-64
    return static_cast<u128>(hi) << 64 | static_cast<u64>(fma(static_cast<double>(hi), -18446744073709551616.0, x));
  }
}

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
  // long rows: pieces of `piece` items, chunks of `span`; workspace
  // and, for the passes that leave little behind, parts of `part` items
  int pieces, piece, parts, part, span, chunks, room;
  float* tops;                     // (rows, parts)
  void* mass;                      // (rows, pieces, kBins) sums
  unsigned* count;
  void* state;                     // (rows) RowState
  unsigned* listed;                // (rows, parts): candidates of the part, which may be more than `room`
  u64* list;                       // (rows, parts, room): their places in the order
  void* chunk;                     // (rows, chunks) sums: weight of what is surely kept
};

struct Row {                       // a row's settings, the same on every thread
  double c;                        // log2(e) / T
  double p, m;                     // m as a scaled weight
  long long k;                     // 0: none
  bool by_p;
};

// a value that every lane holds, into scalar registers: what a row is scaled and compared with would fill a third of the vector
// registers
__device__ __forceinline__ u64 uniform(u64 v) {
  return static_cast<u64>(static_cast<unsigned>(__builtin_amdgcn_readfirstlane(static_cast<int>(v >> 32)))) << 32 |
         static_cast<unsigned>(__builtin_amdgcn_readfirstlane(static_cast<int>(v)));
}
__device__ __forceinline__ u128 uniform(u128 v) {
  return static_cast<u128>(uniform(static_cast<u64>(v >> 64))) << 64 | uniform(static_cast<u64>(v));
}
__device__ __forceinline__ double uniform(double v) {
  return __longlong_as_double(static_cast<long long>(uniform(static_cast<u64>(__double_as_longlong(v)))));
}

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
  r.c = uniform(t > 0.0 ? fmin(1.4426950408889634074 / t, 1e300) : 1.0);      // finite: the top's own 0 times it is 0
  r.m = uniform(m > 0.0 ? ldexp(m, g.bits) : 0.0);
  return r;
}

// an item's place in the order, the largest first: its score as a whole number in the scores' order (both zeros are the same
// score; NaN is dealt with before) above the complement of its index
__device__ __forceinline__ u64 place(float l, int i) {
  const unsigned b = __float_as_uint(l + 0.f);
  return static_cast<u64>(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | static_cast<unsigned>(~i);
}
__device__ __forceinline__ float score_at(u64 place) {
  const unsigned k = static_cast<unsigned>(place >> 32);
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ int index_at(u64 place) { return static_cast<int>(~static_cast<unsigned>(place)); }

// (2^f - 1) / f for |f| <= 1/2: a polynomial that interpolates it at Chebyshev's points, to 4e-14 of 2^f.  Written out because the
// compiler adds onto a copy of each coefficient, made for every item: 8 instructions of 34 (64 rows of 1,000,000: the histogram 61 us
// instead of 79)
__device__ __forceinline__ double exp2_slope(double f) {
  double y;
  asm("v_fma_f64 %0, %2, %1, %3\n\tv_fma_f64 %0, %0, %1, %4\n\tv_fma_f64 %0, %0, %1, %5\n\tv_fma_f64 %0, %0, %1, %6\n\t"
      "v_fma_f64 %0, %0, %1, %7\n\tv_fma_f64 %0, %0, %1, %8\n\tv_fma_f64 %0, %0, %1, %9\n\tv_fma_f64 %0, %0, %1, %10"
      : "=&v"(y)
      : "v"(f), "v"(1.0203121047189341e-07), "s"(1.3255224879317324e-06), "s"(1.525268684635191e-05), "s"(0.0001540345585244999),
        "s"(0.0013333558179042969), "s"(0.009618129159402565), "s"(0.055504108664760424), "s"(0.2402265069581299),
        "s"(0.6931471805599453));
  return y;
}
// max(d, 0) up to 2^-1022: a negative number's high half becomes 0
__device__ __forceinline__ double raised(double d) { return __hiloint2double(max(__double2hiint(d), 0), __double2loint(d)); }

// A row's scale: what turns a score into a bin of the histogram and into a weight.  d = (max - l) log2(e) / T; an item is live
// if d < last: -inf, NaN and what lies so far below that its weight is 0 are not.  In the bit patterns: adding 1.5 * 2^52 to a
// double rounds it to a whole number that stands in its low bits, for a quarter of a conversion's cost.
struct Scale {
  double top, c, last, bins;
  int bits;

  // (max = +inf stands here as a number above every other score with an endless c: what equals it comes out as -inf, live, all
  // else as +inf; live items' d is raised to 0 below)
  __device__ __forceinline__ double below(float l) const { return (top - static_cast<double>(l)) * c; }
  __device__ __forceinline__ bool live(double d) const { return d < last; }
  // of a live item: 0 .. kBins - 2
  __device__ __forceinline__ int bin(double d) const {
    return static_cast<int>(static_cast<unsigned>(__double_as_longlong(fma(raised(d), bins, 6755399441055744.0))));
  }
  // of a live item: 2^(bits - d), to be rounded to a whole number.  exact at d = 0
  __device__ __forceinline__ double weight(double d) const {
    d = raised(d);
    const double t = d + 6755399441055744.0, f = (t - 6755399441055744.0) - d;
    const double y = fma(exp2_slope(f), f, 1.0);
    const int n = static_cast<int>(static_cast<unsigned>(__double_as_longlong(t)));
    return __hiloint2double(__double2hiint(y) + (bits - n) * (1 << 20), __double2loint(y));
  }
};
__device__ __forceinline__ Scale scale_of(float top, const Row& r, int bits) {
  const bool endless = top == __builtin_inff();
  return Scale{uniform(endless ? 1e39 : static_cast<double>(top)), uniform(endless ? 1e300 : r.c), uniform(bits + 1.0),
               uniform((kBins - 2.0) / (bits + 1.0)), bits};
}
__device__ __forceinline__ u64 whole(double w) {                  // w < 2^52, to the nearest
  return static_cast<u64>(__double_as_longlong(w + 4503599627370496.0)) & 0xfffffffffffffull;
}

template <typename S>
struct Histogram {
  Sums<S, kBins> mass;
  unsigned count[kBins];
};

template <typename S>
struct Shared {
  Histogram<S> hist;               // of the row, or of a subdivision
  bool divided;                    // a subdivision has replaced the row's
  u64 few_place[kFew], few_weight[kFew];
  S wave_a[kWaves];
  u64 wave_b[kWaves];
  u64 limit;
  S limit_mass;
  unsigned few;
  // of find_bin, two in turn: what one call leaves is read while the next one starts
  S before_mass[2];
  unsigned before_count[2];
  int found[2];
};

// sum of the lanes below this one
template <typename S>
__device__ __forceinline__ S wave_before(S v) {
  return wave_scan(v, S{0}, [](S a, S b) { return a + b; }) - v;
}

// The bin, counted from bin 0 on, in which the sum of counts reaches need (by_mass: the sum of weights), need = need_of(total
// weight), and the sums before it; kBins if there is none.  Two barriers; `turn` is the calls' own count.  Also starts an empty
// list of candidates.
template <typename S, typename Need>
__device__ __forceinline__ int find_bin(Shared<S>& sh, const Histogram<S>& h, int& turn, bool by_mass, Need need_of,
                                        unsigned& before_count, S& before_mass) {
  const int t = threadIdx.x, wave = t / kWave, lane = t % kWave, k = turn++ & 1;
  if (t == 0) sh.found[k] = kBins, sh.before_count[k] = 0, sh.before_mass[k] = 0, sh.few = 0;
  S m[kPer], ms = 0;
  unsigned c[kPer], cs = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) m[i] = h.mass.get(kPer * t + i), c[i] = h.count[kPer * t + i], ms += m[i], cs += c[i];
  S mb = wave_before(ms), total = 0;
  u64 cb = wave_before(u64{cs});
  if (lane == kWave - 1) sh.wave_a[wave] = mb + ms, sh.wave_b[wave] = cb + cs;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    total += sh.wave_a[i];
    if (i < wave) mb += sh.wave_a[i], cb += sh.wave_b[i];
  }
  const S need = need_of(uniform(total));
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const S a = by_mass ? mb : S{cb}, v = by_mass ? m[i] : S{c[i]};
    if (a < need && need <= a + v) sh.found[k] = kPer * t + i, sh.before_count[k] = static_cast<unsigned>(cb), sh.before_mass[k] = mb;
    mb += m[i], cb += c[i];
  }
  __syncthreads();
  before_count = __builtin_amdgcn_readfirstlane(sh.before_count[k]), before_mass = uniform(sh.before_mass[k]);
  return __builtin_amdgcn_readfirstlane(sh.found[k]);
}

template <typename S>
__device__ __forceinline__ void clear(Histogram<S>& h) {           // a barrier has to follow
  for (int i = threadIdx.x; i < kBins; i += kThreads) h.mass.set(i, 0), h.count[i] = 0;
}

// a cleared histogram
template <typename S, typename Src>
__device__ __forceinline__ void fill(Histogram<S>& h, const Src& src, const Scale& sc, bool counts, bool masses) {
  src([&](float l, int) {
    const double d = sc.below(l);
    if (!sc.live(d)) return;
    const int b = sc.bin(d);
    if (counts) atomicAdd(&h.count[b], 1u);
    if (masses) h.mass.add(b, whole(sc.weight(d)));
  });
  __syncthreads();
}

// total weight of a histogram, on every thread
template <typename S>
__device__ __forceinline__ S total_mass(Shared<S>& sh, const Histogram<S>& h) {
  S v = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) v += h.mass.get(kPer * threadIdx.x + i);
  v = wave_sum(v);
  if (threadIdx.x % kWave == 0) sh.wave_a[threadIdx.x / kWave] = v;
  __syncthreads();
  S s = 0;
#pragma unroll
  for (int i = 0; i < kWaves; ++i) s += sh.wave_a[i];
  __syncthreads();
  return uniform(s);
}

template <typename S>
__device__ __forceinline__ S share(double p, S total) {            // the weight that top-p asks for
  const S need = uniform(as_sum<S>(ceil(p * as_double(total))));
  return need < 1 ? S{1} : need < total ? need : total;
}

// The limit among the live items of `src` in bins lo_bin .. hi_bin, before which `count` items of weight `mass` stand in the
// order: by count, the item with which the count reaches `need`; by mass, the item with which the weight does.  -> its place;
// mass: with the item itself (by count only where `masses`).  The list of candidates is empty.
template <typename S, typename Src>
__device__ __forceinline__ u64 find_limit(Shared<S>& sh, const Src& src, const Scale& sc, int lo_bin, int hi_bin, bool by_mass, bool masses,
                                          S need, unsigned count, S& mass, int& turn) {
  const int t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t / kWave), lane = t % kWave;
  u64 lo = 0, hi = ~u64{0};
  auto members = [&](auto f) {
    src([&](float l, int i) {
      const double d = sc.below(l);
      if (!sc.live(d)) return;
      const int b = sc.bin(d);
      if (b < lo_bin || b > hi_bin) return;
      const u64 at = place(l, i);
      if (at >= lo && at <= hi) f(at, d);
    });
  };
  for (bool first = true;; first = false) {
    members([&](u64 at, double d) {
      const unsigned k = atomicAdd(&sh.few, 1u);
      if (k < kFew) sh.few_place[k] = at, sh.few_weight[k] = masses ? whole(sc.weight(d)) : 0;
    });
    __syncthreads();
    if (sh.few <= kFew) break;
    if (first) {                                         // the range they span
      u64 least = ~u64{0}, most = 0;
      members([&](u64 at, double) { least = min(least, at), most = max(most, at); });
      for (int off = 32; off > 0; off >>= 1) {
        least = min(least, static_cast<u64>(__shfl_xor(least, off)));
        most = max(most, static_cast<u64>(__shfl_xor(most, off)));
      }
      if (lane == 0) sh.wave_a[wave] = least, sh.wave_b[wave] = most;
      __syncthreads();
      lo = static_cast<u64>(sh.wave_a[0]), hi = sh.wave_b[0];
      for (int i = 1; i < kWaves; ++i) lo = min(lo, static_cast<u64>(sh.wave_a[i])), hi = max(hi, sh.wave_b[i]);
      lo = uniform(lo), hi = uniform(hi);
    }
    // all places differ: a turn leaves at most 1 / 1024 of the range, and single places at last
    const int shift = max(0, 53 - __clzll(static_cast<long long>(hi - lo)));
    if (t == 0) sh.divided = true;
    clear(sh.hist);
    __syncthreads();
    members([&](u64 at, double d) {
      const int digit = static_cast<int>((hi - at) >> shift);
      if (!by_mass) atomicAdd(&sh.hist.count[digit], 1u);
      if (masses) sh.hist.mass.add(digit, whole(sc.weight(d)));
    });
    __syncthreads();
    unsigned bc;
    S bm;
    const S rest = need - (by_mass ? mass : S{count});
    const int digit = min(find_bin(sh, sh.hist, turn, by_mass, [&](S) { return rest; }, bc, bm), kBins - 1);
    count += bc, mass += bm;
    hi -= static_cast<u64>(digit) << shift;
    lo = max(lo, hi - ((u64{1} << shift) - 1));
  }
  // each against all: `team` threads a candidate
  const int m = static_cast<int>(sh.few);
  int team = kWave;
  while (team * m > kThreads) team >>= 1;
  const int me = t / team;
  u64 mb = 0;
  unsigned cb = 0;
  const u64 at = me < m ? sh.few_place[me] : 0;
  if (me < m)
    for (int j = t % team; j < m; j += team)
      if (sh.few_place[j] > at) cb += 1, mb += sh.few_weight[j];
  for (int off = 1; off < team; off <<= 1) cb += __shfl_xor(cb, off), mb += __shfl_xor(mb, off);
  if (me < m && t % team == 0) {
    const u64 w = sh.few_weight[me];
    const S before = by_mass ? mass + mb : S{count + cb}, own = by_mass ? w : 1;
    if (before < need && need <= before + own) sh.limit = at, sh.limit_mass = mass + mb + w;
  }
  __syncthreads();
  mass = uniform(sh.limit_mass);
  return uniform(sh.limit);
}

// the weight of an item if it is kept: its place is not below `limit`, the lower of the limits
__device__ __forceinline__ u64 kept(float l, int i, const Scale& sc, u64 limit, double min_weight) {
  const double d = sc.below(l);
  if (!sc.live(d) || place(l, i) < limit) return 0;
  const double w = sc.weight(d);
  return w >= min_weight ? whole(w) : 0;
}

template <typename S>
__device__ __forceinline__ S goal_of(float u, S total) {           // drawn: the first item with more than this up to it
  const double x = u;
  const S goal = x > 0.0 ? as_sum<S>(fmin(x, 1.0) * as_double(total)) : S{0};
  return goal < total ? goal : total - 1;
}

// The wave's V items a lane, kept weights w: where the sum from `before` on passes `goal`, that lane writes the item.  -> whether
// some lane did; before is moved on.
template <int V, typename S>
__device__ __forceinline__ bool draw(const SampleArgs& g, int row, int base, const u64 (&w)[V], S goal, S total, S& before) {
  u64 sum = 0;                                           // 64 lanes of at most 8 weights: below 2^61
#pragma unroll
  for (int j = 0; j < V; ++j) sum += w[j];
  S b = before + wave_before(sum);
  const bool hit = b <= goal && goal < b + sum;
  if (hit) {
    bool done = false;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (!done && goal < b + w[j]) {
        g.ids[row] = base + j;
        g.prob[row] = static_cast<float>(static_cast<double>(w[j]) / as_double(total));
        done = true;
      }
      b += w[j];
    }
  }
  if (__ballot(hit)) return true;
  before += wave_sum(sum);
  return false;
}

__device__ __forceinline__ float group_max(float v, float* red) {
  v = wave_max(v);
  if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = v;
  __syncthreads();
  v = red[0];
  for (int i = 1; i < static_cast<int>(blockDim.x) / kWave; ++i) v = fmaxf(v, red[i]);
  return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v)));
}

// ---- one workgroup a row, the row in LDS ------------------------------------------------------------------------------------
// In registers the compiler keeps what one pass derives from a score for the next, for every score, and spills (69 us instead of
// 43 for 512 rows of 10677).  What bounds a row is 64-bit arithmetic on one compute unit, two passes of ~24 operations an item,
// not its barriers (eleven instead of twenty saved half a microsecond): 14.5 us for 10677 items.
template <typename T>
__global__ __launch_bounds__(kThreads) void sample_row_kernel(const SampleArgs g) {
  __shared__ Shared<u64> sh;
  __shared__ float red[kWaves];
  __shared__ u64 part[kLevels * kWaves];
  extern __shared__ __attribute__((aligned(16))) char lds_row[];
  constexpr int V = 4, LEVEL = kThreads * V;
  static_assert(kLevels * kWaves <= kWave, "one lane a part");
  const int row = blockIdx.x, t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t / kWave), lane = t % kWave;
  const T* l = static_cast<const T*>(g.l) + row * g.ld;
  pack<T, V>* mine = reinterpret_cast<pack<T, V>*>(lds_row) + t;        // level i of a thread: mine[i * kThreads]
  const Row r = row_settings(g, row);
  const int levels = (g.n + LEVEL - 1) / LEVEL;
  clear(sh.hist);
  float top = -__builtin_inff();
  for (int i = 0; i < levels; ++i) {
    const int base = i * LEVEL + t * V, n = g.n - base;
    float x[V];
    load_vec<T, V>(x, l + base, n);
    pack<T, V> a;
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (j >= n) x[j] = -__builtin_inff();
      a.v[j] = from_f32<T>(x[j]);
      top = fmaxf(top, x[j]);
    }
    mine[i * kThreads] = a;
  }
  top = group_max(top, red);
  if (top == -__builtin_inff()) {                        // nothing to draw from (also N = 0)
    if (t == 0) g.ids[row] = -1, g.prob[row] = 0.f;
    return;
  }
  const Scale sc = scale_of(top, r, g.bits);
  auto src = [&](auto f) {
#pragma unroll 1
    for (int i = 0; i < levels; ++i) {
      const int base = i * LEVEL + t * V;
      if (base >= g.n) break;
      const pack<T, V> a = mine[i * kThreads];
#pragma unroll
      for (int j = 0; j < V; ++j) f(to_f32(a.v[j]), base + j);
    }
  };
  u64 limit = 0, total = 0;                              // weight of the top-k items
  int turn = 0;
  bool again = false;
#pragma unroll 1
  for (int by_mass = 0; by_mass < 2; ++by_mass) {        // top-k, then top-p
    if (by_mass ? !r.by_p : r.k == 0) continue;
    if (again) clear(sh.hist), __syncthreads();
    if (again || !turn) {
      if (t == 0) sh.divided = false;
      fill(sh.hist, src, sc, r.k > 0, r.by_p);
    }
    unsigned count;
    u64 mass, need = 0;
    const int b = find_bin(sh, sh.hist, turn, by_mass, [&](u64 all) {
      if (!by_mass || r.k == 0) total = all;
      return need = by_mass ? share(r.p, total) : static_cast<u64>(r.k);
    }, count, mass);
    if (b < kBins) {
      limit = max(limit, find_limit(sh, src, sc, b, b, by_mass, r.by_p, need, count, mass, turn));
      total = mass;
    }
    again = sh.divided;
  }
  // kept weight by index: level i of wave w comes after level i of wave w - 1, and after every wave's level i - 1
  auto weights = [&](int i, u64 (&w)[V]) {
    const int base = i * LEVEL + t * V;
    const pack<T, V> a = mine[i * kThreads];
    u64 sum = 0;
#pragma unroll
    for (int j = 0; j < V; ++j) w[j] = kept(to_f32(a.v[j]), base + j, sc, limit, r.m), sum += w[j];
    return sum;
  };
  u64 w[V];
#pragma unroll 1
  for (int i = 0; i < levels; ++i) {
    const u64 sum = wave_sum(weights(i, w));
    if (lane == 0) part[i * kWaves + wave] = sum;
  }
  __syncthreads();
  const u64 own = lane < levels * kWaves ? part[lane] : 0, all = wave_sum(own), goal = goal_of(g.u[row], all);
  u64 before = wave_before(own);
  const int owner = __ffsll(static_cast<unsigned long long>(__ballot(before <= goal && goal < before + own))) - 1;
  if (owner % kWaves != wave) return;
  before = from_lane(before, owner);
  weights(owner / kWaves, w);
  draw<V>(g, row, owner / kWaves * LEVEL + t * V, w, goal, all, before);
}

// ---- long rows ----------------------------------------------------------------------------------------------------------------

template <typename S>
struct RowState {
  S total, k_mass, p_mass;         // weight of the row; before the top-k bin; before the top-p bins
  unsigned k_count;                // items before the top-k bin
  int k_bin, p_lo, p_hi;           // kBins: no such limit
};

// f(score, index) for the items [lo, hi) of a row.  Whole vectors first, U loads under way at once
template <typename T, typename F>
__device__ __forceinline__ void each(const T* row, int lo, int hi, F f) {
  constexpr int V = 16 / sizeof(T), U = 4;
  const int step = blockDim.x * V, end = lo + (hi - lo) / V * V;
  int base = lo + threadIdx.x * V;
  for (; base + (U - 1) * step < end; base += U * step) {
    pack<T, V> a[U];
#pragma unroll
    for (int u = 0; u < U; ++u) a[u] = load_pack<T, V>(row + base + u * step);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < V; ++j) f(to_f32(a[u].v[j]), base + u * step + j);
  }
  for (; base < end; base += step) {
    const pack<T, V> a = load_pack<T, V>(row + base);
#pragma unroll
    for (int j = 0; j < V; ++j) f(to_f32(a.v[j]), base + j);
  }
  const int i = end + threadIdx.x;
  if (i < hi) f(to_f32(row[i]), i);
}

template <typename T>
__global__ __launch_bounds__(256) void sample_top_kernel(const SampleArgs g) {
  __shared__ float red[4];
  const int row = blockIdx.x / g.parts, z = blockIdx.x % g.parts, lo = z * g.part;
  float top = -__builtin_inff();
  each(static_cast<const T*>(g.l) + row * g.ld, lo, min(g.n, lo + g.part), [&](float x, int) { top = fmaxf(top, x); });
  top = group_max(top, red);
  if (threadIdx.x == 0) g.tops[blockIdx.x] = top;
}

__device__ __forceinline__ float row_top(const SampleArgs& g, int row) {
  float top = -__builtin_inff();
  for (int i = threadIdx.x % kWave; i < g.parts; i += kWave) top = fmaxf(top, g.tops[row * g.parts + i]);
  return wave_max(top);
}

template <typename T, typename S>
__global__ __launch_bounds__(kThreads) void sample_histogram_kernel(const SampleArgs g) {
  __shared__ Histogram<S> hist;
  const int row = blockIdx.x / g.pieces, z = blockIdx.x % g.pieces, lo = z * g.piece, hi = min(g.n, lo + g.piece);
  const Row r = row_settings(g, row);
  if (!(r.k > 0 || r.by_p)) return;
  clear(hist);
  __syncthreads();
  const T* l = static_cast<const T*>(g.l) + row * g.ld;
  fill(hist, [&](auto f) { each(l, lo, hi, f); }, scale_of(row_top(g, row), r, g.bits), r.k > 0, r.by_p);
  S* mass = static_cast<S*>(g.mass) + static_cast<long long>(blockIdx.x) * kBins;
  unsigned* count = g.count + static_cast<long long>(blockIdx.x) * kBins;
  for (int i = threadIdx.x; i < kBins; i += kThreads) {
    if (r.by_p) mass[i] = hist.mass.get(i);
    if (r.k > 0) count[i] = hist.count[i];
  }
}

template <typename S>
__global__ __launch_bounds__(kThreads) void sample_bins_kernel(const SampleArgs g) {
  __shared__ Shared<S> sh;
  Histogram<S>& hist = sh.hist;
  const int row = blockIdx.x, t = threadIdx.x;
  const Row r = row_settings(g, row);
  RowState<S> s{0, 0, 0, 0, kBins, kBins, kBins};
  if (r.k > 0 || r.by_p) {
    static_assert(kPer == 4, "16 bytes of counts a thread");
    const long long at = static_cast<long long>(row) * g.pieces * kBins + kPer * t;      // this thread's bins
    S m[kPer] = {};
    unsigned c[kPer] = {};
    if (r.by_p) {
#pragma unroll 8
      for (int z = 0; z < g.pieces; ++z) {
        const S* piece = static_cast<const S*>(g.mass) + at + static_cast<long long>(z) * kBins;
        if constexpr (sizeof(S) == 8) {
          const ulonglong2* p = reinterpret_cast<const ulonglong2*>(piece);
          const ulonglong2 a = p[0], b = p[1];
          m[0] += a.x, m[1] += a.y, m[2] += b.x, m[3] += b.y;
        } else {
#pragma unroll
          for (int i = 0; i < kPer; ++i) m[i] += piece[i];
        }
      }
    }
    if (r.k > 0) {
#pragma unroll 8
      for (int z = 0; z < g.pieces; ++z) {
        const uint4 a = *reinterpret_cast<const uint4*>(g.count + at + static_cast<long long>(z) * kBins);
        c[0] += a.x, c[1] += a.y, c[2] += a.z, c[3] += a.w;
      }
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) hist.mass.set(kPer * t + i, m[i]), hist.count[kPer * t + i] = c[i];
    __syncthreads();
    int turn = 0;
    S most = 0, least = 0;                               // the weight of the top-k items lies between them
    if (r.by_p) least = most = s.total = total_mass(sh, hist);
    if (r.k > 0) {
      s.k_bin = find_bin(sh, hist, turn, false, [&](S) { return static_cast<S>(r.k); }, s.k_count, s.k_mass);
      if (s.k_bin < kBins) least = s.k_mass, most = s.k_mass + hist.mass.get(s.k_bin);
    }
    if (r.by_p && s.total > 0) {                         // no total: a row of nothing but -inf and NaN
      unsigned c;
      S m;
      s.p_hi = find_bin(sh, hist, turn, true, [&](S) { return share(r.p, most); }, c, m);
      s.p_lo = least > 0 ? find_bin(sh, hist, turn, true, [&](S) { return share(r.p, least); }, c, s.p_mass) : 0;
    }
  }
  if (t == 0) static_cast<RowState<S>*>(g.state)[row] = s;
}

template <typename S>
__device__ __forceinline__ bool surely_kept(const RowState<S>& s, int bin) { return bin < s.k_bin && bin < s.p_lo; }
template <typename S>
__device__ __forceinline__ bool candidate(const RowState<S>& s, int bin) { return bin == s.k_bin || (bin >= s.p_lo && bin <= s.p_hi); }

// one wave a chunk of the part
template <typename T, typename S>
__global__ __launch_bounds__(256) void sample_parts_kernel(const SampleArgs g) {
  __shared__ unsigned listed;
  constexpr int V = 16 / sizeof(T), U = 4;
  const int row = blockIdx.x / g.parts, z = blockIdx.x % g.parts;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
  const T* l = static_cast<const T*>(g.l) + row * g.ld;
  const Row r = row_settings(g, row);
  const Scale sc = scale_of(row_top(g, row), r, g.bits);
  RowState<S> s{0, 0, 0, 0, kBins, kBins, kBins};
  if (r.k > 0 || r.by_p) s = static_cast<const RowState<S>*>(g.state)[row];
  u64* list = g.list + static_cast<long long>(blockIdx.x) * g.room;
  if (threadIdx.x == 0) listed = 0;
  __syncthreads();
  const int c0 = z * (g.part / g.span), c1 = min(g.chunks, c0 + g.part / g.span);
  for (int ch = c0 + wave; ch < c1; ch += 4) {
    u64 sum = 0;                                         // of a lane: at most 4096 items of a chunk, so below 2^64
    const int end = min(g.n, (ch + 1) * g.span);
    auto item = [&](float x, int i) {
      const double d = sc.below(x);
      if (!sc.live(d)) return;
      const int b = sc.bin(d);
      if (surely_kept(s, b)) {
        const double w = sc.weight(d);
        if (w >= r.m) sum += whole(w);
      } else if (candidate(s, b)) {
        const unsigned k = atomicAdd(&listed, 1u);
        if (k < static_cast<unsigned>(g.room)) list[k] = place(x, i);
      }
    };
    int base = ch * g.span + lane * V;
    if ((ch + 1) * g.span <= g.n) {                      // a whole chunk: a multiple of U vectors a lane
      for (; base < end; base += U * kWave * V) {
        pack<T, V> a[U];
#pragma unroll
        for (int u = 0; u < U; ++u) a[u] = load_pack<T, V>(l + base + u * kWave * V);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int j = 0; j < V; ++j) item(to_f32(a[u].v[j]), base + u * kWave * V + j);
      }
    } else {
      for (; base < end; base += kWave * V)
#pragma unroll
        for (int j = 0; j < V; ++j)
          if (base + j < end) item(to_f32(l[base + j]), base + j);
    }
    const S all = wave_sum(S{sum});
    if (lane == 0) static_cast<S*>(g.chunk)[static_cast<long long>(row) * g.chunks + ch] = all;
  }
  __syncthreads();
  if (threadIdx.x == 0) g.listed[blockIdx.x] = listed;
}

template <typename T, typename S>
__global__ __launch_bounds__(kThreads) void sample_draw_kernel(const SampleArgs g) {
  __shared__ Shared<S> sh;
  __shared__ Sums<S, kChunks> chunk;
  __shared__ u64 lds_list[kListed];
  constexpr int V = 16 / sizeof(T);
  const int row = blockIdx.x, t = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t / kWave), lane = t % kWave;
  const T* l = static_cast<const T*>(g.l) + row * g.ld;
  const Row r = row_settings(g, row);
  const float top = row_top(g, row);
  if (top == -__builtin_inff()) {
    if (t == 0) g.ids[row] = -1, g.prob[row] = 0.f;
    return;
  }
  const Scale sc = scale_of(top, r, g.bits);
  RowState<S> s{0, 0, 0, 0, kBins, kBins, kBins};
  if (r.k > 0 || r.by_p) s = static_cast<const RowState<S>*>(g.state)[row];
  for (int i = t; i < g.chunks; i += kThreads) chunk.set(i, static_cast<const S*>(g.chunk)[static_cast<long long>(row) * g.chunks + i]);
  u64 limit = 0;
  if (s.k_bin < kBins || s.p_lo < kBins) {
    // the parts' lists, one behind the other in LDS if they fit
    int listed = 0;
    bool whole_list = true;
    for (int z = 0; z < g.parts; ++z) {
      const unsigned n = g.listed[row * g.parts + z];
      whole_list = whole_list && n <= static_cast<unsigned>(g.room);
      if (!whole_list) break;
      if (z % kWaves == wave)
        for (int i = lane; i < static_cast<int>(n) && listed + i < kListed; i += kWave)
          lds_list[listed + i] = g.list[(static_cast<long long>(row) * g.parts + z) * g.room + i];
      listed += static_cast<int>(n);
    }
    whole_list = whole_list && listed <= kListed;
    auto limits = [&](auto src) {
      int turn = 0;
      S total = s.total;
#pragma unroll 1
      for (int by_mass = 0; by_mass < 2; ++by_mass) {    // top-k, then top-p
        if ((by_mass ? s.p_lo : s.k_bin) == kBins) continue;
        S mass = by_mass ? s.p_mass : s.k_mass;
        __syncthreads();
        if (t == 0) sh.few = 0;
        __syncthreads();
        limit = max(limit, find_limit(sh, src, sc, by_mass ? s.p_lo : s.k_bin, by_mass ? s.p_hi : s.k_bin, by_mass, r.by_p,
                                      by_mass ? share(r.p, total) : static_cast<S>(r.k), s.k_count, mass, turn));
        total = mass;
      }
    };
    if (whole_list) {
      auto src = [&](auto f) {
        for (int i = t; i < listed; i += kThreads) {
          const u64 at = lds_list[i];
          f(score_at(at), index_at(at));
        }
      };
      __syncthreads();
      limits(src);
      src([&](float x, int i) {
        const u64 w = kept(x, i, sc, limit, r.m);
        if (w) chunk.add(i / g.span, w);
      });
    } else {                                             // too many candidates for the list: over the row itself
      limits([&](auto f) { each(l, 0, g.n, f); });
      __syncthreads();
      for (int ch = wave; ch < g.chunks; ch += kWaves) {
        u64 sum = 0;
        const int end = min(g.n, (ch + 1) * g.span);
        for (int base = ch * g.span + lane * V; base < end; base += kWave * V) {
          float x[V];
          load_vec<T, V>(x, l + base, end - base);
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (base + j < end) sum += kept(x[j], base + j, sc, limit, r.m);
        }
        const S all = wave_sum(S{sum});
        if (lane == 0) chunk.set(ch, all);
      }
    }
  }
  __syncthreads();
  if (wave != 0) return;
  // the chunk, then the item, at which the sum passes the drawn share
  const int per = (g.chunks + kWave - 1) / kWave, c0 = min(g.chunks, lane * per), c1 = min(g.chunks, c0 + per);
  S mine = 0;
  for (int i = c0; i < c1; ++i) mine += chunk.get(i);
  const S total = wave_sum(mine), goal = goal_of(g.u[row], total);
  S before = wave_before(mine);
  int at = -1;
  if (before <= goal && goal < before + mine)
    for (at = c0; before + chunk.get(at) <= goal; ++at) before += chunk.get(at);
  const int owner = __ffsll(static_cast<unsigned long long>(__ballot(at >= 0))) - 1;
  at = __builtin_amdgcn_readlane(at, owner);
  before = from_lane(before, owner);
  const int end = min(g.n, (at + 1) * g.span);
  for (int base0 = at * g.span; base0 < end; base0 += kWave * V) {
    const int base = base0 + lane * V;
    float x[V];
    load_vec<T, V>(x, l + base, end - base);
    u64 w[V];
#pragma unroll
    for (int j = 0; j < V; ++j) w[j] = base + j < end ? kept(x[j], base + j, sc, limit, r.m) : 0;
    if (draw<V>(g, row, base, w, goal, total, before)) return;
  }
}

// items of a row that one workgroup holds
constexpr int kRowItems = kLevels * kThreads * 4;
static_assert(kRowItems <= kNarrowItems, "short rows are summed in 64 bits");

// Long rows are done this many at a time, one batch after the other in the same workspace: their histograms and lists are as large as
// their scores (69878 x 20000 fp32: 1.1 GB of workspace instead of 4.6).  In batches of 4096 rows 20000 x 20000 fp32 takes 8 % longer: the ends of five launches each.
constexpr int64_t kRowsAtOnce = 16384;

// long rows: the workspace, from `base` on (null: its size alone)
inline size_t lay_out(SampleArgs& g, int64_t rows, int64_t n, int size, char* base) {
  const int64_t vec = 16 / size;
  g.span = static_cast<int>(4 * kWave * vec);            // four vectors a lane
  while ((n + g.span - 1) / g.span > kChunks) g.span *= 2;
  g.chunks = static_cast<int>((n + g.span - 1) / g.span);
  // enough for four workgroups a compute unit, of at least 8192 items (a piece leaves a histogram to be read: 32 a row at most)
  auto cut = [&](int64_t most, int& count, int& length) {
    const int64_t want = std::min<int64_t>({most, std::max<int64_t>(1, 1024 / rows), std::max<int64_t>(1, n / 8192)});
    const int64_t per = (g.chunks + want - 1) / want;    // chunks
    length = static_cast<int>(std::min<int64_t>(per * g.span, int64_t{1} << 30));
    count = static_cast<int>((g.chunks + per - 1) / per);
  };
  cut(kMaxPieces, g.pieces, g.piece);
  cut(kMaxParts, g.parts, g.part);
  g.room = std::min(kListed, g.part / 4);
  size_t at = 0;
  auto take_bytes = [&](auto*& p, size_t bytes) {
    p = reinterpret_cast<std::remove_reference_t<decltype(p)>>(base + at);
    at += (bytes + 255) & ~size_t{255};
  };
  auto take = [&](auto*& p, size_t count) { take_bytes(p, count * sizeof(*p)); };
  const size_t pieces = static_cast<size_t>(rows) * g.pieces, parts = static_cast<size_t>(rows) * g.parts;
  take(g.tops, parts);
  const bool narrow = n <= kNarrowItems;
  const size_t sum = narrow ? sizeof(u64) : sizeof(u128);
  take_bytes(g.mass, pieces * kBins * sum);
  take(g.count, pieces * kBins);
  take_bytes(g.state, rows * (narrow ? sizeof(RowState<u64>) : sizeof(RowState<u128>)));
  take(g.listed, parts);
  take(g.list, parts * g.room);
  take_bytes(g.chunk, static_cast<size_t>(rows) * g.chunks * sum);
  return at;
}

template <typename T, typename S>
void launch_long(const SampleArgs& g, bool limits, hipStream_t st) {
  const dim3 block(kThreads), rows(static_cast<unsigned>(g.rows)), pieces(static_cast<unsigned>(g.rows) * g.pieces),
      parts(static_cast<unsigned>(g.rows) * g.parts);
  hipLaunchKernelGGL(sample_top_kernel<T>, parts, dim3(256), 0, st, g);
  if (limits) {
    hipLaunchKernelGGL((sample_histogram_kernel<T, S>), pieces, block, 0, st, g);
    hipLaunchKernelGGL(sample_bins_kernel<S>, rows, block, 0, st, g);
  }
  hipLaunchKernelGGL((sample_parts_kernel<T, S>), parts, dim3(256), 0, st, g);
  hipLaunchKernelGGL((sample_draw_kernel<T, S>), rows, block, 0, st, g);
}

template <typename T>
void launch(const SampleArgs& g, bool limits, hipStream_t st) {
  constexpr int LEVEL = kThreads * 4;
  const size_t lds = static_cast<size_t>((g.n + LEVEL - 1) / LEVEL) * LEVEL * sizeof(T);
  const long long most = g.n <= kRowItems ? 1 << 22 : kRowsAtOnce;      // a launch has to stay below 2^32 threads
  for (long long r = 0; r < g.rows; r += most) {
    SampleArgs a = g;
    a.rows = static_cast<int>(std::min<long long>(most, g.rows - r));
    a.ids += r, a.prob += r, a.u += r, a.l = static_cast<const T*>(g.l) + r * g.ld;
    if (g.temperature) a.temperature += r;
    if (g.top_k) a.top_k += r;
    if (g.top_p) a.top_p += r;
    if (g.min_p) a.min_p += r;
    if (g.n <= kRowItems) hipLaunchKernelGGL(sample_row_kernel<T>, dim3(static_cast<unsigned>(a.rows)), dim3(kThreads), lds, st, a);
    else if (g.n <= kNarrowItems) launch_long<T, u64>(a, limits, st);
    else launch_long<T, u128>(a, limits, st);
  }
}

}  // namespace
}  // namespace sg

using namespace sg;

SG_API size_t sg_sample_rows_workspace_bytes(int64_t rows, int64_t n, int dtype) {
  if (rows <= 0 || n >= SG_SAMPLE_MAX_ITEMS || !valid_dtype(dtype)) return 0;
  const int size = dtype == SG_DTYPE_F32 ? 4 : 2;
  SampleArgs g{};
  return n <= kRowItems ? 0 : lay_out(g, std::min(rows, kRowsAtOnce), n, size, nullptr);
}

SG_API int sg_sample_rows_hip(int32_t* ids, float* prob, const void* logits, int64_t ld, int dtype, const float* u, int64_t rows,
                              int64_t n, double temperature, int64_t top_k, double top_p, double min_p, const float* temperature_rows,
                              const int32_t* top_k_rows, const float* top_p_rows, const float* min_p_rows, void* workspace,
                              size_t workspace_bytes, void* stream) {
  if (!valid_dtype(dtype)) return fail(SG_ERR_INVALID, "sample_rows: unknown dtype %d", dtype);
  if (rows < 0 || n < 0) return fail(SG_ERR_INVALID, "sample_rows: negative size");
  if (rows >= (1ll << 31) || n >= SG_SAMPLE_MAX_ITEMS) return fail(SG_ERR_UNSUPPORTED, "sample_rows: fewer than %d items", SG_SAMPLE_MAX_ITEMS);
  if (rows == 0) return SG_OK;
  if (!ids || !prob || !u || (n > 0 && !logits)) return fail(SG_ERR_INVALID, "sample_rows: null pointer argument");
  if (ld < n) return fail(SG_ERR_INVALID, "sample_rows: rows overlap");
  if (!(temperature >= 0.0) || !(top_p >= 0.0) || !(min_p >= 0.0) || top_k < 0)
    return fail(SG_ERR_INVALID, "sample_rows: temperature, top_k, top_p and min_p must not be negative");
  const int size = dtype == SG_DTYPE_F32 ? 4 : 2;
  const bool long_rows = n > kRowItems;
  if (long_rows && rows >= (1ll << 23)) return fail(SG_ERR_UNSUPPORTED, "sample_rows: too many rows");
  if (workspace_bytes < sg_sample_rows_workspace_bytes(rows, n, dtype) || (long_rows && !workspace))
    return fail(SG_ERR_WORKSPACE, "sample_rows workspace too small");
  if (long_rows && !aligned(workspace, 16)) return fail(SG_ERR_WORKSPACE, "sample_rows workspace has to be 16-byte aligned");
  int log_n = 0;
  while ((1ll << log_n) < n) ++log_n;
  SampleArgs g{};
  g.ids = ids, g.prob = prob, g.l = logits, g.u = u;
  g.temperature = temperature_rows, g.top_k = top_k_rows, g.top_p = top_p_rows, g.min_p = min_p_rows;
  g.t0 = temperature, g.p0 = top_p, g.m0 = min_p, g.k0 = top_k;
  g.ld = ld, g.rows = static_cast<int>(rows), g.n = static_cast<int>(n), g.bits = n <= kNarrowItems ? std::min(51, 63 - log_n) : 51;
  if (long_rows) lay_out(g, std::min(rows, kRowsAtOnce), n, size, static_cast<char*>(workspace));
  // whether any row can have a limit: otherwise the histogram has no reader
  const bool limits = top_k_rows || top_p_rows || temperature_rows || min_p_rows || (top_k > 0 && top_k < n) || top_p < 1.0 ||
                      temperature == 0.0 || min_p > 1.0;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == SG_DTYPE_F32) launch<float>(g, limits, st);
  else if (dtype == SG_DTYPE_F16) launch<f16>(g, limits, st);
  else launch<bf16>(g, limits, st);
  return check_launch("sample_rows");
}
