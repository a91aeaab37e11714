// Drawing a token from each row of logits (pa_sample): temperature, top-k, top-p
// and min-p, one uniform number a row.
//
// With M the row's largest logit a token weighs w = exp((x - M) / T).  Weights are
// formed in f64 (an error of about 2^-48) and summed as integers of 2^-shift (44
// bits for vocabularies up to 2^18): a sum does not depend on its order, so equal
// calls draw equal tokens, and a border between two tokens lies where the exact sums
// have it but for a few 2^-44 of the row's total.  (Sums of 10^5 f32 weights would
// move the borders by more than many tokens' weights.)
//
// Nothing is sorted.  What top-k and top-p keep of a row is all above a threshold
// value and the first `ties` tokens equal to it:
//   1  sample_max_kernel    the row's largest and least logit, in slices
//   2  sample_hist_kernel   counts and weights of 2048 equal intervals of the logits
//   3  sample_pick_kernel   the values in the interval where a threshold lies
//   4  sample_draw_kernel   the threshold among those values (radix selection),
//                           the kept weight of every slice, and, in the last
//                           workgroup of the row, the token
// 2 and 3 only where the call gives top_k or top_p; rows that do not use them pass
// through.  Each kernel reads the logits once, in workgroups of a slice of a row.
#include <algorithm>
#include <climits>

#include "pa_common.hpp"
#include "pa_internal.hpp"
#include "../../include/pa_dense.h"

namespace pa {
namespace {

constexpr int kThreads = 256;
constexpr int kBins = 2048;
constexpr int kMaxSlices = 64;
constexpr int kListMax = 4096;  // values that step 3 collects; more are read from the row again
constexpr int kDigits = 11;     // bits a round of the selection

// What a row has in the workspace.
struct Stats {  // of a slice
  float max, min;
  int at;  // of the first largest
  int pad;
};
struct Part {  // of a slice: what is kept of it
  unsigned long long mass;
  unsigned int ties, pad;
};
struct Row {
  Stats stats[kMaxSlices];
  Part part[kMaxSlices];
  unsigned long long mass[kBins];
  unsigned int count[kBins];
  unsigned int list[kListMax];
  unsigned int listed, arrived, pad[2];
};

struct Args {
  int64_t* out;
  const void* logits;
  int64_t row_stride;
  const float* uniform;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  Row* rows;
  int cols, slices, per;  // per: 16-byte chunks a slice
  int shift;              // weights in units of 2^-shift
};

__device__ const double kPow[16] = {  // 2^(-i / 16)
    0x1p+0,               0x1.ea4afa2a490dap-1, 0x1.d5818dcfba487p-1, 0x1.c199bdd85529cp-1,
    0x1.ae89f995ad3adp-1, 0x1.9c49182a3f090p-1, 0x1.8ace5422aa0dbp-1, 0x1.7a11473eb0187p-1,
    0x1.6a09e667f3bcdp-1, 0x1.5ab07dd485429p-1, 0x1.4bfdad5362a27p-1, 0x1.3dea64c123422p-1,
    0x1.306fe0a31b715p-1, 0x1.2387a6e756238p-1, 0x1.172b83c7d517bp-1, 0x1.0b5586cf9890fp-1};

// A row's settings and the measure of its weights.
struct Settings {
  float max, min;       // of the row; min of the values above -inf
  float t, p;
  double rate, least;   // 1 / T; min_p
  int k;
  bool greedy, by_k, by_p;
  float range, step;    // intervals: of d = max - x up to range, step a unit
};

// The order of the values as unsigned integers (0 stands for no value: NaN).
__device__ inline uint32_t key_of(float x) {
  if (x != x) return 0;
  const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.f);  // -0 as 0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ inline float value_of(uint32_t key) {
  return __builtin_bit_cast(float, key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}

// exp(-z) 2^shift to the nearest integer, z >= 0: 2^(-n / 16) from the table, n the
// nearest to 16 z / ln 2, and the series of the exponential for the rest (below
// 0.022, to the sixth power).
__device__ inline unsigned long long fixed_exp(double z, int shift, const double* pow16) {
#pragma clang fp contract(off)  // a value's weight is the same in every kernel
  const double y = z * 0x1.71547652b82fep+4;
  if (!(y < 16.0 * 64.0)) return 0;
  const double n = __builtin_rint(y);
  const double r = (n - y) * 0x1.62e42fefa39efp-5;
  double s = 1.0 / 720;
  s = __builtin_fma(s, r, 1.0 / 120);
  s = __builtin_fma(s, r, 1.0 / 24);
  s = __builtin_fma(s, r, 1.0 / 6);
  s = __builtin_fma(s, r, 0.5);
  s = __builtin_fma(s, r, 1.0);
  s = __builtin_fma(s, r, 1.0);
  const int i = (int)n;
  const double w = __builtin_amdgcn_ldexp(s * pow16[i & 15], shift - (i >> 4));
  return (unsigned long long)__builtin_rint(w);
}

// The weight of a value (a value at the largest: exactly 1).
__device__ inline unsigned long long weight_of(float x, const Settings& s, int shift,
                                               const double* pow16) {
#pragma clang fp contract(off)
  if (x == s.max) return 1ull << shift;
  return fixed_exp(((double)s.max - (double)x) * s.rate, shift, pow16);
}
// The weight if min-p keeps it, else 0.  The test is on w = exp(-z) itself: z in f64
// against -ln(min_p).
__device__ inline unsigned long long kept_weight(float x, const Settings& s, int shift,
                                                 const double* pow16) {
#pragma clang fp contract(off)
  if (x == s.max) return 1ull << shift;
  const double z = ((double)s.max - (double)x) * s.rate;
  return z <= s.least ? fixed_exp(z, shift, pow16) : 0;
}

// The interval of a value, -1 outside (weights there are 0).
__device__ inline int bin_of(float x, const Settings& s) {
#pragma clang fp contract(off)
  if (x == s.max) return 0;
  const float d = s.max - x;
  if (!(d <= s.range) || !(d < INFINITY)) return -1;
  return min((int)(d * s.step), kBins - 1);
}

__device__ inline Settings settings_of(const Args& a, int row) {
  Settings s;
  s.t = a.temperature ? a.temperature[row] : 1.f;
  s.k = a.top_k ? a.top_k[row] : 0;
  s.p = a.top_p ? a.top_p[row] : 1.f;
  const float m = a.min_p ? a.min_p[row] : 0.f;
  s.greedy = !(s.t > 0.f);
  s.by_k = !s.greedy && s.k > 0 && s.k < a.cols;
  s.by_p = !s.greedy && s.p < 1.f;
  s.rate = 1.0 / (double)s.t;
  s.least = m > 0.f ? -log((double)m) : (double)INFINITY;
  return s;
}

// The row's extremes from its slices (all threads; `red` of 2 floats).
__device__ inline void extremes(const Row& row, int slices, Settings& s, float* red) {
  if (threadIdx.x < 64) {
    float mx = -INFINITY, mn = INFINITY;
    if ((int)threadIdx.x < slices) {
      mx = row.stats[threadIdx.x].max;
      mn = row.stats[threadIdx.x].min;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      mx = fmaxf(mx, __shfl_xor(mx, o, 64));
      mn = fminf(mn, __shfl_xor(mn, o, 64));
    }
    if (threadIdx.x == 0) {
      red[0] = mx;
      red[1] = mn;
    }
  }
  __syncthreads();
  s.max = red[0];
  s.min = red[1];
  // Weights end at exp(-(shift + 1) ln 2), shift <= 62: d / T <= 44.
  s.range = fminf(44.f * s.t, s.max - s.min);
  s.step = s.range > 0.f ? kBins / s.range : 0.f;
}

// A row's memory in 16-byte chunks at 16-byte addresses; the elements of the first
// and the last that are not the row's read as NaN.
template <typename T>
struct Chunks {
  static constexpr int E = 16 / sizeof(T);
  const T* base;  // of the row
  int lead, cols, count;
  __device__ Chunks(const Args& a, int row) {
    base = (const T*)a.logits + (int64_t)row * a.row_stride;
    lead = (int)((uintptr_t)base % 16 / sizeof(T));
    cols = a.cols;
    count = (lead + cols + E - 1) / E;
  }
  __device__ int index(int chunk, int i) const { return chunk * E + i - lead; }
  __device__ void load(int chunk, float (&x)[E]) const {
    const int at = chunk * E - lead;
    if (at >= 0 && at + E <= cols) {
      const uint4 w = *reinterpret_cast<const uint4*>(base + at);
      const uint32_t d[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < E; ++i)
        x[i] = sizeof(T) == 4 ? __builtin_bit_cast(float, d[i])
                              : bf16_bits_to_f32((uint16_t)(d[i / 2] >> (16 * (i & 1))));
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i)
        x[i] = at + i >= 0 && at + i < cols ? Elem<T>::load(base + at + i) : __builtin_nanf("");
    }
  }
};
template <>
__device__ inline void Chunks<float>::load(int chunk, float (&x)[4]) const {
  const int at = chunk * E - lead;
  if (at >= 0 && at + E <= cols) {
    const float4 w = *reinterpret_cast<const float4*>(base + at);
    x[0] = w.x;
    x[1] = w.y;
    x[2] = w.z;
    x[3] = w.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      x[i] = at + i >= 0 && at + i < cols ? base[at + i] : __builtin_nanf("");
  }
}

// f(value) for each value of this workgroup's slice.
template <typename T, typename F>
__device__ inline void each_of_slice(const Args& a, int row, int slice, F f) {
  const Chunks<T> c(a, row);
  const int end = min(c.count, (slice + 1) * a.per);
  for (int ch = slice * a.per + threadIdx.x; ch < end; ch += kThreads) {
    float x[Chunks<T>::E];
    c.load(ch, x);
#pragma unroll
    for (int i = 0; i < Chunks<T>::E; ++i) f(x[i], c.index(ch, i));
  }
}

// The sum of the values of the threads before this one; total of all.
template <typename V>
__device__ inline V scan_before(V v, V* red, V& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  V incl = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const V up = __shfl_up(incl, o, 64);
    if (lane >= o) incl += up;
  }
  __syncthreads();
  if (lane == 63) red[wave] = incl;
  __syncthreads();
  V before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    if (w < wave) before += red[w];
    total += red[w];
  }
  return before + incl - v;
}

// Where the running sum of n = kBins entries first reaches `want` (1 or more): its
// index and the sum before it; index kBins where it does not.  All threads.
struct Cross {
  int at;
  unsigned long long before;
};
template <typename V>
__device__ inline Cross cross(const V* h, unsigned long long want, unsigned long long* red,
                              Cross* found, unsigned long long& total) {
  constexpr int N = kBins / kThreads;
  V v[N];
  unsigned long long sum = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = h[threadIdx.x * N + i];
    sum += v[i];
  }
  unsigned long long run = scan_before(sum, red, total);
  if (threadIdx.x == 0) *found = Cross{kBins, total};
  __syncthreads();
  if (run < want && want <= run + sum) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (run < want && want <= run + v[i]) *found = Cross{(int)threadIdx.x * N + i, run};
      run += v[i];
    }
  }
  __syncthreads();
  const Cross c = *found;
  __syncthreads();
  return c;
}

// ceil(f w) for 0 < f < 1, at least 1; floor(f w), below w.  Exact: f has 24 bits.
__device__ inline unsigned long long share_up(float f, unsigned long long w) {
  if (!(f > 0.f)) return 1;
  const uint32_t u = __builtin_bit_cast(uint32_t, f);
  const int e = (int)(u >> 23);  // f = m 2^(e - 150)
  const unsigned long long m = e ? (u & 0x7FFFFF) | 0x800000 : u & 0x7FFFFF;
  const int down = 150 - (e ? e : 1);  // 24 and more
  const unsigned __int128 x = (unsigned __int128)m * w;
  if (down >= 100) return 1;
  const unsigned long long q = (unsigned long long)(x >> down);
  const bool rest = (x & (((unsigned __int128)1 << down) - 1)) != 0;
  return max(q + (rest ? 1 : 0), 1ull);
}
__device__ inline unsigned long long share_down(float f, unsigned long long w) {
  if (!(f > 0.f)) return 0;
  if (f >= 1.f) return w - 1;
  const uint32_t u = __builtin_bit_cast(uint32_t, f);
  const int e = (int)(u >> 23);
  const unsigned long long m = e ? (u & 0x7FFFFF) | 0x800000 : u & 0x7FFFFF;
  const int down = 150 - (e ? e : 1);
  if (down >= 100) return 0;
  return (unsigned long long)(((unsigned __int128)m * w) >> down);
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_max_kernel(const Args a) {
  const int row = blockIdx.y, slice = blockIdx.x;
  Row& r = a.rows[row];
  float mx = -INFINITY, mn = INFINITY;
  int at = INT_MAX;
  each_of_slice<T>(a, row, slice, [&](float x, int i) {
    if (x > mx) {
      mx = x;
      at = i;
    }
    if (x > -INFINITY) mn = fminf(mn, x);
  });
  // what the next kernels add to
  if (a.top_k || a.top_p) {
    for (int b = slice * kThreads + threadIdx.x; b < kBins; b += a.slices * kThreads) {
      r.mass[b] = 0;
      r.count[b] = 0;
    }
  }
  if (slice == 0 && threadIdx.x == 0) r.listed = r.arrived = 0;
  __shared__ Stats red[kThreads / 64];
  auto join = [&](float ox, float on, int oat) {
    if (ox > mx || (ox == mx && oat < at)) {
      mx = ox;
      at = oat;
    }
    mn = fminf(mn, on);
  };
#pragma unroll
  for (int o = 32; o > 0; o >>= 1)
    join(__shfl_xor(mx, o, 64), __shfl_xor(mn, o, 64), __shfl_xor(at, o, 64));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = Stats{mx, mn, at, 0};
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kThreads / 64; ++w) join(red[w].max, red[w].min, red[w].at);
    r.stats[slice] = Stats{mx, mn, at, 0};
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_hist_kernel(const Args a) {
  const int row = blockIdx.y, slice = blockIdx.x;
  Settings s = settings_of(a, row);
  if (!s.by_k && !s.by_p) return;
  __shared__ unsigned long long mass[kBins];
  __shared__ unsigned int count[kBins];
  __shared__ double pow16[16];
  __shared__ float red[2];
  Row& r = a.rows[row];
  for (int b = threadIdx.x; b < kBins; b += kThreads) {
    mass[b] = 0;
    count[b] = 0;
  }
  if (threadIdx.x < 16) pow16[threadIdx.x] = kPow[threadIdx.x];
  extremes(r, a.slices, s, red);
  each_of_slice<T>(a, row, slice, [&](float x, int) {
    const int b = bin_of(x, s);
    if (b < 0) return;
    if (s.by_k) atomicAdd(&count[b], 1u);
    if (s.by_p) atomicAdd(&mass[b], weight_of(x, s, a.shift, pow16));
  });
  __syncthreads();
  for (int b = threadIdx.x; b < kBins; b += kThreads) {
    if (count[b]) atomicAdd(&r.count[b], count[b]);
    if (mass[b]) atomicAdd(&r.mass[b], mass[b]);
  }
}

// Where the thresholds lie, as far as the intervals tell: top-k's is in interval kb
// (kBins: none, fewer values than k), before it `above` values.  All threads.
struct Found {
  int kb;
  unsigned long long above;
};
__device__ inline Found find_k(const Row& r, const Settings& s, unsigned long long* red,
                               Cross* found) {
  if (!s.by_k) return Found{kBins, 0};
  unsigned long long total;
  const Cross c = cross(r.count, (unsigned long long)s.k, red, found, total);
  return Found{c.at, c.before};
}

// Sum of the intervals' weights before interval b.
__device__ inline unsigned long long mass_before(const Row& r, int b, unsigned long long* red) {
  unsigned long long v = 0, total;
  for (int i = threadIdx.x; i < b; i += kThreads) v += r.mass[i];
  scan_before(v, red, total);
  return total;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_pick_kernel(const Args a) {
  const int row = blockIdx.y, slice = blockIdx.x;
  Settings s = settings_of(a, row);
  if (!s.by_k && !s.by_p) return;
  __shared__ unsigned long long red[kThreads / 64];
  __shared__ Cross found;
  __shared__ float ext[2];
  Row& r = a.rows[row];
  extremes(r, a.slices, s, ext);
  const Found f = find_k(r, s, red, &found);
  int lo = kBins, hi = -1;  // top-p's interval is one of these
  if (s.by_p) {
    // the weight that top-k leaves lies between that before its interval and that
    // with all of it
    const unsigned long long least = mass_before(r, f.kb, red);
    const unsigned long long most = least + (f.kb < kBins ? r.mass[f.kb] : 0);
    unsigned long long total;
    lo = min(cross(r.mass, share_up(s.p, least), red, &found, total).at, f.kb);
    hi = min(cross(r.mass, share_up(s.p, most), red, &found, total).at, f.kb);
  }
  each_of_slice<T>(a, row, slice, [&](float x, int) {
    const int b = bin_of(x, s);
    if (b >= 0 && (b == f.kb || (b >= lo && b <= hi))) {
      const unsigned int at = atomicAdd(&r.listed, 1u);
      if (at < kListMax) r.list[at] = key_of(x);
    }
  });
}

// The largest value v of the interval `bin` so that the values >= v weigh `want` or
// more (each 1, or its weight), and the sum of those above it.  Rounds of kDigits
// bits from the highest in which the interval's keys differ.  `each(f)` calls f(key)
// for the candidates.
struct Select {
  unsigned long long hist[kBins];
  unsigned long long red[kThreads / 64];
  Cross found;
  uint32_t lo, hi;
};
struct Threshold {
  uint32_t key;
  unsigned long long above;
};
template <typename Each, typename Weight>
__device__ inline Threshold select(Each each, Weight weight, unsigned long long want, Select& l) {
  if (threadIdx.x == 0) {
    l.lo = 0xFFFFFFFFu;
    l.hi = 0;
  }
  __syncthreads();
  uint32_t lo = 0xFFFFFFFFu, hi = 0;
  each([&](uint32_t key) {
    lo = min(lo, key);
    hi = max(hi, key);
  });
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    lo = min(lo, (uint32_t)__shfl_xor((int)lo, o, 64));
    hi = max(hi, (uint32_t)__shfl_xor((int)hi, o, 64));
  }
  if ((threadIdx.x & 63) == 0) {
    atomicMin(&l.lo, lo);
    atomicMax(&l.hi, hi);
  }
  __syncthreads();
  lo = l.lo;
  hi = l.hi;
  int left = lo == hi ? 0 : 32 - __builtin_clz(lo ^ hi);  // bits still open
  Threshold t{hi, 0};
  while (left > 0) {
    const int shift = max(left - kDigits, 0);
    const uint32_t digits = (1u << (left - shift)) - 1;
    __syncthreads();
    for (int b = threadIdx.x; b < kBins; b += kThreads) l.hist[b] = 0;
    __syncthreads();
    each([&](uint32_t key) {
      if (left == 32 || (key >> left) == (t.key >> left))
        atomicAdd(&l.hist[digits - ((key >> shift) & digits)], weight(key));
    });
    __syncthreads();
    unsigned long long total;
    const Cross c = cross(l.hist, want, l.red, &l.found, total);
    const uint32_t digit = c.at < kBins ? digits - c.at : 0;  // (always found: want <= the sum)
    t.key = (t.key & ~((digits << shift) | ((1u << shift) - 1))) | (digit << shift);
    if (c.at < kBins) {
      t.above += c.before;
      want -= c.before;
    }
    left = shift;
  }
  __syncthreads();
  return t;
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_draw_kernel(const Args a) {
  const int row = blockIdx.y, slice = blockIdx.x;
  Settings s = settings_of(a, row);
  Row& r = a.rows[row];
  __shared__ float ext[2];
  __shared__ double pow16[16];
  __shared__ Select l;
  __shared__ unsigned int last;
  extremes(r, a.slices, s, ext);
  if (s.greedy || s.max == -INFINITY) {
    // the first largest; 0 where nothing is above -inf
    if (slice == 0 && threadIdx.x == 0) {
      int at = INT_MAX;
      for (int i = 0; i < a.slices; ++i)
        if (r.stats[i].max == s.max) at = min(at, r.stats[i].at);
      a.out[row] = s.max == -INFINITY || at == INT_MAX ? 0 : at;
    }
    return;
  }
  if (threadIdx.x < 16) pow16[threadIdx.x] = kPow[threadIdx.x];
  __syncthreads();
  // Kept: the values above `cut` and the first `ties` at it.
  uint32_t cut = 0;
  unsigned long long ties = 0;
  if (s.by_k || s.by_p) {
    // the values of interval b, from the list or, where that overflowed, the row
    const unsigned int listed = r.listed;
    auto values = [&](int b) {
      return [&, b](auto f) {
        if (listed <= kListMax) {
          for (unsigned int i = threadIdx.x; i < listed; i += kThreads) {
            const uint32_t key = r.list[i];
            if (bin_of(value_of(key), s) == b) f(key);
          }
        } else {
          const Chunks<T> c(a, row);
          for (int ch = threadIdx.x; ch < c.count; ch += kThreads) {
            float x[Chunks<T>::E];
            c.load(ch, x);
#pragma unroll
            for (int i = 0; i < Chunks<T>::E; ++i)
              if (bin_of(x[i], s) == b) f(key_of(x[i]));
          }
        }
      };
    };
    auto weight = [&](uint32_t key) { return weight_of(value_of(key), s, a.shift, pow16); };
    const Found f = find_k(r, s, l.red, &l.found);
    unsigned long long total = 0;
    if (f.kb < kBins) {
      const unsigned long long want = (unsigned long long)s.k - f.above;
      const Threshold t = select(values(f.kb), [](uint32_t) { return 1ull; }, want, l);
      cut = t.key;
      ties = want - t.above;
      if (s.by_p) {
        unsigned long long mine = 0, sum;
        values(f.kb)([&](uint32_t key) { mine += key > cut ? weight(key) : 0; });
        scan_before(mine, l.red, sum);
        total = mass_before(r, f.kb, l.red) + sum + ties * weight(cut);
      }
    } else if (s.by_p) {
      total = mass_before(r, kBins, l.red);
    }
    if (s.by_p) {
      const unsigned long long want = share_up(s.p, total);
      unsigned long long all;
      const Cross c = cross(r.mass, want, l.red, &l.found, all);
      const Threshold t = select(values(c.at), weight, want - c.before, l);
      cut = t.key;
      const unsigned long long w = max(weight(cut), 1ull);
      ties = (want - c.before - t.above + w - 1) / w;
    }
  }
  // The slice's share.
  unsigned long long mass = 0;
  unsigned int equal = 0;
  each_of_slice<T>(a, row, slice, [&](float x, int) {
    const uint32_t key = key_of(x);
    if (key > cut) mass += kept_weight(x, s, a.shift, pow16);
    equal += cut && key == cut;
  });
  unsigned long long mass_all;
  unsigned int equal_all;
  scan_before(mass, l.red, mass_all);
  scan_before(equal, (unsigned int*)&l.hist[0], equal_all);
  // The last workgroup of the row to get here has every slice's share: written
  // through by agent-scope stores before a releasing count, read behind an acquiring
  // fence.
  if (threadIdx.x == 0) {
    __hip_atomic_store(&r.part[slice].mass, mass_all, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(&r.part[slice].ties, equal_all, __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
    last = __hip_atomic_fetch_add(&r.arrived, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) ==
           (unsigned int)a.slices - 1;
  }
  __syncthreads();
  if (!last) return;
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
  const unsigned long long even = cut ? kept_weight(value_of(cut), s, a.shift, pow16) : 0;
  unsigned long long part = 0;
  unsigned int eq = 0;
  if ((int)threadIdx.x < a.slices) {
    part = __hip_atomic_load(&r.part[threadIdx.x].mass, __ATOMIC_RELAXED,
                             __HIP_MEMORY_SCOPE_AGENT);
    eq = __hip_atomic_load(&r.part[threadIdx.x].ties, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  // of n tokens at the threshold with `before` of them in front, those that are kept
  auto tied = [&](unsigned long long before, unsigned long long n) -> unsigned long long {
    return before >= ties ? 0 : min(n, ties - before);
  };
  unsigned long long all, dummy;
  unsigned long long eq_before = scan_before((unsigned long long)eq, l.red, dummy);
  part += tied(eq_before, eq) * even;
  const unsigned long long part_before = scan_before(part, l.red, all);
  // the first kept token with a running sum above uniform * the total
  const unsigned long long target = share_down(a.uniform[row], all);
  __shared__ int in_slice;
  __shared__ unsigned long long from, eq_from;
  __syncthreads();
  if (part_before <= target && target < part_before + part) {
    in_slice = threadIdx.x;
    from = part_before;
    eq_from = eq_before;
  }
  __syncthreads();
  // its slice, each thread a run of chunks
  const Chunks<T> c(a, row);
  const int begin = in_slice * a.per, end = min(c.count, begin + a.per);
  const int run = (end - begin + kThreads - 1) / kThreads;
  const int c0 = min(end, begin + (int)threadIdx.x * run), c1 = min(end, c0 + run);
  mass = 0;
  equal = 0;
  for (int ch = c0; ch < c1; ++ch) {
    float x[Chunks<T>::E];
    c.load(ch, x);
#pragma unroll
    for (int i = 0; i < Chunks<T>::E; ++i) {
      const uint32_t key = key_of(x[i]);
      if (key > cut) mass += kept_weight(x[i], s, a.shift, pow16);
      equal += cut && key == cut;
    }
  }
  eq_before = eq_from + scan_before((unsigned long long)equal, l.red, dummy);
  mass += tied(eq_before, equal) * even;
  unsigned long long sum = from + scan_before(mass, l.red, dummy);
  if (sum <= target && target < sum + mass) {
    bool done = false;
    for (int ch = c0; ch < c1 && !done; ++ch) {
      float x[Chunks<T>::E];
      c.load(ch, x);
      for (int i = 0; i < Chunks<T>::E && !done; ++i) {
        const uint32_t key = key_of(x[i]);
        if (key > cut) {
          sum += kept_weight(x[i], s, a.shift, pow16);
        } else if (cut && key == cut) {
          if (eq_before < ties) sum += even;
          ++eq_before;
        }
        if (sum > target) {
          a.out[row] = c.index(ch, i);
          done = true;
        }
      }
    }
  }
}

int slices_of(int rows, int cols, int es) {
  const int chunks = (int)(((int64_t)cols * es + 15) / 16) + 1;
  const int most = std::max(1, std::min(kMaxSlices, chunks / kThreads));
  return std::max(1, std::min(most, (512 + rows - 1) / std::max(rows, 1)));
}

}  // namespace
}  // namespace pa

using namespace pa;

extern "C" size_t pa_sample_workspace_size(int32_t rows) {
  return rows > 0 ? (size_t)rows * sizeof(Row) : 0;
}

extern "C" int32_t pa_sample(int64_t* out, const void* logits, const float* uniform,
                             const float* temperature, const int32_t* top_k, const float* top_p,
                             const float* min_p, int32_t rows, int32_t cols, int64_t row_stride,
                             void* workspace, size_t workspace_bytes, int32_t dtype,
                             pa_stream_t stream) {
  clear_error();
  PA_REQUIRE(dtype_ok(dtype), PA_ERR_INVALID_ARG, "pa_sample: unknown dtype %d", dtype);
  PA_REQUIRE(rows >= 0 && cols > 0, PA_ERR_INVALID_ARG, "pa_sample: bad sizes");
  if (row_stride == 0) row_stride = cols;
  PA_REQUIRE(row_stride >= cols, PA_ERR_INVALID_ARG, "pa_sample: row stride %lld below cols %d",
             (long long)row_stride, cols);
  PA_REQUIRE(cols <= 1 << 22 && rows <= 65535, PA_ERR_UNSUPPORTED,
             "pa_sample: %d rows of %d (at most 65535 of 2^22)", rows, cols);
  if (rows == 0) return PA_OK;
  PA_REQUIRE(out && logits && uniform, PA_ERR_INVALID_ARG, "pa_sample: null pointer");
  const int es = dtype == PA_DTYPE_BF16 ? 2 : 4;
  PA_REQUIRE((uintptr_t)logits % es == 0, PA_ERR_INVALID_ARG, "pa_sample: logits not aligned");
  const size_t need = pa_sample_workspace_size(rows);
  PA_REQUIRE(workspace && workspace_bytes >= need && (uintptr_t)workspace % 16 == 0,
             PA_ERR_WORKSPACE, "pa_sample: workspace of %zu bytes (16-byte aligned) needed, %zu given",
             need, workspace ? workspace_bytes : 0);
  const int slices = slices_of(rows, cols, es);
  const int chunks = (int)(((int64_t)cols * es + 15) / 16) + 1;
  int bits = 1;
  while ((1 << bits) < cols) ++bits;
  const Args a{out, logits, row_stride, uniform, temperature, top_k, top_p, min_p, (Row*)workspace,
               cols, slices, (chunks + slices - 1) / slices, 62 - bits};
  const dim3 grid(slices, rows);
  hipStream_t s = (hipStream_t)stream;
#define PA_LAUNCH_SAMPLE(KERNEL)                                                   \
  (dtype == PA_DTYPE_BF16 ? KERNEL<uint16_t><<<grid, kThreads, 0, s>>>(a)          \
                          : KERNEL<float><<<grid, kThreads, 0, s>>>(a))
  PA_LAUNCH_SAMPLE(sample_max_kernel);
  if (top_k || top_p) {
    PA_LAUNCH_SAMPLE(sample_hist_kernel);
    PA_LAUNCH_SAMPLE(sample_pick_kernel);
  }
  PA_LAUNCH_SAMPLE(sample_draw_kernel);
#undef PA_LAUNCH_SAMPLE
  return check_launch("pa_sample");
}
