// Drawing a token from each row of logits (pa_sample): temperature, top-k, top-p
// and min-p, one uniform number a row.
//
// With M the row's largest logit a token weighs w = exp((x - M) / T).  Weights are
// formed in f64 (an error of about 2^-48) and summed as integers of 2^-shift (51
// bits, 44 for vocabularies up to 2^18): a sum does not depend on its order, so equal
// calls draw equal tokens, and a border between two tokens lies where the exact sums
// have it but for a few 2^-44 of the row's total.  (Sums of 10^5 f32 weights would
// move the borders by more than many tokens' weights.)
//
// Nothing is sorted.  What top-k and top-p keep of a row is all above a threshold
// value and the first `ties` tokens equal to it:
//   1  sample_max_kernel    the row's largest and least logit
//   2  sample_hist_kernel   counts and weights of 512 equal intervals of the logits
//   3  sample_pick_kernel   the values in the intervals in which the thresholds lie, and
//                           (in the row's last workgroup) the thresholds among them, by
//                           radix selection
//   4  sample_draw_kernel   the kept weight of every wavefront's run of tokens and, in
//                           the row's last workgroup, the token
// 2 and 3 only where the call gives top_k or top_p; rows that do not use them pass
// through.  Each kernel reads the logits once, in workgroups of a slice of a row.  Rows
// of few tokens, and many rows, take all steps in one launch, a workgroup a row
// (sample_row_kernel), with the same results.
//
// Bound by the launches and what each does once a row, one thing after the other, for
// few rows: 1 x 151936 bf16 29 us, 32 rows 43; by f64 weights, formed twice, for many:
// 253 x 50257 f32 80 us, of which the first kernel 11, at a copy's rate.
#include <algorithm>
#include <climits>

#include "pa_common.hpp"
#include "pa_internal.hpp"
#include "../../include/pa_dense.h"

namespace pa {
namespace {

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
constexpr int kBins = 512;
constexpr int kWorkgroups = 1024;  // of a launch where its rows allow: four a CU
constexpr int kMaxSlices = 32;
constexpr int kLaneParts = kMaxSlices * kThreads / 64 / 64;  // of a row, to a wavefront
constexpr int kListMax = 4096;  // values that step 3 collects; more are read from the row again
constexpr int kDigits = 9;      // bits a round of the selection

// What a row has in the workspace.
struct Stats {  // of a slice
  float max, min;
  int at;  // of the first largest
  int pad;
};
struct Part {  // of a wavefront's run: what is kept of it
  unsigned long long mass;
  unsigned int ties, pad;
};
struct Row {
  Stats stats[kMaxSlices];
  unsigned long long mass[kBins];
  unsigned int count[kBins];
  uint32_t cut;  // kept: the values above `cut` and the first `ties` at it
  unsigned long long ties;
  unsigned int listed, arrived[2];
};
struct RowSpace : Row {
  uint32_t list[kListMax];
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
  RowSpace* rows;
  Part* parts;  // of (row, slice, wavefront)
  int cols, slices;
  int shift;  // weights in units of 2^-shift, at most 51
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
  double top;           // max
  double rate, least;   // of y = 16 (max - x) / (T ln 2): the factor, and min-p's bound
  int k;
  bool greedy, by_k, by_p;
  // intervals: of d = (max - x) / 2, which is a float where max - x is not, up to range,
  // step a unit
  float half, range, step;  // half: max / 2
  __device__ bool narrows() const { return (by_k || by_p) && max > -INFINITY; }
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

// The weight of a value in units of 2^-shift: exp(-z), z = (max - x) / T, to the nearest
// integer.  y = 16 z / ln 2 = n - f with n whole and |f| <= 1/2: exp(-z) =
// 2^(-n / 16) 2^(f / 16), the one from the table, the other the series of the
// exponential to the sixth power (its rest below 2^-51).  Both roundings to integers
// are additions of a number whose unit is 1 in f64, so shift is at most 51.
constexpr double kUnit = 0x1.8p+52, kWhole = 0x1p+52;
__device__ inline unsigned long long weigh(double y, int shift, const double* pow16) {
#pragma clang fp contract(off)  // a value's weight is the same in every kernel
  const double m = y + kUnit;
  const double f = (m - kUnit) - y;
  const uint32_t n = (uint32_t)__builtin_bit_cast(unsigned long long, m);
  constexpr double c = 0x1.62e42fefa39efp-5;  // ln 2 / 16
  double s = c * c * c * c * c * c / 720;
  s = __builtin_fma(s, f, c * c * c * c * c / 120);
  s = __builtin_fma(s, f, c * c * c * c / 24);
  s = __builtin_fma(s, f, c * c * c / 6);
  s = __builtin_fma(s, f, c * c / 2);
  s = __builtin_fma(s, f, c);
  s = __builtin_fma(s, f, 1.0);
  const unsigned long long p = __builtin_bit_cast(unsigned long long, pow16[n & 15]) +
                               ((unsigned long long)(uint32_t)(shift - (int)(n >> 4)) << 52);
  const double w = __builtin_fma(s, __builtin_bit_cast(double, p), kWhole);
  return y < 16.0 * 64.0 ? __builtin_bit_cast(unsigned long long, w) & 0xFFFFFFFFFFFFFull : 0;
}
// (a value at the largest, which may be infinite: exactly 1)
__device__ inline unsigned long long weight_of(float x, const Settings& s, int shift,
                                               const double* pow16) {
#pragma clang fp contract(off)
  const unsigned long long w = weigh((s.top - (double)x) * s.rate, shift, pow16);
  return x == s.max ? 1ull << shift : w;
}
// The weight if min-p keeps it, else 0.  The test is on exp(-z) itself: z in f64
// against -ln(min_p).
__device__ inline unsigned long long kept_weight(float x, const Settings& s, int shift,
                                                 const double* pow16) {
#pragma clang fp contract(off)
  const double y = (s.top - (double)x) * s.rate;
  const unsigned long long w = y <= s.least ? weigh(y, shift, pow16) : 0;
  return x == s.max ? 1ull << shift : w;
}

// The interval of a value, -1 outside (weights there are 0).
__device__ inline int bin_of(float x, const Settings& s) {
#pragma clang fp contract(off)
  if (x == s.max) return 0;
  const float d = __builtin_fmaf(x, -0.5f, s.half);
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
  constexpr double k = 0x1.71547652b82fep+4;  // 16 / ln 2
  s.rate = k / (double)s.t;
  s.least = m > 0.f ? -log((double)m) * k : (double)INFINITY;
  return s;
}

// What a wavefront's lanes give, joined by f: `none` for lanes that give nothing.
template <int CTRL, int ROWS>
__device__ inline uint32_t dpp(uint32_t v, uint32_t none = 0) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)none, (int)v, CTRL, ROWS, 0xF, false);
}
__device__ inline uint32_t lane_of(uint32_t v, int lane) {
  return (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}
template <typename F>
__device__ inline uint32_t wave_join(uint32_t v, uint32_t none, F f) {
  v = f(v, dpp<0x111, 0xF>(v, none));  // within 16 lanes, with 1, 2, 4 and 8 before
  v = f(v, dpp<0x112, 0xF>(v, none));
  v = f(v, dpp<0x114, 0xF>(v, none));
  v = f(v, dpp<0x118, 0xF>(v, none));
  v = f(v, dpp<0x142, 0xA>(v, none));  // the first and third sixteen's, with the next
  v = f(v, dpp<0x143, 0xC>(v, none));  // the first half's, with the second
  return lane_of(v, 63);
}

// The row's settings and, from its slices, extremes: formed by the first wavefront (a
// CU's wavefronts share its issue slots), for all behind the next barrier.
__device__ inline void prepare(const Args& a, int row, const Row& r, Settings& to) {
  if (threadIdx.x >= 64) return;
  Settings s = settings_of(a, row);
  const Stats& mine = r.stats[min((int)threadIdx.x, a.slices - 1)];
  auto f32 = [](uint32_t v) { return __builtin_bit_cast(float, v); };
  auto u32 = [](float v) { return __builtin_bit_cast(uint32_t, v); };
  s.max = f32(wave_join(u32(mine.max), u32(-INFINITY), [&](uint32_t v, uint32_t w) {
    return u32(fmaxf(f32(v), f32(w)));
  }));
  s.min = f32(wave_join(u32(mine.min), u32(INFINITY), [&](uint32_t v, uint32_t w) {
    return u32(fminf(f32(v), f32(w)));
  }));
  s.top = (double)s.max;
  // Weights end at exp(-(shift + 1) ln 2), shift <= 51: 2 d / T <= 36.1.
  s.half = 0.5f * s.max;
  s.range = fminf(18.5f * s.t, __builtin_fmaf(s.min, -0.5f, s.half));
  s.step = s.range > 0.f ? kBins / s.range : 0.f;
  if (threadIdx.x == 0) to = s;
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

// The run of chunks of part `part` of a row (a wavefront's: slice by slice, wavefront by
// wavefront), lane by lane in turn: whole 64s, evenly.  The first chunks are on their
// way from construction on, the next while these are used.
template <typename T>
struct Run {
  static constexpr int E = Chunks<T>::E;
  Chunks<T> c;
  int at, end;
  float next[E];
  __device__ Run(const Args& a, int row, int part) : c(a, row) {
    const uint32_t units = (c.count + 63) / 64, parts = a.slices * kWaves;  // 2^16 x 2^8
    at = (int)(units * part / parts) * 64 + (threadIdx.x & 63);
    end = min((int)(units * (part + 1) / parts) * 64, c.count);
    if (at < end) c.load(at, next);
  }
  // f(x, chunk) for each chunk's values
  template <typename F>
  __device__ void each(F f) {
    while (at < end) {
      float x[E];
#pragma unroll
      for (int i = 0; i < E; ++i) x[i] = next[i];
      const int now = at;
      at += 64;
      if (at < end) c.load(at, next);
      f(x, now);
    }
  }
};

// The running sums of a wavefront's values, lane by lane (the last lane's: the total),
// of 64 and 32 bits.
template <int CTRL, int ROWS>
__device__ inline unsigned long long dpp(unsigned long long v) {
  return (unsigned long long)dpp<CTRL, ROWS>((uint32_t)(v >> 32)) << 32 |
         dpp<CTRL, ROWS>((uint32_t)v);
}
__device__ inline unsigned long long lane_of(unsigned long long v, int lane) {
  return (unsigned long long)lane_of((uint32_t)(v >> 32), lane) << 32 |
         lane_of((uint32_t)v, lane);
}
template <typename V>
__device__ inline V wave_scan(V v) {
  v += dpp<0x111, 0xF>(v);  // within 16 lanes, from 1, 2, 4 and 8 before
  v += dpp<0x112, 0xF>(v);
  v += dpp<0x114, 0xF>(v);
  v += dpp<0x118, 0xF>(v);
  v += dpp<0x142, 0xA>(v);  // the first and third sixteen's total, to the next
  v += dpp<0x143, 0xC>(v);  // the first half's, to the second
  return v;
}
template <typename V>
__device__ inline V wave_sum(V v) {
  return lane_of(wave_scan(v), 63);
}
// Where the running sum of the kBins entries at h first reaches `want` (1 or more): its
// index and the sum before it; index kBins and the total where it does not.  By a
// wavefront; a lane has 8 entries in turn.
constexpr int kLaneBins = kBins / 64;
struct Cross {
  int at;
  unsigned long long before;
};
template <typename V>
struct Entries {
  V v[kLaneBins];
  unsigned long long sum, before, total;
  __device__ explicit Entries(const V* h) {
    const int lane = threadIdx.x & 63;
    sum = 0;
#pragma unroll
    for (int i = 0; i < kLaneBins; ++i) {
      v[i] = h[lane * kLaneBins + i];
      sum += v[i];
    }
    before = wave_scan(sum);
    total = lane_of(before, 63);
    before -= sum;
  }
  __device__ Cross cross(unsigned long long want) const {
    const unsigned long long here =
        __builtin_amdgcn_ballot_w64(before < want && want <= before + sum);
    if (here == 0) return Cross{kBins, total};
    const int lane = __builtin_ctzll(here);
    unsigned long long run = before, from = 0;
    int at = 0;
#pragma unroll
    for (int i = 0; i < kLaneBins; ++i) {
      if (run < want && want <= run + v[i]) {
        at = i;
        from = run;
      }
      run += v[i];
    }
    return Cross{lane * kLaneBins + (int)lane_of((unsigned int)at, lane), lane_of(from, lane)};
  }
  // the sum before entry b, and with it
  __device__ unsigned long long upto(int b, bool with) const {
    unsigned long long s = 0;
#pragma unroll
    for (int i = 0; i < kLaneBins; ++i) {
      const int at = (threadIdx.x & 63) * kLaneBins + i;
      if (at < b || (with && at == b)) s += v[i];
    }
    return wave_sum(s);
  }
};

// The sum over all threads (with two barriers).
__device__ inline unsigned long long sum_of(unsigned long long v, unsigned long long* red) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return wave_sum((threadIdx.x & 63) < kWaves ? red[threadIdx.x & 63] : 0ull);
}

// What wavefronts of a row leave for its last workgroup is written and read as
// agent-scope atomics, which pass by the XCDs' L2s, and every wavefront waits until its
// own are done before the barrier in front of the count.  (So nothing lies dirty in an
// L2 and nothing stale there: releasing and acquiring fences of whole L2s, by every
// wavefront, took 70 us for 512 workgroups.)
template <typename V>
__device__ inline void put(V* p, V v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename V>
__device__ inline V get(const V* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// Whether this is the last of the row's workgroups to get here: to the first wavefront;
// the others get false.
__device__ inline bool last_of_row(unsigned int* arrived, int slices) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x >= 64) return false;
  unsigned int before = 0;
  if (threadIdx.x == 0)
    before = __hip_atomic_fetch_add(arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return lane_of(before, 0) == (unsigned int)slices - 1;
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

// Step 1 for a slice.
template <typename T>
__device__ inline void max_of_slice(const Args& a, int row, int slice, Row& r) {
  const int wave = threadIdx.x >> 6;
  Run<T> run(a, row, slice * kWaves + wave);
  // what the next kernels add to
  if (a.top_k || a.top_p) {
    for (int b = slice * kThreads + threadIdx.x; b < kBins; b += a.slices * kThreads) {
      r.mass[b] = 0;
      r.count[b] = 0;
    }
  }
  if (slice == 0 && threadIdx.x == 0) r.listed = r.arrived[0] = r.arrived[1] = 0;
  float mx = -INFINITY, mn = INFINITY;
  int at = INT_MAX;
  run.each([&](const auto& x, int chunk) {
#pragma unroll
    for (int i = 0; i < Chunks<T>::E; ++i) {
      if (x[i] > mx) {
        mx = x[i];
        at = run.c.index(chunk, i);
      }
      if (x[i] > -INFINITY) mn = fminf(mn, x[i]);
    }
  });
  __shared__ Stats red[kWaves];
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
  if ((threadIdx.x & 63) == 0) red[wave] = Stats{mx, mn, at, 0};
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kWaves; ++w) join(red[w].max, red[w].min, red[w].at);
    r.stats[slice] = Stats{mx, mn, at, 0};
  }
}
template <typename T>
__global__ __launch_bounds__(kThreads) void sample_max_kernel(const Args a) {
  max_of_slice<T>(a, blockIdx.y, blockIdx.x, a.rows[blockIdx.y]);
}

// Step 2 for a slice, into arrays in LDS (cleared; a barrier behind).
template <typename T>
__device__ inline void hist_of_slice(const Args& a, const Settings& s, Run<T>& run,
                                     unsigned long long* mass, unsigned int* count,
                                     const double* pow16) {
  run.each([&](const auto& x, int) {
#pragma unroll
    for (int i = 0; i < Chunks<T>::E; ++i) {
      const int b = bin_of(x[i], s);
      if (b < 0) continue;
      if (s.by_k) atomicAdd(&count[b], 1u);
      if (s.by_p) atomicAdd(&mass[b], weight_of(x[i], s, a.shift, pow16));
    }
  });
  __syncthreads();
}
template <typename T>
__global__ __launch_bounds__(kThreads) void sample_hist_kernel(const Args a) {
  const int row = blockIdx.y, slice = blockIdx.x, wave = threadIdx.x >> 6;
  __shared__ Settings settings;
  __shared__ unsigned long long mass[kBins];
  __shared__ unsigned int count[kBins];
  __shared__ double pow16[16];
  Row& r = a.rows[row];
  Run<T> run(a, row, slice * kWaves + wave);
  for (int b = threadIdx.x; b < kBins; b += kThreads) {
    mass[b] = 0;
    count[b] = 0;
  }
  if (threadIdx.x < 16) pow16[threadIdx.x] = kPow[threadIdx.x];
  prepare(a, row, r, settings);
  __syncthreads();
  const Settings s = settings;
  if (!s.narrows()) return;
  hist_of_slice<T>(a, s, run, mass, count, pow16);
  for (int b = threadIdx.x; b < kBins; b += kThreads) {
    if (count[b]) atomicAdd(&r.count[b], count[b]);
    if (mass[b]) atomicAdd(&r.mass[b], mass[b]);
  }
}

// The largest value v among the candidates so that those >= v weigh `want` or more
// (each 1, or its weight); `want` becomes what those above it leave of it.  Rounds of
// up to kDigits bits from the highest in which the keys differ to the lowest (values of
// 16 bits need few).  `each(f)` calls f(key) for a thread's candidates.  A round's
// histogram has a digit's sum in as many copies as fit, by lanes: few digits are many
// candidates for each.  One of two: while it is filled the next is cleared.  The first
// wavefront finds the digit.
struct Select {
  unsigned long long hist[2][kBins];
  unsigned long long red[kWaves];
  unsigned long long want;
  uint32_t ones, zeros;  // bits that some key has set, and clear
  uint32_t found;
};
template <typename Each, typename Weight>
__device__ inline uint32_t select(Each each, Weight weight, unsigned long long& want, Select& l) {
  uint32_t ones = 0, zeros = 0;
  each([&](uint32_t key) {
    ones |= key;
    zeros |= ~key;
  });
  auto either = [](uint32_t a, uint32_t b) { return a | b; };
  ones = wave_join(ones, 0, either);
  zeros = wave_join(zeros, 0, either);
  __syncthreads();  // the last use of l
  if (threadIdx.x == 0) l.ones = l.zeros = 0;
  if (threadIdx.x < kBins) l.hist[0][threadIdx.x] = 0;
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
    atomicOr(&l.ones, ones);
    atomicOr(&l.zeros, zeros);
  }
  __syncthreads();
  ones = l.ones;
  const uint32_t differ = ones & l.zeros;
  uint32_t found = ones & ~differ;
  if (differ == 0) return found;
  const int stop = __builtin_ctz(differ);  // below it the keys agree
  int left = 32 - __builtin_clz(differ);   // bits still open
  for (int round = 0; left > stop; ++round) {
    const int shift = max(left - kDigits, stop), bits = left - shift;
    const uint32_t digits = (1u << bits) - 1, copies = (uint32_t)kBins >> bits;
    unsigned long long* h = l.hist[round % 2];
    if (threadIdx.x < kBins) l.hist[(round + 1) % 2][threadIdx.x] = 0;
    each([&](uint32_t key) {
      if (left == 32 || (key >> left) == (found >> left))
        atomicAdd(&h[(digits - ((key >> shift) & digits)) * copies +
                     (threadIdx.x & (copies - 1))],
                  weight(key));
    });
    __syncthreads();
    if (threadIdx.x < 64) {
      const Entries<unsigned long long> e(h);
      const Cross c = e.cross(want);
      const uint32_t place = c.at < kBins ? c.at / copies : digits;  // (found: want <= the sum)
      const unsigned long long above = copies > 1 ? e.upto((int)(place * copies), false) : c.before;
      if (threadIdx.x == 0) {
        l.found = found | (digits - place) << shift;
        l.want = want - above;
      }
    }
    __syncthreads();
    found = l.found;
    want = l.want;
    left = shift;
  }
  return found;
}

// Step 3 for a slice and, in the row's last workgroup, for the row.  WHOLE: the slice is
// the row, its Row is in LDS.
struct Pick {
  uint32_t list[kListMax];
  unsigned int n, at, last;
  // Top-k's threshold is in interval kb (kBins: none, fewer values than k): `above`
  // values and the weight `least` come before it.  Top-p's is in one of lo to hi; in
  // pb, `before` it, where that is one for all that top-k may leave (else kBins).
  int kb, lo, hi, pb;
  unsigned long long above, least, before;
  Select l;
};
template <typename T, bool WHOLE>
__device__ inline void pick_of_slice(const Args& a, const Settings& s, Run<T>& run, Row& r,
                                     uint32_t* row_list, const double* pow16, Pick& sh) {
  const int wave = threadIdx.x >> 6;
  uint32_t* list = sh.list;
  if (wave == 0) {
    Cross k{kBins, 0}, p{kBins, 0};
    if (s.by_k) k = Entries<unsigned int>(r.count).cross((unsigned long long)s.k);
    int p0 = kBins, p1 = -1;
    unsigned long long w = 0;
    if (s.by_p) {
      // the weight that top-k leaves lies between that before its interval and that
      // with all of it
      const Entries<unsigned long long> m(r.mass);
      w = k.at == kBins ? m.total : m.upto(k.at, false);
      p = m.cross(share_up(s.p, w));
      p0 = min(p.at, k.at);
      p1 = k.at == kBins ? p0 : min(m.cross(share_up(s.p, m.upto(k.at, true))).at, k.at);
    }
    if (threadIdx.x == 0) {
      sh.n = 0;
      sh.kb = k.at;
      sh.above = k.before;
      sh.least = w;
      sh.lo = p0;
      sh.hi = p1;
      sh.pb = p0 == p1 && p.at == p0 ? p0 : kBins;
      sh.before = p.before;
    }
  }
  __syncthreads();
  const int kb = sh.kb;
  {
    const int b0 = kb, b1 = sh.lo, b2 = sh.hi;
    run.each([&](const auto& x, int) {
#pragma unroll
      for (int i = 0; i < Chunks<T>::E; ++i) {
        const int b = bin_of(x[i], s);
        if (b >= 0 && (b == b0 || (b >= b1 && b <= b2))) {
          const unsigned int to = atomicAdd(&sh.n, 1u);
          if (to < kListMax) list[to] = key_of(x[i]);
        }
      }
    });
  }
  __syncthreads();
  unsigned int listed = sh.n;
  if constexpr (!WHOLE) {
    const unsigned int n = listed;
    if (threadIdx.x == 0 && n > 0) sh.at = atomicAdd(&r.listed, n);
    __syncthreads();
    const unsigned int at = sh.at;
    if (n > 0 && at < kListMax) {
      const unsigned int room = min(n, kListMax - at);
      for (unsigned int i = threadIdx.x; i < room; i += kThreads) put(&row_list[at + i], list[i]);
    }
    const bool is_last = last_of_row(&r.arrived[0], a.slices);
    if (threadIdx.x == 0) sh.last = is_last;
    __syncthreads();
    if (!sh.last) return;
    listed = get(&r.listed);
    if (listed <= kListMax)
      for (unsigned int i = threadIdx.x; i < listed; i += kThreads) list[i] = get(&row_list[i]);
    __syncthreads();
  }
  // the values of interval b, from the list or, where that overflowed, the row
  const bool in_list = listed <= kListMax;
  const unsigned int candidates = in_list ? listed : (unsigned int)a.cols;
  auto values = [&](int b) {
    return [&, b](auto f) {
      for (unsigned int i = threadIdx.x; i < candidates; i += kThreads) {
        const float x = in_list ? value_of(list[i]) : Elem<T>::load(run.c.base + i);
        if (bin_of(x, s) == b) f(key_of(x));
      }
    };
  };
  // top-k's threshold, then top-p's
  uint32_t cut = 0;
  unsigned long long ties = 0;
  for (int by_p = kb < kBins ? 0 : 1; by_p <= (s.by_p ? 1 : 0); ++by_p) {
    auto weight = [&](uint32_t key) {
      return by_p ? weight_of(value_of(key), s, a.shift, pow16) : 1ull;
    };
    Cross c{kb, sh.above};
    unsigned long long want = (unsigned long long)s.k;
    if (by_p) {
      unsigned long long total = sh.least;
      if (kb < kBins) {
        unsigned long long more = 0;
        values(kb)([&](uint32_t key) {
          if (key > cut) more += weight(key);
        });
        total += sum_of(more, sh.l.red) + ties * weight(cut);
      }
      want = share_up(s.p, total);
      c = Cross{sh.pb, sh.before};
      if (c.at == kBins) c = Entries<unsigned long long>(r.mass).cross(want);
    }
    want -= c.before;
    cut = select(values(c.at), weight, want, sh.l);
    // as many as reach it: want / weight, rounded up (below 2^23: the quotient in f64
    // is off by one at most)
    const unsigned long long w = max(weight(cut), 1ull);
    ties = (unsigned long long)((double)want / (double)w);
    while (ties * w < want) ++ties;
    while (ties > 0 && (ties - 1) * w >= want) --ties;
  }
  if (threadIdx.x == 0) {
    r.cut = cut;
    r.ties = ties;
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(8))) void
sample_pick_kernel(const Args a) {
  const int row = blockIdx.y, slice = blockIdx.x, wave = threadIdx.x >> 6;
  __shared__ Settings settings;
  __shared__ double pow16[16];
  __shared__ Pick sh;
  RowSpace& r = a.rows[row];
  Run<T> run(a, row, slice * kWaves + wave);
  if (threadIdx.x < 16) pow16[threadIdx.x] = kPow[threadIdx.x];
  prepare(a, row, r, settings);
  __syncthreads();
  const Settings s = settings;
  if (s.narrows()) pick_of_slice<T, false>(a, s, run, r, r.list, pow16, sh);
}

// Step 4 for a slice and, in the row's last workgroup, for the row.
template <typename T, bool WHOLE>
__device__ inline void draw_of_slice(const Args& a, int row, int slice, const Settings& s,
                                     Run<T>& run, Row& r, Part* parts, const double* pow16) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
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
  const uint32_t cut = s.narrows() ? r.cut : 0;
  const unsigned long long ties = s.narrows() ? r.ties : 0;
  // What is kept of the wavefront's run.
  unsigned long long mass = 0;
  unsigned int equal = 0;
  run.each([&](const auto& x, int) {
#pragma unroll
    for (int i = 0; i < Chunks<T>::E; ++i) {
      const uint32_t key = key_of(x[i]);
      if (key > cut) mass += kept_weight(x[i], s, a.shift, pow16);
      equal += cut && key == cut;
    }
  });
  mass = wave_sum(mass);
  equal = wave_sum(equal);
  if constexpr (WHOLE) {
    if (lane == 0) parts[wave] = Part{mass, equal, 0};
    __syncthreads();
    if (wave != 0) return;
  } else {
    if (lane == 0) {
      put(&parts[slice * kWaves + wave].mass, mass);
      put(&parts[slice * kWaves + wave].ties, equal);
    }
    if (!last_of_row(&r.arrived[1], a.slices)) return;
  }
  // The row's last workgroup has every part; its first wavefront draws.
  const unsigned long long even = cut ? kept_weight(value_of(cut), s, a.shift, pow16) : 0;
  // of n tokens at the threshold with `before` of them in front, the weight of those kept
  auto tied = [&](unsigned long long before, unsigned int n) -> unsigned long long {
    return before >= ties ? 0 : min((unsigned long long)n, ties - before) * even;
  };
  const int count = a.slices * kWaves, each = (count + 63) / 64;
  unsigned long long m[kLaneParts], eq = 0, sum = 0;
  unsigned int n_eq[kLaneParts];
#pragma unroll
  for (int i = 0; i < kLaneParts; ++i) {
    const int at = lane * each + i;
    const bool there = i < each && at < count;
    m[i] = !there ? 0 : WHOLE ? parts[at].mass : get(&parts[at].mass);
    n_eq[i] = !there ? 0 : WHOLE ? parts[at].ties : get(&parts[at].ties);
  }
#pragma unroll
  for (int i = 0; i < kLaneParts; ++i) eq += n_eq[i];
  unsigned long long eq_run = wave_scan(eq) - eq;
#pragma unroll
  for (int i = 0; i < kLaneParts; ++i) {
    m[i] += tied(eq_run, n_eq[i]);
    sum += m[i];
    eq_run += n_eq[i];
  }
  eq_run -= eq;
  const unsigned long long upto = wave_scan(sum);
  // the first kept token with a running sum above uniform * the total
  const unsigned long long target = share_down(a.uniform[row], lane_of(upto, 63));
  unsigned long long from = upto - sum;
  const unsigned long long hit =
      __builtin_amdgcn_ballot_w64(from <= target && target < upto);
  const int holder = hit ? __builtin_ctzll(hit) : 0;
  int part = lane * each;
#pragma unroll
  for (int i = 0; i < kLaneParts - 1; ++i) {
    const bool past = part == lane * each + i && i + 1 < each && target >= from + m[i];
    part += past;
    from += past ? m[i] : 0;
    eq_run += past ? n_eq[i] : 0;
  }
  part = min((int)lane_of((uint32_t)part, holder), count - 1);
  from = lane_of(from, holder);
  eq_run = lane_of(eq_run, holder);
  // its chunks, 64 at a time
  const Run<T> chosen(a, row, part);
  for (int c0 = chosen.at - lane; c0 < chosen.end; c0 += 64) {
    const bool have = c0 + lane < chosen.end;
    float x[Chunks<T>::E];
    unsigned long long w[Chunks<T>::E];
    unsigned int n = 0;
    mass = 0;
    if (have) {
      chosen.c.load(c0 + lane, x);
#pragma unroll
      for (int i = 0; i < Chunks<T>::E; ++i) {
        const uint32_t key = key_of(x[i]);
        w[i] = key > cut ? kept_weight(x[i], s, a.shift, pow16) : 0;
        mass += w[i];
        n += cut && key == cut;
      }
    }
    const unsigned int n_upto = wave_scan(n);
    unsigned long long before_eq = eq_run + (n_upto - n);
    mass += tied(before_eq, n);
    const unsigned long long m_upto = wave_scan(mass);
    unsigned long long at = from + (m_upto - mass);
    const bool mine = at <= target && target < at + mass;
    if (mine) {
      int token = 0;
      bool done = false;
#pragma unroll
      for (int i = 0; i < Chunks<T>::E; ++i) {
        if (cut && key_of(x[i]) == cut) {
          w[i] = tied(before_eq, 1);
          ++before_eq;
        }
        at += w[i];
        if (!done && at > target) {
          token = chosen.c.index(c0 + lane, i);
          done = true;
        }
      }
      a.out[row] = token;
    }
    if (__builtin_amdgcn_ballot_w64(mine) != 0) return;
    from += lane_of(m_upto, 63);
    eq_run += lane_of(n_upto, 63);
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(8))) void
sample_draw_kernel(const Args a) {
  const int row = blockIdx.y, slice = blockIdx.x, wave = threadIdx.x >> 6;
  __shared__ Settings settings;
  __shared__ double pow16[16];
  Row& r = a.rows[row];
  Run<T> run(a, row, slice * kWaves + wave);
  if (threadIdx.x < 16) pow16[threadIdx.x] = kPow[threadIdx.x];
  prepare(a, row, r, settings);
  __syncthreads();
  draw_of_slice<T, false>(a, row, slice, settings, run, r,
                          a.parts + (int64_t)row * a.slices * kWaves, pow16);
}

// All steps for a row.
template <typename T>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(4))) void
sample_row_kernel(const Args a) {
  const int row = blockIdx.x, wave = threadIdx.x >> 6;
  __shared__ Row r;
  __shared__ Settings settings;
  __shared__ double pow16[16];
  __shared__ Pick sh;
  __shared__ Part parts[kWaves];
  if (threadIdx.x < 16) pow16[threadIdx.x] = kPow[threadIdx.x];
  max_of_slice<T>(a, row, 0, r);
  __syncthreads();
  prepare(a, row, r, settings);
  __syncthreads();
  const Settings s = settings;
  if (s.narrows()) {
    Run<T> run(a, row, wave);
    hist_of_slice<T>(a, s, run, r.mass, r.count, pow16);
    Run<T> again(a, row, wave);
    pick_of_slice<T, true>(a, s, again, r, nullptr, pow16, sh);
    __syncthreads();
  }
  Run<T> run(a, row, wave);
  draw_of_slice<T, true>(a, row, 0, s, run, r, parts, pow16);
}

// Slices of a row: workgroups of 512 threads, four a CU, a chunk a thread or more.  One,
// and so one launch, where the row is short: us in four launches and in one, 32 rows of
// 4096 28 / 18 bf16 and 27 / 21 f32, 1 x 8192 24.4 / 22.4 and 22.8 / 23.8, 32 x 8192 30 /
// 25.6 and 28.7 / 28.2, 253 x 8192 36 / 27 and 37 / 30, but 32 x 16384 30 / 35; and for
// many rows: 512 x 50257 128 / 122 and 134 / 125, 400 x 50257 111 / 120.
constexpr int kManyRows = 512;
int most_slices(int rows) {
  return std::max(1, std::min(kMaxSlices, kWorkgroups / std::max(rows, 1)));
}
int slices_of(int rows, int cols, int chunks) {
  if (cols <= 8192 || rows >= kManyRows) return 1;
  return std::max(1, std::min(most_slices(rows), (chunks + kThreads - 1) / kThreads));
}

}  // namespace
}  // namespace pa

using namespace pa;

extern "C" size_t pa_sample_workspace_size(int32_t rows) {
  if (rows <= 0 || rows >= kManyRows) return 0;  // (many: a workgroup a row)
  return (size_t)rows * (sizeof(RowSpace) + most_slices(rows) * kWaves * sizeof(Part));
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
  PA_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && (uintptr_t)workspace % 16 == 0),
             PA_ERR_WORKSPACE, "pa_sample: workspace of %zu bytes (16-byte aligned) needed, %zu given",
             need, workspace ? workspace_bytes : 0);
  const int chunks = (int)(((int64_t)cols * es + 15) / 16) + 1;
  const int slices = slices_of(rows, cols, chunks);
  int bits = 1;
  while ((1 << bits) < cols) ++bits;
  const Args a{out, logits, row_stride, uniform, temperature, top_k, top_p, min_p, (RowSpace*)workspace,
               (Part*)((RowSpace*)workspace + rows), cols, slices, std::min(62 - bits, 51)};
  const dim3 grid(slices, rows);
  hipStream_t s = (hipStream_t)stream;
#define PA_LAUNCH_SAMPLE(KERNEL)                                                   \
  (dtype == PA_DTYPE_BF16 ? KERNEL<uint16_t><<<grid, kThreads, 0, s>>>(a)          \
                          : KERNEL<float><<<grid, kThreads, 0, s>>>(a))
  if (slices == 1) {
    if (dtype == PA_DTYPE_BF16)
      sample_row_kernel<uint16_t><<<rows, kThreads, 0, s>>>(a);
    else
      sample_row_kernel<float><<<rows, kThreads, 0, s>>>(a);
    return check_launch("pa_sample");
  }
  PA_LAUNCH_SAMPLE(sample_max_kernel);
  if (top_k || top_p) {
    PA_LAUNCH_SAMPLE(sample_hist_kernel);
    PA_LAUNCH_SAMPLE(sample_pick_kernel);
  }
  PA_LAUNCH_SAMPLE(sample_draw_kernel);
#undef PA_LAUNCH_SAMPLE
  return check_launch("pa_sample");
}
