// MXFP8 rows and weights (pa_dense.h): quantising rows, RMSNorm with an MXFP8
// output, and the weights' layout.
#include <algorithm>
#include <type_traits>

#include "mx_common.hpp"
#include "pa_common.hpp"
#include "pa_internal.hpp"
#include "../../include/pa_dense.h"

// Times here are a call's on the device, calls in a row, over sets of operands
// that together pass the last-level cache.

namespace pa {
namespace {

template <typename T>
struct Vec8;  // eight elements at any element's alignment
template <>
struct Vec8<uint16_t> {
  typedef __bf16 V __attribute__((ext_vector_type(8), aligned(2)));
};
template <>
struct Vec8<float> {
  typedef float V __attribute__((ext_vector_type(8), aligned(4)));
};

// Columns 8 ch .. 8 ch + 7 of a row, 0 behind the last.  A chunk that ends
// behind the row is the end of the row's last eight elements, moved down:
// loaded one by one behind a branch, its elements held up the whole wavefront.
template <typename T>
__device__ inline typename Vec8<T>::V load8(const T* row, int ch, int cols) {
  typename Vec8<T>::V v = 0;
  if (cols >= 8) {
    const int at = min(8 * ch, cols - 8), past = 8 * ch - at;
    v = *reinterpret_cast<const typename Vec8<T>::V*>(row + at);
    if (past) {
#pragma unroll
      for (int by = 1; by <= 4; by *= 2)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (past & by) v[e] = e + by < 8 ? v[e + by] : 0;
      if (past >= 8) v = 0;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (8 * ch + e < cols) v[e] = Elem<T>::load(row + 8 * ch + e);
  }
  return v;
}
template <typename T>
__device__ inline void store8(T* row, int ch, int cols, const typename Vec8<T>::V& v) {
  if (8 * ch + 8 <= cols) {
    *reinterpret_cast<typename Vec8<T>::V*>(row + 8 * ch) = v;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (8 * ch + e < cols) Elem<T>::store(row + 8 * ch + e, v[e]);
  }
}

// Where the codes of columns 8 ch .. and the scale dword of step s of a row go.
struct RowLayout {
  uint8_t *codes, *scales;
  int64_t steps, pad_rows;
  __device__ uint2* code(int64_t row, int64_t ch) const {
    return reinterpret_cast<uint2*>(codes + row * steps * 128 + 8 * ch);
  }
  __device__ uint32_t* scale(int64_t row, int64_t s) const {
    return reinterpret_cast<uint32_t*>(scales) + s * pad_rows + row;
  }
  RowLayout from(int64_t row) const {
    return {codes + row * steps * 128, scales + row * 4, steps, pad_rows};
  }
};
struct WeightLayout {
  uint8_t *codes, *scales;
  int64_t steps;
  __device__ uint2* code(int64_t row, int64_t ch) const {
    return reinterpret_cast<uint2*>(codes + (row / 16 * steps + ch / 16) * 2048 +
                                    ch % 16 / 2 * 256 + row % 16 * 16 + ch % 2 * 8);
  }
  __device__ uint32_t* scale(int64_t row, int64_t s) const {
    return reinterpret_cast<uint32_t*>(scales) + (row / 16 * steps + s) * 16 + row % 16;
  }
  WeightLayout from(int64_t row) const {  // row: a multiple of 16
    return {codes + row / 16 * steps * 2048, scales + row / 16 * steps * 64, steps};
  }
};

// The first of a workgroup's R rows (R a power of two up to 32).  near:
// workgroups are dealt round-robin to the 8 XCDs; the rows of a group of 32,
// whose scales share cache lines, then go to one XCD, so that its L2 puts the
// lines together.  Norm of rows x 4096 with and without, us: 512 6.7 and 6.7,
// 2048 16.0 and 17.2, 7569 43.6 and 45.8.
__device__ inline int64_t first_row(int64_t block, int R, int near) {
  if (!near) return block * R;
  const int64_t i = block / 8;
  const int per = 32 / R;
  return (i / per * 8 + block % 8) * 32 + i % per * R;
}
constexpr int64_t kNearRows = 2048;
inline int64_t row_groups(int64_t rows, int R) {
  return rows >= kNearRows ? (rows + 255) / 256 * (256 / R) : (rows + R - 1) / R;
}

// Eight columns per thread, 16 threads per (row, step of 128 columns), a
// workgroup 2^lg steps of 16 / 2^lg rows at a time, and `times` of these one
// after another.  Rows `rows` .. `out_rows` are written as zeros (the padding
// of a weight).  Bound by memory: 7569 x 4096 bf16 20.3 us, 4.6 TB/s, f32 30.4 us,
// 5.1 TB/s (a large copy: 5.2); 32 x 896 is a launch, 2.5 us.
template <typename T, typename Layout>
__global__ __launch_bounds__(256) void quantize_mx_kernel(Layout out, const T* __restrict__ x,
                                                          int64_t rows, int64_t out_rows, int cols,
                                                          int64_t stride, int lg, int times,
                                                          int near) {
  typedef typename Vec8<T>::V V;
  const int unit = threadIdx.x / 16;
  const int64_t row = first_row(blockIdx.x, 16 >> lg, near) + (unit >> lg);
  int s = ((int)blockIdx.y * times << lg) + (unit & ((1 << lg) - 1));
  const int end = min((int)out.steps, ((int)blockIdx.y + 1) * times << lg);
  if (row >= out_rows || s >= end) return;  // 16 lanes together
  auto load = [&](int st) __attribute__((always_inline)) {
    V v = 0;
    if (row < rows) v = load8(x + row * stride, 16 * st + threadIdx.x % 16, cols);
    return v;
  };
  V v = load(s);
  for (;;) {
    const int next = s + (1 << lg);
    const V v1 = next < end ? load(next) : v;
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = (float)v[e];
    uint32_t dword;
    *out.code(row, 16 * s + threadIdx.x % 16) = mx_quantize8(y, dword);
    if (threadIdx.x % 16 == 0) *out.scale(row, s) = dword;
    if (next >= end) break;
    s = next;
    v = v1;
  }
}

// The sum over a row's G lanes: within 16 lanes by lane permutations, across
// them by shuffles, and for a workgroup per row over its four wavefronts in
// LDS.
template <int CTRL>
__device__ inline double dpp_add(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint64_t o = dpp<CTRL>((uint32_t)u) | (uint64_t)dpp<CTRL>((uint32_t)(u >> 32)) << 32;
  return v + __builtin_bit_cast(double, o);
}
template <int G>
__device__ inline double row_sum(double v, double* red) {
  v = dpp_add<kDppXor1>(v);
  v = dpp_add<kDppXor2>(v);
  v = dpp_add<kDppHalfMirror>(v);
  v = dpp_add<kDppMirror>(v);
  v += __shfl_xor(v, 16, 64);
  v += __shfl_xor(v, 32, 64);
  if constexpr (G == 256) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = (red[0] + red[1]) + (red[2] + red[3]);
  }
  return v;
}

// v w / rms with d = 1 / rms, for a rounding to fewer bits: the f32 nearest to
// the product (v w is exact in f64, and d's error and the product's are 2^-52 of
// it), moved to the odd float beside it on the side where the product lies if
// that f32 is even and not the product itself.  The borders between codes are
// even floats, so the code is that of the product, as if it had not been rounded
// to f32 in between.
__device__ inline float scaled_odd(float v, float w, double d) {
  const double q = (double)v * (double)w * d;
  const float y = (float)q;
  const double low = q - (double)y;
  const int bits = __builtin_bit_cast(int, y);
  // +1: away from zero
  const int side = (((int)(__builtin_bit_cast(uint64_t, low) >> 32) ^ bits) >> 31) | 1;
  constexpr int kFiniteNotZero = 0x198;  // of either sign
  const bool move = __builtin_amdgcn_class(low, kFiniteNotZero) && !(bits & 1);
  return __builtin_bit_cast(float, bits + (move ? side : 0));
}

// G lanes per row (64: a wavefront, 256: the workgroup), chunk i of lane l is
// columns 8 (l + G i) ..  C > 0: the row fits C chunks a lane and stays in
// registers; C = 0: it is read again for the second pass.  The sum of squares
// and, where f32 leaves a code open, the scaling are f64, so that they are the
// codes of the formula, whatever the order of the sum, unless it lies within
// hidden 2^-53 of a border between codes (in f32 throughout, 5 of 10^7 fell to
// the other side).
// Bound by memory: 7569 x 4096 with add, bf16 45 us, 4.9 TB/s, f32 80 us, 5.1
// TB/s, f32 without 33 us, 4.8 TB/s (a large copy: 5.2); short of rows, by its
// latencies: 32 x 896 3.0 us, with add 3.2.  bf16 without add, where a byte takes
// the most arithmetic: 25.4 us, 3.7 TB/s.
template <typename T, int G, int C>
__global__ __launch_bounds__(256) void rms_norm_mx_kernel(RowLayout out, T* sum, const T* residual,
                                                          const T* __restrict__ add,
                                                          const T* __restrict__ w, int64_t rows,
                                                          int hidden, float eps, int near) {
  typedef typename Vec8<T>::V V;
  using E = std::conditional_t<sizeof(T) == 2, __bf16, float>;
  __shared__ double red[4];
  const int lane = threadIdx.x % G;
  const int64_t row = first_row(blockIdx.x, 256 / G, near) + threadIdx.x / G;
  if (row >= rows) return;  // a whole wavefront, or at G = 256 the workgroup
  const int nch = (int)out.steps * 16;
  const T* x = residual + row * hidden;
  const T* a = add ? add + row * hidden : nullptr;
  T* o = add ? sum + row * hidden : nullptr;
  double ss = 0.;
  // the row's value: with add the sum, kept in the storage dtype and stored
  auto take = [&](int ch, V& v, const V& av) __attribute__((always_inline)) {
    if (a) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = (E)((float)v[e] + (float)av[e]);
      store8(o, ch, hidden, v);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fma((double)v[e], (double)v[e], ss);
  };
  double d;
  float r;
  bool usual;  // r 2^kMxUp has all its bits
  auto finish = [&]() __attribute__((always_inline)) {
    d = rsqrt(row_sum<G>(ss, red) / hidden + (double)eps);
    r = (float)(d * __builtin_ldexp(1., kMxUp));
    usual = r >= 0x1p-126f && r < __builtin_inff();
  };
  auto write = [&](int ch, const V& v, const V& wv) __attribute__((always_inline)) {
    // 2^kMxUp times the values: three roundings, r's among them, each at most
    // 2^-24 where v r and the values are normal floats.  So they are wherever a
    // code is not zero, if the block's largest value is at least 2^-40: such
    // values are above 2^-59, and v r, with any weight, above 2^(kMxUp - 187).
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = (float)v[e] * r * (float)wv[e];
    uint32_t dword, top;
    bool sure;
    uint2 codes = mx_quantize8_up(y, dword, top, sure);
    constexpr uint32_t kSmall = (127u + kMxUp - 40) << 23;
    if (__any(top < kSmall)) {  // zeros are exact
      bool zero = true;
#pragma unroll
      for (int e = 0; e < 8; ++e) zero = zero && (float)v[e] == 0.f;
      sure = sure && (top >= kSmall || zero);
    }
    if (!__all(sure && usual)) {  // about 1 of 100 times
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = scaled_odd((float)v[e], (float)wv[e], d);
      codes = mx_quantize8(y, dword);
    }
    *out.code(row, ch) = codes;
    if (threadIdx.x % 16 == 0) *out.scale(row, ch / 16) = dword;
  };
  if constexpr (C > 0) {
    // all loads first: sum may be residual itself, so none moves over a store
    V v[C], av[C], wv[C];
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (lane + G * i < nch) {
        v[i] = load8(x, lane + G * i, hidden);
        if (a) av[i] = load8(a, lane + G * i, hidden);
        wv[i] = load8(w, lane + G * i, hidden);
      }
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (lane + G * i < nch) take(lane + G * i, v[i], av[i]);
    finish();
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (lane + G * i < nch) write(lane + G * i, v[i], wv[i]);
  } else {
    for (int ch = lane; ch < nch; ch += G) {
      V v = load8(x, ch, hidden), av;
      if (a) av = load8(a, ch, hidden);
      take(ch, v, av);
    }
    finish();
    for (int ch = lane; ch < nch; ch += G)
      write(ch, load8<T>(a ? o : x, ch, hidden), load8(w, ch, hidden));
  }
}

template <typename T, typename Layout>
int32_t launch_quantize(const char* what, const Layout& out, const void* x, int64_t rows,
                        int64_t out_rows, int cols, int64_t stride, hipStream_t s) {
  int lg = 0;  // as many steps side by side as there are, up to 16
  while (lg < 4 && 1 << lg < out.steps) ++lg;
  // many rows: whole rows to a workgroup (7569 x 4096: 20.1 us, 21.4 with the
  // steps over workgroups); few: the steps too (512 x 4096: 3.5, 3.7 by rows)
  const int across = (int)((out.steps + (1 << lg) - 1) >> lg);
  const int times = out_rows >= kNearRows ? across : 1;
  int32_t rc = PA_OK;
  for (int64_t at = 0; at < out_rows && rc == PA_OK; at += kLaunchRows) {
    const int64_t n = std::min(kLaunchRows, out_rows - at);
    const dim3 grid((uint32_t)row_groups(n, 16 >> lg), (uint32_t)((across + times - 1) / times));
    quantize_mx_kernel<T, Layout><<<grid, 256, 0, s>>>(
        out.from(at), (const T*)x + at * stride, std::min(rows - at, n), n, cols, stride, lg,
        times, n >= kNearRows);
    rc = check_launch(what);
  }
  return rc;
}

template <typename T, int G, int C>
int32_t launch_norm(const RowLayout& out, void* sum, const void* residual, const void* add,
                    const void* w, int64_t rows, int hidden, float eps, hipStream_t s) {
  int32_t rc = PA_OK;
  for (int64_t at = 0; at < rows && rc == PA_OK; at += kLaunchRows) {
    const int64_t n = std::min(kLaunchRows, rows - at), first = at * hidden;
    rms_norm_mx_kernel<T, G, C><<<(uint32_t)row_groups(n, 256 / G), 256, 0, s>>>(
        out.from(at), add ? (T*)sum + first : nullptr, (const T*)residual + first,
        add ? (const T*)add + first : nullptr, (const T*)w, n, hidden, eps, n >= kNearRows);
    rc = check_launch("pa_rms_norm_mx");
  }
  return rc;
}
// The fewest chunks of 8 columns a lane that hold the row (us with add, bf16 and
// f32: 2048 x 4096 16.0 and 26.5 in 2, 17.6 and 26.4 in 4, 17.9 and 27.7 in 8;
// 2048 x 6144 22.8 and 37.6 in 3, 23.5 and 37.1 in 4; 64 x 16384 10.3 and 10.1 in
// 8, 14.0 and 13.7 read again; but 1500 x 12288 33.8 and 56.0 in 8, 40.7 and 54.4
// in 6).  A wavefront a row up to 512 columns (7569 x 256 7.8 and 8.8, by a
// workgroup 10.3 and 11.8; 2048 x 512 4.7 and 5.8, by one 4.9 and 5.5); in bf16 up
// to 1024 where the rows fill the chip many times over (7569 x 896 15.1, by one
// 16.4; 2048 x 896 6.3 and 6.2, 32 x 896 3.7 and 3.2), in f32 not (7569 x 896 22.5,
// by one 20.6; 7569 x 640 17.9 and 17.8).
template <typename T>
auto choose_norm(int64_t chunks, int64_t rows) {
  if constexpr (sizeof(T) == 2)
    if (chunks > 64 && chunks <= 128 && rows >= 4096) return launch_norm<T, 64, 2>;
  return chunks <= 64     ? launch_norm<T, 64, 1>
         : chunks <= 256  ? launch_norm<T, 256, 1>
         : chunks <= 512  ? launch_norm<T, 256, 2>
         : chunks <= 768  ? launch_norm<T, 256, 3>
         : chunks <= 1024 ? launch_norm<T, 256, 4>
         : chunks <= 2048 ? launch_norm<T, 256, 8>
                          : launch_norm<T, 256, 0>;
}

}  // namespace
}  // namespace pa

using namespace pa;

#define PA_MX_ALIGNED(what, codes, scales)                                                    \
  PA_REQUIRE((uintptr_t)(codes) % 16 == 0 && (uintptr_t)(scales) % 4 == 0, PA_ERR_INVALID_ARG, \
             what ": codes must be 16-byte and scales 4-byte aligned")

extern "C" size_t pa_mx_row_bytes(int32_t cols) {
  return cols > 0 ? (size_t)mx_steps(cols) * 128 : 0;
}
extern "C" size_t pa_mx_scale_bytes(int32_t rows, int32_t cols) {
  return rows > 0 && cols > 0 ? (size_t)mx_scale_bytes(rows, cols) : 0;
}
extern "C" size_t pa_mx_weight_bytes(int32_t rows, int32_t cols) {
  return rows > 0 && cols > 0 ? (size_t)mx_pad_rows(rows) * mx_steps(cols) * 128 : 0;
}

extern "C" int32_t pa_quantize_mx(uint8_t* codes, uint8_t* scales, const void* x, int32_t rows,
                                  int32_t cols, int64_t x_stride, int32_t dtype,
                                  pa_stream_t stream) {
  clear_error();
  PA_REQUIRE(dtype_ok(dtype), PA_ERR_INVALID_ARG, "pa_quantize_mx: unknown dtype %d", dtype);
  PA_REQUIRE(rows >= 0 && cols > 0, PA_ERR_INVALID_ARG, "pa_quantize_mx: bad sizes");
  PA_REQUIRE(cols <= kMxMaxCols, PA_ERR_UNSUPPORTED, "pa_quantize_mx: %d columns", cols);
  PA_REQUIRE(x_stride == 0 || x_stride >= cols, PA_ERR_INVALID_ARG,
             "pa_quantize_mx: rows overlap");
  if (rows == 0) return PA_OK;
  PA_REQUIRE(x_stride <= INT64_MAX / 8 / rows, PA_ERR_INVALID_ARG, "pa_quantize_mx: bad stride");
  PA_REQUIRE(codes && scales && x, PA_ERR_INVALID_ARG, "pa_quantize_mx: null pointer");
  PA_MX_ALIGNED("pa_quantize_mx", codes, scales);
  PA_REQUIRE((uintptr_t)x % dtype_size(dtype) == 0, PA_ERR_INVALID_ARG,
             "pa_quantize_mx: x is not aligned to its elements");
  {
    const int64_t nc = (int64_t)rows * mx_steps(cols) * 128, ns = mx_scale_bytes(rows, cols);
    const int64_t nx =
        ((rows - 1) * (x_stride ? x_stride : cols) + cols) * (int64_t)dtype_size(dtype);
    PA_REQUIRE(!mx_overlap(codes, nc, scales, ns) && !mx_overlap(codes, nc, x, nx) &&
                   !mx_overlap(scales, ns, x, nx),
               PA_ERR_INVALID_ARG, "pa_quantize_mx: arrays overlap");
  }
  const RowLayout out{codes, scales, mx_steps(cols), mx_pad_rows(rows)};
  const int64_t stride = x_stride ? x_stride : cols;
  return (dtype == PA_DTYPE_BF16 ? launch_quantize<uint16_t, RowLayout>
                                 : launch_quantize<float, RowLayout>)(
      "pa_quantize_mx", out, x, rows, rows, cols, stride, (hipStream_t)stream);
}

extern "C" int32_t pa_linear_mx_pack(uint8_t* codes, uint8_t* scales, const void* weight,
                                     int32_t rows, int32_t cols, int32_t dtype,
                                     pa_stream_t stream) {
  clear_error();
  PA_REQUIRE(dtype_ok(dtype), PA_ERR_INVALID_ARG, "pa_linear_mx_pack: unknown dtype %d", dtype);
  PA_REQUIRE(rows > 0 && cols > 0, PA_ERR_INVALID_ARG, "pa_linear_mx_pack: bad sizes");
  PA_REQUIRE(cols <= kMxMaxCols, PA_ERR_UNSUPPORTED, "pa_linear_mx_pack: %d columns", cols);
  PA_REQUIRE(codes && scales && weight, PA_ERR_INVALID_ARG, "pa_linear_mx_pack: null pointer");
  PA_MX_ALIGNED("pa_linear_mx_pack", codes, scales);
  PA_REQUIRE((uintptr_t)weight % dtype_size(dtype) == 0, PA_ERR_INVALID_ARG,
             "pa_linear_mx_pack: the weight is not aligned to its elements");
  {
    const int64_t nc = mx_pad_rows(rows) * mx_steps(cols) * 128, ns = mx_scale_bytes(rows, cols);
    const int64_t nw = (int64_t)rows * cols * (int64_t)dtype_size(dtype);
    PA_REQUIRE(!mx_overlap(codes, nc, scales, ns) && !mx_overlap(codes, nc, weight, nw) &&
                   !mx_overlap(scales, ns, weight, nw),
               PA_ERR_INVALID_ARG, "pa_linear_mx_pack: arrays overlap");
  }
  const WeightLayout out{codes, scales, mx_steps(cols)};
  return (dtype == PA_DTYPE_BF16 ? launch_quantize<uint16_t, WeightLayout>
                                 : launch_quantize<float, WeightLayout>)(
      "pa_linear_mx_pack", out, weight, rows, mx_pad_rows(rows), cols, cols,
      (hipStream_t)stream);
}

extern "C" int32_t pa_rms_norm_mx(uint8_t* codes, uint8_t* scales, void* sum,
                                  const void* residual, const void* add, const void* weight,
                                  int32_t rows, int32_t hidden, float eps, int32_t dtype,
                                  pa_stream_t stream) {
  clear_error();
  PA_REQUIRE(dtype_ok(dtype), PA_ERR_INVALID_ARG, "pa_rms_norm_mx: unknown dtype %d", dtype);
  PA_REQUIRE(rows >= 0 && hidden > 0, PA_ERR_INVALID_ARG, "pa_rms_norm_mx: bad sizes");
  PA_REQUIRE(hidden <= kMxMaxCols, PA_ERR_UNSUPPORTED, "pa_rms_norm_mx: %d columns", hidden);
  if (rows == 0) return PA_OK;
  PA_REQUIRE(codes && scales && residual && weight, PA_ERR_INVALID_ARG,
             "pa_rms_norm_mx: null pointer");
  PA_REQUIRE(!add || sum, PA_ERR_INVALID_ARG, "pa_rms_norm_mx: add needs sum");
  PA_MX_ALIGNED("pa_rms_norm_mx", codes, scales);
  PA_REQUIRE(((uintptr_t)residual | (uintptr_t)add | (uintptr_t)sum | (uintptr_t)weight) %
                     dtype_size(dtype) == 0,
             PA_ERR_INVALID_ARG, "pa_rms_norm_mx: rows are not aligned to their elements");
  {
    const int64_t nc = (int64_t)rows * mx_steps(hidden) * 128, ns = mx_scale_bytes(rows, hidden);
    const int64_t nw = hidden * (int64_t)dtype_size(dtype), nx = rows * nw;
    const void* total = add ? sum : nullptr;
    auto meets = [&](const void* p, int64_t n) {
      return mx_overlap(p, n, residual, nx) || mx_overlap(p, n, add, nx) ||
             mx_overlap(p, n, weight, nw);
    };
    PA_REQUIRE(!mx_overlap(codes, nc, scales, ns) && !mx_overlap(codes, nc, total, nx) &&
                   !mx_overlap(scales, ns, total, nx) && !meets(codes, nc) && !meets(scales, ns) &&
                   !mx_overlap(total, nx, add, nx) && !mx_overlap(total, nx, weight, nw) &&
                   (total == residual || !mx_overlap(total, nx, residual, nx)),
               PA_ERR_INVALID_ARG, "pa_rms_norm_mx: arrays overlap");
  }
  const RowLayout out{codes, scales, mx_steps(hidden), mx_pad_rows(rows)};
  return (dtype == PA_DTYPE_BF16 ? choose_norm<uint16_t>
                                 : choose_norm<float>)(out.steps * 16, rows)(
      out, sum, residual, add, weight, rows, hidden, eps, (hipStream_t)stream);
}
