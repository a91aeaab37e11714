// MXFP8 rows and weights (pa_dense.h): quantising rows, RMSNorm with an MXFP8
// output, and the weights' layout.
#include <algorithm>

#include "mx_common.hpp"
#include "pa_common.hpp"
#include "pa_internal.hpp"
#include "../../include/pa_dense.h"

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

// Columns 8 ch .. 8 ch + 7 of a row, 0 behind the last.
template <typename T>
__device__ inline void load8(const T* row, int64_t ch, int cols, float (&y)[8]) {
  if (8 * ch + 8 <= cols) {
    const auto v = *reinterpret_cast<const typename Vec8<T>::V*>(row + 8 * ch);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = (float)v[e];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = 8 * ch + e < cols ? Elem<T>::load(row + 8 * ch + e) : 0.f;
  }
}
template <typename T>
__device__ inline void store8(T* row, int64_t ch, int cols, const float (&y)[8]) {
  if (8 * ch + 8 <= cols) {
    typename Vec8<T>::V v;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (sizeof(T) == 2)
        v[e] = (__bf16)y[e];
      else
        v[e] = y[e];
    }
    *reinterpret_cast<typename Vec8<T>::V*>(row + 8 * ch) = v;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (8 * ch + e < cols) Elem<T>::store(row + 8 * ch + e, y[e]);
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
};

// Eight columns per thread, 16 threads per (row, step of 128 columns).  Rows
// `rows` .. `out_rows` are written as zeros (the padding of a weight).
template <typename T, typename Layout>
__global__ __launch_bounds__(256) void quantize_mx_kernel(Layout out, const T* __restrict__ x,
                                                          int64_t rows, int64_t out_rows, int cols,
                                                          int64_t stride) {
  const int64_t unit = blockIdx.x * (int64_t)16 + threadIdx.x / 16;
  const int64_t row = unit / out.steps, s = unit % out.steps;
  if (row >= out_rows) return;  // 16 lanes together
  const int64_t ch = 16 * s + threadIdx.x % 16;
  float y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (row < rows) load8(x + row * stride, ch, cols, y);
  uint32_t dword;
  *out.code(row, ch) = mx_quantize8(y, dword);
  if (threadIdx.x % 16 == 0) *out.scale(row, s) = dword;
}

template <int G>
__device__ inline float row_sum(float v, float* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  if constexpr (G == 256) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = (red[0] + red[1]) + (red[2] + red[3]);
  }
  return v;
}

// G lanes per row (64: a wavefront, 256: the workgroup), chunk i of lane l is
// columns 8 (l + G i) ..; kHeld: the row fits kNormHeld chunks a lane and stays
// in registers, else it is read again for the second pass.
constexpr int kNormHeld = 4;
template <typename T, int G, bool kHeld>
__global__ __launch_bounds__(256) void rms_norm_mx_kernel(RowLayout out, T* sum, const T* residual,
                                                          const T* __restrict__ add,
                                                          const T* __restrict__ w, int64_t rows,
                                                          int hidden, float eps) {
  __shared__ float red[4];
  const int lane = threadIdx.x % G;
  const int64_t row = blockIdx.x * (int64_t)(256 / G) + threadIdx.x / G;
  if (row >= rows) return;  // a whole wavefront, or at G = 256 never
  const int nch = (int)out.steps * 16;
  const T* x = residual + row * hidden;
  const T* a = add ? add + row * hidden : nullptr;
  T* o = add ? sum + row * hidden : nullptr;
  float ss = 0.f;
  // the row's value: with add the sum, kept in the storage dtype and stored
  auto take = [&](int ch, float (&v)[8], const float (&av)[8]) __attribute__((always_inline)) {
    if (a) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] += av[e];
        if constexpr (sizeof(T) == 2) v[e] = (float)(__bf16)v[e];
      }
      store8(o, ch, hidden, v);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += v[e] * v[e];
  };
  auto write = [&](int ch, float (&v)[8], float inv) __attribute__((always_inline)) {
    float wv[8];
    load8(w, ch, hidden, wv);
    // the product with the weight first: exact for bf16
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = v[e] * wv[e] * inv;
    uint32_t dword;
    *out.code(row, ch) = mx_quantize8(v, dword);
    if (threadIdx.x % 16 == 0) *out.scale(row, ch / 16) = dword;
  };
  if constexpr (kHeld) {
    // all loads first: sum may be residual itself, so none moves over a store
    float v[kNormHeld][8], av[kNormHeld][8];
#pragma unroll
    for (int i = 0; i < kNormHeld; ++i)
      if (lane + G * i < nch) {
        load8(x, lane + G * i, hidden, v[i]);
        if (a) load8(a, lane + G * i, hidden, av[i]);
      }
#pragma unroll
    for (int i = 0; i < kNormHeld; ++i)
      if (lane + G * i < nch) take(lane + G * i, v[i], av[i]);
    const float inv = 1.0f / sqrtf(row_sum<G>(ss, red) / (float)hidden + eps);
#pragma unroll
    for (int i = 0; i < kNormHeld; ++i)
      if (lane + G * i < nch) write(lane + G * i, v[i], inv);
  } else {
    float v[8], av[8];
    for (int ch = lane; ch < nch; ch += G) {
      load8(x, ch, hidden, v);
      if (a) load8(a, ch, hidden, av);
      take(ch, v, av);
    }
    const float inv = 1.0f / sqrtf(row_sum<G>(ss, red) / (float)hidden + eps);
    for (int ch = lane; ch < nch; ch += G) {
      load8<T>(a ? o : x, ch, hidden, v);
      write(ch, v, inv);
    }
  }
}

template <typename T, typename Layout>
int32_t launch_quantize(const char* what, const Layout& out, const void* x, int64_t rows,
                        int64_t out_rows, int cols, int64_t stride, hipStream_t s) {
  const int64_t groups = (out_rows * out.steps + 15) / 16;
  PA_REQUIRE(groups < (1ll << 31), PA_ERR_UNSUPPORTED, "%s: %lld x %d is too large", what,
             (long long)rows, cols);
  quantize_mx_kernel<T, Layout><<<(uint32_t)groups, 256, 0, s>>>(out, (const T*)x, rows, out_rows,
                                                                 cols, stride);
  return check_launch(what);
}

template <typename T>
int32_t launch_norm(const RowLayout& out, void* sum, const void* residual, const void* add,
                    const void* w, int rows, int hidden, float eps, hipStream_t s) {
  auto run = [&](auto kernel, int per) {
    kernel<<<(rows + per - 1) / per, 256, 0, s>>>(out, (T*)sum, (const T*)residual, (const T*)add,
                                                  (const T*)w, rows, hidden, eps);
    return check_launch("pa_rms_norm_mx");
  };
  const int64_t nch = out.steps * 16;
  if (nch <= 64 * kNormHeld) return run(rms_norm_mx_kernel<T, 64, true>, 4);
  if (nch <= 256 * kNormHeld) return run(rms_norm_mx_kernel<T, 256, true>, 1);
  return run(rms_norm_mx_kernel<T, 256, false>, 1);
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
  return rows > 0 && cols > 0 ? (size_t)mx_pad_rows(rows) * mx_steps(cols) * 4 : 0;
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
  PA_REQUIRE(codes && scales && x, PA_ERR_INVALID_ARG, "pa_quantize_mx: null pointer");
  PA_MX_ALIGNED("pa_quantize_mx", codes, scales);
  PA_REQUIRE((uintptr_t)x % dtype_size(dtype) == 0, PA_ERR_INVALID_ARG,
             "pa_quantize_mx: x is not aligned to its elements");
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
  const RowLayout out{codes, scales, mx_steps(hidden), mx_pad_rows(rows)};
  return (dtype == PA_DTYPE_BF16 ? launch_norm<uint16_t> : launch_norm<float>)(
      out, sum, residual, add, weight, rows, hidden, eps, (hipStream_t)stream);
}
