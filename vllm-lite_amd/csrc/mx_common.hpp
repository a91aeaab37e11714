// MXFP8 blocks on the device: 32 columns, one power-of-two scale, E4M3 codes
// (the format's definition and layouts: include/pa_dense.h).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace pa {

// MXFP8 column steps of 128 (one dword of scale bytes per row).
inline int64_t mx_steps(int64_t cols) { return (cols + 127) / 128; }
inline int64_t mx_pad_rows(int64_t rows) { return (rows + 15) / 16 * 16; }
constexpr int kMxMaxCols = 1 << 22;
inline int64_t mx_scale_bytes(int64_t rows, int64_t cols) {
  return mx_pad_rows(rows) * mx_steps(cols) * 4;
}
// Whether n bytes at p and m at q (NULL: none) have any in common.
inline bool mx_overlap(const void* p, int64_t n, const void* q, int64_t m) {
  const uintptr_t a = (uintptr_t)p, b = (uintptr_t)q;
  return a && b && (a < b ? b - a < (uintptr_t)n : a - b < (uintptr_t)m);
}

// Lane permutations within 16 lanes.  Once a value is equal over each aligned
// group of 4 (8) lanes, the half mirror (mirror) brings the other group's.
template <int CTRL>
__device__ inline uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true);
}
constexpr int kDppXor1 = 0xB1, kDppXor2 = 0x4E, kDppHalfMirror = 0x141, kDppMirror = 0x140;

// The largest finite magnitude of N values, as the bits of a float (0 if none
// is finite).  A maximum of floats finds it wherever all are finite; a NaN or
// an infinity among them shows in the maximum, or (a quiet NaN) is passed over.
// finite: whether none shows in the wavefront's maxima.
template <int N>
__device__ inline uint32_t mx_top(const float (&y)[N], bool& finite) {
  float m = 0.f;
#pragma unroll
  for (int e = 0; e < N; ++e) m = fmaxf(m, __builtin_fabsf(y[e]));
  finite = !__any(!(m < __builtin_inff()));
  if (!finite) {
    uint32_t a = 0;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const uint32_t u = __builtin_bit_cast(uint32_t, y[e]) & 0x7FFFFFFFu;
      a = max(a, u < 0x7F800000u ? u : 0u);
    }
    return a;
  }
  return __builtin_bit_cast(uint32_t, m);
}
template <int N>
__device__ inline uint32_t mx_top(const float (&y)[N]) {
  bool finite;
  return mx_top(y, finite);
}
// The scale byte of a block whose largest finite magnitude has bits a: with
// a = 1.m 2^x, a <= 448 2^e = 1.75 2^(8 + e) asks for e >= x - 8, and one more
// where m is above .75 (the carry); at least 0 (subnormal and zero blocks).
__device__ inline uint32_t mx_scale_byte(uint32_t a) {
  const uint32_t x = (a + 0x1FFFFFu) >> 23;
  return x > 8 ? x - 8 : 0;
}
// 2^(127 - byte), by which a block's values are multiplied (bytes 0 .. 247).
__device__ inline float mx_inverse(uint32_t byte) {
  return __builtin_bit_cast(float, (254u - byte) << 23);
}
// Four codes, rounded to nearest even in the conversion: at most 448, or a NaN
// code for a NaN and (E4M3 has no infinities) an infinity.
__device__ inline uint32_t mx_codes4(float a, float b, float c, float d, float inv) {
  int v = __builtin_amdgcn_cvt_pk_fp8_f32(a * inv, b * inv, 0, false);
  v = __builtin_amdgcn_cvt_pk_fp8_f32(c * inv, d * inv, v, true);
  return (uint32_t)v;
}

// silu(g) u = g u / (1 + e^-g) by the exponential and reciprocal instructions: a
// tile's epilogue runs with one or two wavefronts per SIMD, where expf and the
// division took 9 us of a 256 x 256 tile.  Off by (1.5 |g| + 8) 2^-24 of it at
// most: e^-g is exp2 of the rounded g log2(e), so its error grows with |g| (2^-17
// at -87).  Below -87.3 the reciprocal is below the normal floats, and the result
// 0.
__device__ inline float mx_silu_mul(float g, float u) {
  return g * __builtin_amdgcn_rcpf(1.0f + __expf(-g)) * u;
}

// Eight consecutive columns per lane, a block over 4 lanes, 128 columns over
// 16 lanes, which all run this: the largest magnitude of the lane's block, and
// the four scale bytes of the 128 columns (in every lane) from the lane's own.
__device__ inline uint32_t mx_block_top8(const float (&y)[8], bool& finite) {
  uint32_t a = mx_top(y, finite);
  a = max(a, dpp<kDppXor1>(a));
  return max(a, dpp<kDppXor2>(a));
}
__device__ inline uint32_t mx_scale_dword8(uint32_t byte) {
  uint32_t d = byte << (8 * ((threadIdx.x >> 2) & 3));
  d |= dpp<kDppHalfMirror>(d);
  return d | dpp<kDppMirror>(d);
}
__device__ inline uint2 mx_codes8(const float (&y)[8], float inv) {
  return uint2{mx_codes4(y[0], y[1], y[2], y[3], inv), mx_codes4(y[4], y[5], y[6], y[7], inv)};
}
// Codes and scale bytes of y.
__device__ inline uint2 mx_quantize8(const float (&y)[8], uint32_t& dword) {
  bool finite;
  const uint32_t byte = mx_scale_byte(mx_block_top8(y, finite));
  dword = mx_scale_dword8(byte);
  return mx_codes8(y, mx_inverse(byte));
}
// The same of values of which y has 2^kMxUp times, within 2^-21 of their size;
// top: mx_block_top8 of y; sure: whether the lane's codes and scale are theirs
// all the same, i.e. equal at both ends (never where a y of the wavefront is not
// finite, as times 2^kMxUp it may not be).
constexpr int kMxUp = 64;
__device__ inline uint2 mx_quantize8_up(const float (&y)[8], uint32_t& dword, uint32_t& top,
                                        bool& sure) {
  bool finite;
  top = mx_block_top8(y, finite);
  auto scale_byte = [](uint32_t a) __attribute__((always_inline)) {
    const uint32_t x = (a + 0x1FFFFFu) >> 23;
    return x > 8 + kMxUp ? x - (8 + kMxUp) : 0;
  };
  const uint32_t byte = scale_byte(top);  // up to 183, as top is finite
  const float inv = __builtin_bit_cast(float, (254u - kMxUp - byte) << 23);
  dword = mx_scale_dword8(byte);
  const uint2 lo = mx_codes8(y, inv * (1.f - 0x1p-21f)), hi = mx_codes8(y, inv * (1.f + 0x1p-21f));
  // 8 steps of a float are at least 2^-21 of it
  sure = finite && lo.x == hi.x && lo.y == hi.y &&
         scale_byte(max(top, 8u) - 8) == scale_byte(top + 8);
  return lo;
}

}  // namespace pa
