// The choice among the tilings of the MXFP8 GEMM (mx_gemm.hip); host code
// only, so that the rule can be tested without a GPU.
#pragma once
#include <algorithm>
#include <cmath>
#include <cstdint>

namespace pa {

// The tilings, and the time each would take: rounds of workgroups over the
// 256 CUs, each round `us` plus `ns_per_k` for every unit of K.
enum MxTiling { kMx256x256, kMx256x128, kMx128x128Pair, kMx128x128, kMx64x64 };
inline MxTiling choose_mx_tiling(int M, int wrows, int K) {
  constexpr int kCUs = 256;
  struct Cost {
    MxTiling t;
    int bm, bn;
    float us, ns_per_k;
  };
  static constexpr Cost costs[] = {{kMx256x256, 256, 256, 8.f, 12.5f},
                                   {kMx256x128, 256, 128, 6.f, 7.0f},
                                   {kMx128x128, 128, 128, 5.f, 4.2f},
                                   {kMx64x64, 64, 64, 4.f, 1.45f}};
  auto tiles = [&](int bm, int bn) {
    return (double)((M + (int64_t)bm - 1) / bm) * ((wrows + (int64_t)bn - 1) / bn);
  };
  MxTiling best = kMx64x64;
  double best_us = 1e30;
  for (const Cost& c : costs) {
    const double us = std::ceil(tiles(c.bm, c.bn) / kCUs) * (c.us + c.ns_per_k * 1e-3 * K);
    if (us < best_us) {
      best_us = us;
      best = c.t;
    }
  }
  // more 128 x 128 tiles than CUs: two workgroups share a CU
  if (const double n = tiles(128, 128); n > kCUs) {
    const double us = std::ceil(n / (2 * kCUs)) * (8. + 7.2e-3 * K);
    if (us < best_us) best = kMx128x128Pair;
  }
  return best;
}

// The kernel for few rows: W tiles per wavefront and wavefronts that share K
// (kw 0: the tiled kernel instead).  Measured at 32 rows, us:
//   N x K                4096 x 12288  4096 x 4096  896 x 4864  1152 x 896
//   1 tile, 16 wavefronts    16.4          7.9          8.5        3.8
//   2 tiles, 4               17.9          9.0         10.3        3.8
//   64 x 64 tiling           21.7         10.6         10.7        5.6
//                        6144 x 4096  12288 x 4096  24576 x 4096  151936 x 896
//   1 tile, 16 wavefronts    13.2         19.4         37.4         61.2
//   2 tiles, 4                9.7         15.4         23.0         32.5
//   64 x 64 tiling           10.5         12.5         26.3         56.9
// (one tile reads X from L2 twice as often and fills the chip sooner; the 64 x
// 64 tiling wins where its tiles fill one round of the CUs.)  SwiGLU, where a
// workgroup is two groups of kw wavefronts: kw 4 / 2 / the tiling at 4864 x
// 896 6.1 / 6.2 / 6.4, at 12288 x 4096 28.2 / 27.1 / 27.6.  Above 32 rows the
// 64 x 64 tiling is faster (64 rows: 4096 x 12288 21.9 against 28.5).
struct MxSkinny {
  int nt, kw;
};
inline MxSkinny choose_mx_skinny(int M, int N, bool silu) {
  if (M > 32) return {0, 0};
  if (silu) return {2, N <= 8192 ? 4 : 2};
  if (N <= 4096) return {1, 16};
  if (N > 7168 && N <= 64 * 256) return {0, 0};
  return {2, 4};
}

}  // namespace pa
