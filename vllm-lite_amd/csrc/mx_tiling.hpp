// The choice among the tilings of the MXFP8 GEMM (mx_gemm.hip); host code
// only, so that the rule can be tested without a GPU.
#pragma once
#include <cstdint>

namespace pa {

// The tilings, and the time each would take: rounds of workgroups over the
// 256 CUs (two a CU for the pairs of 128 x 128 tiles), each round `us` plus
// `ns_per_k` for every column of K, the last one `tail` of a round and the rest
// by how full it is.  Fitted to each tiling's times over 127 shapes (M 40 to
// 7569, wrows 896 to 24576, K 160 to 12288; rms error 7 to 9%), over which the
// smallest estimate is the fastest tiling or within 4.6% of it, 0.2% on
// average.  Measured, us (M x wrows x K):
//                     333 x 896 x 4864  618 x 6144 x 4096  2048 x 4096 x 4096  7569 x 4096 x 4096
//   256 x 256               51.8              46.5               48.6                116.8
//   256 x 128               30.0              28.1               34.7                131.7
//   128 x 128, pairs        28.2              25.5               36.8                133.3
//   128 x 128               20.4              21.4               42.7                163.6
//    64 x  64               12.2              38.3               76.2                270.7
enum MxTiling { kMx256x256, kMx256x128, kMx128x128Pair, kMx128x128, kMx64x64 };
inline MxTiling choose_mx_tiling(int M, int64_t wrows, int K) {
  struct Cost {
    MxTiling t;
    int bm, bn, slots;
    double base, us, ns_per_k, tail;
  };
  static constexpr Cost costs[] = {{kMx256x256, 256, 256, 256, 3.7, 11.1, 11.3, .70},
                                   {kMx256x128, 256, 128, 256, 1.75, 5.5, 6.87, .68},
                                   {kMx128x128Pair, 128, 128, 512, 2.0, 4.5, 7.62, .54},
                                   {kMx128x128, 128, 128, 256, 2.3, 4.1, 4.03, .71},
                                   {kMx64x64, 64, 64, 256, 1.8, 3.0, 1.65, .85}};
  MxTiling best = kMx64x64;
  double best_us = 1e300;
  for (const Cost& c : costs) {
    const int64_t tiles = ((M + (int64_t)c.bm - 1) / c.bm) * ((wrows + c.bn - 1) / c.bn);
    const int64_t rest = tiles % c.slots;
    const double rounds =
        tiles / c.slots + (rest ? c.tail + (1 - c.tail) * rest / c.slots : 0.);
    const double us = c.base + rounds * (c.us + c.ns_per_k * 1e-3 * ((K + 127) / 128 * 128));
    if (us < best_us) {
      best_us = us;
      best = c.t;
    }
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
