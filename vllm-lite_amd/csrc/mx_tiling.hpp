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
// smallest estimate is the fastest tiling or within 7.5% of it, 0.2% on
// average.  Measured, us (M x wrows x K):
//                     256 x 4096 x 4096  618 x 6144 x 4096  2048 x 4096 x 4096  7569 x 4096 x 4096
//   256 x 256               41.9              43.0               45.0                109.0
//   256 x 128               25.8              27.5               33.9                125.7
//   128 x 128, pairs        23.8              24.7               35.0                127.4
//   128 x 128               17.9              19.8               37.8                152.8
//    64 x  64               11.3              36.0               68.7                255.8
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
// (kw 0: the tiled kernel instead).  Measured, us (rows: N x K):
//                      32: 896 x 4864  4096 x 4096  4096 x 12288  6144 x 4096
//   1 tile, 8 wavefronts       6.7         6.7          17.0         10.1
//   2 tiles, 4                 8.6         7.7          19.6          8.6
//   64 x 64 tiling            10.5        10.2          21.3         10.2
//                      32: 8192 x 8192  12288 x 4096  24576 x 4096  151936 x 896
//   1 tile, 8 wavefronts      19.9          16.8          29.1          59.9
//   2 tiles, 4                16.9          13.8          21.5          30.8
//   64 x 64 tiling            16.3          12.2          25.4          52.8
//                      64: 896 x 4864  4096 x 4096  24576 x 4096  151936 x 896
//   1 tile, 8 wavefronts       8.7         8.8          45.5         117.1
//   2 tiles, 4                11.1         9.9          30.7          46.5
//   64 x 64 tiling            10.6        10.6          28.6          57.2
// (one tile copies X twice as often and fills the chip sooner; the 64 x 64
// tiling wins where its tiles fill one round of the CUs.)  SwiGLU, where a
// workgroup is two groups of kw wavefronts:
//                   16: 4864 x 896  2048 x 8192  12288 x 4096   32: 4864 x 896  2048 x 8192  12288 x 4096
//   kw 4                   5.0         16.5          22.2             5.5          20.6          24.9
//   kw 2                   5.0         18.4          20.5             5.4          21.0          23.4
//   64 x 64 tiling         5.8         15.9          25.4             5.9          15.8          26.3
struct MxSkinny {
  int nt, kw;
};
inline MxSkinny choose_mx_skinny(int M, int N, int K, bool silu) {
  constexpr MxSkinny tiled = {0, 0};
  if (M > (silu ? 32 : 64)) return tiled;
  if (silu) {
    if (M > 16 && N <= 8192 && K >= 4096) return tiled;
    return M <= 16 && N <= 8192 ? MxSkinny{2, 4} : MxSkinny{2, 2};
  }
  if (N <= 4096) return {1, 8};
  if (N > 64 * 512 || (M <= 32 && (N <= 7168 || N > 64 * 256))) return {2, 4};
  return tiled;
}

}  // namespace pa
