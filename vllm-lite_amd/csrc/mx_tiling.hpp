// The choice among the tilings of the MXFP8 GEMM (mx_gemm.hip); host code
// only, so that the rule can be tested without a GPU.
#pragma once
#include <cstdint>

namespace pa {

// The tilings, and the time each would take: rounds of workgroups over the
// 256 CUs (two a CU for the pairs of 128 x 128 tiles), each round `us` plus
// `ns_per_k` for every column of K, the last one `tail` of a round and the rest
// by how full it is.  Fitted to each tiling's times over 289 shapes (M 40 to
// 8192, wrows 256 to 24576, K 160 to 12288; where it is within half as much
// again of the fastest, rms error 3 to 6%), over which the smallest estimate is
// the fastest tiling or within 6% of it, 0.1% on average.  Measured, us:
//                  rows:    333    256    449    618   2048   7569
//                 wrows:    896   4096   3000   6144   4096   4096
//                     K:   4864   4096   6200   4096   4096   4096
//   256 x 256              46.9   39.9   58.5   40.9   43.9  107.1
//   256 x 128              28.9   25.4   36.0   27.2   34.6  126.0
//   128 x 128, pairs       26.6   23.2   33.4   24.2   35.6  128.7
//   128 x 128              19.0   17.6   24.1   20.3   41.7  153.9
//   128 x  64              14.8   13.5   18.6   25.5   53.8  193.1
//    64 x  64              10.9   10.7   24.8   34.1   67.7  238.5
//    64 x  32               9.3   15.2   28.7   51.3  100.5  373.4
// (64 x 32 tiles of SwiGLU would hold half a block of 32 output columns.)
enum MxTiling {
  kMx256x256,
  kMx256x128,
  kMx128x128Pair,
  kMx128x128,
  kMx128x64,
  kMx64x64,
  kMx64x32
};
inline MxTiling choose_mx_tiling(int M, int64_t wrows, int K, bool silu) {
  struct Cost {
    MxTiling t;
    int bm, bn, slots;
    double base, us, ns_per_k, tail;
  };
  static constexpr Cost costs[] = {{kMx256x256, 256, 256, 256, 1.9, 7.7, 11.61, .65},
                                   {kMx256x128, 256, 128, 256, 0.9, 4.8, 7.10, .61},
                                   {kMx128x128Pair, 128, 128, 512, 1.8, 3.3, 7.91, .42},
                                   {kMx128x128, 128, 128, 256, 1.6, 2.7, 4.20, .66},
                                   {kMx128x64, 128, 64, 256, 1.3, 2.2, 2.64, .82},
                                   {kMx64x64, 64, 64, 256, 1.6, 1.9, 1.67, .83},
                                   {kMx64x32, 64, 32, 256, 1.6, 1.6, 1.25, .88}};
  MxTiling best = kMx64x64;
  double best_us = 1e300;
  for (const Cost& c : costs) {
    if (silu && c.t == kMx64x32) continue;
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
//                      32: 4096 x 4096  4096 x 12288  6144 x 4096  8192 x 8192  24576 x 4096
//   1 tile, 8 wavefronts       6.7          16.9         10.1         19.9          28.9
//   2 tiles, 4                 7.7          19.4          8.4         16.9          21.6
//   64 x 32 tiling             8.5          17.2          8.8         13.8          25.5
//   64 x 64 tiling             9.7          20.5          9.7         15.5          24.3
//                      64: 1152 x 896  4096 x 4096  4096 x 12288  8192 x 8192  151936 x 896
//   1 tile, 8 wavefronts       3.7          8.8          21.2         27.3         116.7
//   2 tiles, 4                 4.4          9.9          24.1         20.5          46.4
//   64 x 32 tiling             4.3          8.8          17.5         14.5          76.0
//   64 x 64 tiling             4.8         10.0          21.0         15.9          52.7
// (one tile copies X twice as often and fills the chip sooner; a tiling wins
// where its tiles fill one round of the CUs.)  SwiGLU, where a workgroup is two
// groups of kw wavefronts:
//             rows, N x K: 16, 4864 x 896  2048 x 8192  12288 x 4096
//   kw 4                         5.0          16.5          22.2
//   kw 2                         5.0          18.4          20.5
//   64 x 64 tiling               5.8          15.9          25.4
//                          32, 4864 x 896  2048 x 8192  12288 x 4096
//   kw 4                         5.5          20.6          24.9
//   kw 2                         5.4          21.0          23.4
//   64 x 64 tiling               5.9          15.8          26.3
struct MxSkinny {
  int nt, kw;
};
inline MxSkinny choose_mx_skinny(int M, int N, int K, bool silu) {
  constexpr MxSkinny tiled = {0, 0}, one = {1, 8}, two = {2, 4};
  if (M > (silu ? 32 : 64)) return tiled;
  if (silu) {
    if (M > 16 && N <= 8192 && K >= 4096) return tiled;
    return M <= 16 && N <= 8192 ? MxSkinny{2, 4} : MxSkinny{2, 2};
  }
  if (M > 32) return N > 64 * 512 ? two : N <= 4096 && K < 4096 ? one : tiled;
  return N <= 4096 ? one : N <= 7168 || N > 64 * 256 ? two : tiled;
}

}  // namespace pa
