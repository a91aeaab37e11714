// The choice among the tilings of the MXFP8 GEMM (mx_gemm.hip); host code
// only, so that the rule can be tested without a GPU.
#pragma once
#include <cstdint>

namespace pa {

// The tilings, and the time each would take: rounds of workgroups over the
// 256 CUs (two a CU for the pairs of 128 x 128 tiles), each round `us` plus
// `ns_per_k` for every column of K, the last one `tail` of a round and the rest
// by how full it is.  Fitted to each tiling's times over 197 shapes (M 40 to
// 7569, wrows 896 to 24576, K 160 to 12288; where it is within half as much
// again of the fastest, rms error 4 to 12%), over which the smallest estimate is
// the fastest tiling or within 9% of it, 0.2% on average.  Measured, us:
//                   rows:    333    256    618   2048   7569
//                  wrows:    896   4096   6144   4096   4096
//                      K:   4864   4096   4096   4096   4096
//   256 x 256              47.0   40.1   41.5   44.0  111.1
//   256 x 128              29.0   25.3   27.2   33.8  127.5
//   128 x 128, pairs       26.7   23.2   24.3   34.4  128.6
//   128 x 128              19.3   17.2   20.0   38.4  148.6
//    64 x  64              11.3   10.9   33.8   64.0  240.3
//    64 x  32               9.7   15.4   52.7  103.4  384.2
// (64 x 32 tiles of SwiGLU would hold half a block of 32 output columns.)
enum MxTiling { kMx256x256, kMx256x128, kMx128x128Pair, kMx128x128, kMx64x64, kMx64x32 };
inline MxTiling choose_mx_tiling(int M, int64_t wrows, int K, bool silu) {
  struct Cost {
    MxTiling t;
    int bm, bn, slots;
    double base, us, ns_per_k, tail;
  };
  static constexpr Cost costs[] = {{kMx256x256, 256, 256, 256, 3.0, 7.3, 11.7, .63},
                                   {kMx256x128, 256, 128, 256, 1.1, 4.5, 6.99, .64},
                                   {kMx128x128Pair, 128, 128, 512, 1.8, 3.2, 7.77, .46},
                                   {kMx128x128, 128, 128, 256, 2.0, 2.5, 4.14, .64},
                                   {kMx64x64, 64, 64, 256, 1.3, 2.4, 1.66, .86},
                                   {kMx64x32, 64, 32, 256, 1.6, 1.7, 1.25, .91}};
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
