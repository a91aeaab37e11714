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
// the fastest tiling or within 6% of it, 0.1% on average (operands in the
// last-level cache; from memory the short ones take up to a quarter longer, the
// fastest are the same).  Measured from memory, us:
//                  rows:    333    256    449    618   2048   7569
//                 wrows:    896   4096   3000   6144   4096   4096
//                     K:   4864   4096   6200   4096   4096   4096
//   256 x 256              46.8   47.0   68.7   51.6   55.7  111.2
//   256 x 128              28.9   26.8   38.3   31.5   39.9  129.0
//   128 x 128, pairs       26.5   27.8   42.6   32.5   40.4  129.1
//   128 x 128              19.0   19.8   27.8   24.5   45.4  155.5
//   128 x  64              14.9   14.8   20.1   31.0   59.5  196.3
//    64 x  64              10.9   12.1   26.6   41.3   84.1  235.4
//    64 x  32               9.1   17.0   31.7   60.7  122.2  373.5
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
// (kw 0: the tiled kernel instead).  Measured, us (rows: N x K), from memory and,
// where it settles the choice, in brackets with the operands in the last-level
// cache, as a step's own rows and its smaller weights are:
//                      32: 4096 x 4096  4096 x 12288  6144 x 4096   8192 x 8192   24576 x 4096
//   1 tile, 8 wavefronts       7.7      17.2 (16.9)      11.1       20.4 (19.9)      29.1
//   2 tiles, 4                 7.9      19.9              9.0       17.1 (16.9)      21.8
//   64 x 32 tiling             8.0      20.8 (17.2)      10.2       18.3 (13.8)      27.6
//   64 x 64 tiling             9.3      26.7             11.8       24.2             25.9
//                      64: 1152 x 896  4096 x 4096  4096 x 12288  8192 x 8192
//   1 tile, 8 wavefronts       3.8          9.4      21.4 (21.2)  27.7
//   2 tiles, 4                 4.7         10.3      24.4         20.5 (20.5)
//   64 x 32 tiling             4.1          8.2      24.7 (17.5)  21.6 (14.5)
//   64 x 64 tiling             4.8          9.5      31.9         26.3
//                      64: 24576 x 4096  32768 x 4096  40000 x 896  50000 x 2048  151936 x 896
//   1 tile, 8 wavefronts      45.0          59.5          30.6         55.1          111.2
//   2 tiles, 4                30.5          34.9          14.8         30.6           45.5
//   64 x 32 tiling            31.8          42.9          21.7         41.0           74.5
//   64 x 64 tiling            28.6          32.3          17.4         33.2           52.6
// (one tile copies X twice as often and fills the chip sooner; a tiling wins
// where its tiles fill one round of the CUs.  Narrow outputs with a long K, which
// no kernel here splits over workgroups, take about the same in either: one tile
// and the 64 x 32 tiling at 64 rows, 32 x 12288 17.9 and 16.2, 512 x 4096 8.1 and
// 8.1, 512 x 12288 18.7 and 17.3; at 33 rows 512 x 4096 6.8 and 7.9, at 40 rows
// 16 x 8192 10.2 and 11.7.)  SwiGLU, where a workgroup is two groups of kw
// wavefronts:
//             rows, N x K: 16, 4864 x 896   2048 x 8192   12288 x 4096
//   kw 4                         4.9      16.6               22.8
//   kw 2                         5.0      18.7               20.5
//   64 x 64 tiling               6.1      19.6               27.6
//                          32, 4864 x 896   2048 x 8192   12288 x 4096
//   kw 4                         5.6      20.7               25.3
//   kw 2                         5.5      21.2 (21.0)        23.8
//   64 x 64 tiling               6.1      20.9 (15.8)        28.4
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
