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

}  // namespace pa
