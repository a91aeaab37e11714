// Prints the kernel that pa_linear_mx takes for each "rows, outputs, K, SwiGLU"
// read from stdin (vllm-lite_amd/csrc/mx_tiling.hpp).
#include <cstdio>

#include "mx_tiling.hpp"

int main() {
  static const char* names[] = {"256x256", "256x128", "128x128 pair", "128x128",
                                "128x64",  "64x64",   "64x32"};
  int m, n, k, silu;
  while (std::scanf("%d %d %d %d", &m, &n, &k, &silu) == 4) {
    const pa::MxSkinny s = pa::choose_mx_skinny(m, n, k, silu != 0);
    if (s.kw)
      std::printf("few rows %d/%d\n", s.nt, s.kw);
    else
      std::printf("%s\n", names[pa::choose_mx_tiling(m, (int64_t)n * (silu ? 2 : 1), k, silu != 0)]);
  }
}
