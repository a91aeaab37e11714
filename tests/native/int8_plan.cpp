// int8_plan and int8_most_parts of each line of stdin (sequences, query heads, kv heads,
// head_dim, context): wavefronts, tokens of a part, parts, the most parts.
#include <cstdio>

#include "int8_plan.hpp"

int main() {
  int b, hq, hkv, d, ctx;
  while (std::scanf("%d %d %d %d %d", &b, &hq, &hkv, &d, &ctx) == 5) {
    const pa::Int8Plan p = pa::int8_plan(b, hq, hkv, d, ctx);
    std::printf("%d %d %d %lld\n", p.waves, p.part_len, p.parts,
                pa::int8_most_parts(b, hq, hkv, d, ctx));
  }
}
