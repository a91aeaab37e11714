// How pa_decode_int8 cuts a launch (int8_decode.hip); host code only, so that the rule
// can be tested without a GPU.
#pragma once
#include <algorithm>

namespace pa {

constexpr int kInt8Step = 64;  // tokens of a wavefront's step

// How a launch over contexts of up to max_ctx tokens is cut, after sweeps of 1 to 96
// parts and 4 or 8 wavefronts over 37 launches of 2 to 1600 (sequence, kv head) pairs
// and 130 to 120000 tokens: within 3 % of the best of them in the mean, 14 % at worst.
//   One part where contexts are short (the merge's launch takes 3 us) or fill the card
//     by pairs: 32 x 320-768, 14 / 2 heads of 64, 6.6 us and 8.0 as four; 64 x 4096,
//     32 / 8 of 128, 88 and 93 as two; but 16 x 8192-32768 145 as two, 128 as 48.
//   Else as many as put one workgroup on each of 256 CUs (1 x 1537 of 32 / 8 x 128:
//     15 us whole, 10 as 8 to 24 parts; 8 x 8000-16000 of 14 / 2 x 64: 50 whole, 12 as
//     16), and for many or long sequences, whose lengths differ, no longer than 1344 tokens (11 x
//     37-29000 of 24 / 4 x 96: 38 us as 6, 35 as 22 to 24, 40 as 64).  Not where head_dim
//     256 leaves one workgroup to a CU: 5 x 968-20891 67 us as 6, 87 as 16.
//   8 wavefronts a workgroup where workgroups are few, 4 where they are many (1024 pairs
//     of 100-1000 tokens 36 us with 4, 44 with 8) or short.
struct Int8Plan {
  int waves, part_len, parts;
};
constexpr int kInt8Longest = 21 * kInt8Step;  // tokens of a part where there are many
// Contexts up to this are left whole by so many pairs.
constexpr int kInt8WholeCtx = 7 * kInt8Longest / 2;
constexpr long long kInt8WholePairs = 160;

inline Int8Plan int8_plan(int num_seqs, int num_heads, int num_kv_heads, int head_dim,
                          int max_ctx) {
  const int groups = (num_heads / num_kv_heads + 15) / 16;
  const long long pairs = (long long)num_seqs * num_kv_heads * groups;
  long long parts = 1;
  if (max_ctx > 768 && !(pairs >= kInt8WholePairs && max_ctx <= kInt8WholeCtx)) {
    parts = std::min({256 / pairs, (long long)max_ctx / 96, 32ll});
    if (head_dim <= 192 && pairs > 8)
      parts = std::max(parts, ((long long)max_ctx + kInt8Longest - 1) / kInt8Longest);
    parts = std::max(parts, 1ll);
  }
  const long long len = ((max_ctx + parts - 1) / parts + kInt8Step - 1) / kInt8Step * kInt8Step;
  parts = std::max(1ll, (max_ctx + len - 1) / std::max(len, 1ll));
  const bool eight = head_dim < 256 && pairs * parts <= 300 &&
                     !(parts == 1 && head_dim > 64 && max_ctx <= 640);
  return {eight ? 8 : 4, (int)std::max(len, (long long)kInt8Step), (int)parts};
}

// At least the parts, over all its sequences, of a launch in several that has these sizes
// or fewer sequences or shorter contexts; 0 where none of those has.  (int8_plan grows with
// neither: fewer sequences take more parts each, and in parts of whole steps a longer
// context may take fewer.)
inline long long int8_most_parts(int num_seqs, int num_heads, int num_kv_heads, int head_dim,
                                 int max_ctx) {
  if (max_ctx <= 768) return 0;
  const long long per_seq = (long long)num_kv_heads * ((num_heads / num_kv_heads + 15) / 16);
  // the sequences of a launch that is not left whole
  const long long n = max_ctx <= kInt8WholeCtx
                          ? std::min((long long)num_seqs, (kInt8WholePairs - 1) / per_seq)
                          : num_seqs;
  long long most = std::min({256 / per_seq, n * (max_ctx / 96), 32 * n});
  const long long longest = ((long long)max_ctx + kInt8Longest - 1) / kInt8Longest;
  if (head_dim <= 192 && longest > 1) most = std::max(most, n * longest);
  return most > 1 ? most : 0;
}

}  // namespace pa
