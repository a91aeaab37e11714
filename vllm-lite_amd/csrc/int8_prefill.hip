// Chunked causal attention over the int8 cache (pa_prefill_int8).
//
// A wavefront takes 16 query rows of one head against the keys up to their own,
// straight from the cache.
#include <algorithm>

#include "int8_wave.hpp"
#include "pa_internal.hpp"

namespace pa {
namespace {

constexpr int kStep = 4 * kBlock;  // keys a step
constexpr int kPrefillWaves = 4;

template <int D>
__global__ __launch_bounds__(64 * kPrefillWaves) void prefill_int8_kernel(
    uint16_t* __restrict__ out, const uint16_t* __restrict__ q, int64_t q_row,
    const int8_t* __restrict__ kc, const int8_t* __restrict__ vc, const uint8_t* __restrict__ ks,
    const uint8_t* __restrict__ vs, const int32_t* __restrict__ tables, int mbs,
    const int32_t* __restrict__ cu_q, const int32_t* __restrict__ past_lens, int Hq, int Hkv,
    int G, int num_blocks, float scale_log2, int total_q, int max_q) {
  constexpr int DT = D / 16;
  const int lane = threadIdx.x & 63, c = lane & 15, j = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int head = blockIdx.y, kvh = head / G, seq = blockIdx.z;
  const int q_begin = min(max(cu_q[seq], 0), total_q);
  const int len = min(min(max(cu_q[seq + 1], q_begin), total_q) - q_begin, max_q);
  const int past = max(past_lens[seq], 0);
  const int r0 = (blockIdx.x * kPrefillWaves + wave) * 16;
  if (r0 >= len) return;
  const int row = r0 + c;
  Int8Query<D> qv;
  int8_query<D>(row < len ? q + (int64_t)(q_begin + row) * q_row + (int64_t)head * D : nullptr, j,
                scale_log2, qv);
  // keys in all, and of this lane's row
  const int64_t cap = (int64_t)mbs * kBlock;
  const int end = (int)min((int64_t)past + min(len, r0 + 16), cap);
  const int mine = (int)min((int64_t)past + row + 1, cap);
  const int32_t* tab = tables + (int64_t)seq * mbs;
  const Int8Blocks<D> blocks{kc, vc, ks, vs, Hkv, kvh};
  Int8State<D> S;
  S.init();
  int32_t ids = -1;
  const int steps = (end + kStep - 1) / kStep;
  for (int s = 0; s < steps; ++s) {
    const int b = 4 * s;
    if (s % 16 == 0) ids = b + lane < mbs ? tab[b + lane] : -1;
    const int at = 4 * (s % 16);
    int kid = __shfl(ids, at + (c >> 2), 64), vid = __shfl(ids, at + j, 64);
    const bool ok = vid >= 0 && vid < num_blocks;
    const int lim = ok ? min(max(mine - (b + j) * kBlock, 0), kBlock) : 0;
    const bool whole = __builtin_amdgcn_ballot_w64(lim < kBlock) == 0;
    if (!ok) vid = 0;
    if (kid < 0 || kid >= num_blocks) kid = 0;
    Int8Keys<D> k;
    Int8Values<D> v;
    blocks.load_keys(kid, vid, c, j, k);
    blocks.load_values(vid, c, v);
    i32x4 a[4];
    bf16x8 p0, p1;
    int8_scores<D>(k, qv, a);
    int8_softmax<D>(a, k.scale, v.scale, qv.factor, whole, lim, S, p0, p1);
    int8_output<D>(v, p0, p1, S);
  }
  float lsum = S.lsum;
  lsum += __shfl_xor(lsum, 16, 64);
  lsum += __shfl_xor(lsum, 32, 64);
  if (row >= len) return;
  const float inv = lsum != 0.f ? 1.f / lsum : 0.f;
  uint16_t* o = out + ((int64_t)(q_begin + row) * Hq + head) * D + 4 * j;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
    struct __attribute__((aligned(8))) W {
      uint16_t v[4];
    } w;
#pragma unroll
    for (int r = 0; r < 4; ++r) w.v[r] = f32_to_bf16_bits(S.o[dt][r] * inv);
    *reinterpret_cast<W*>(o + 16 * dt) = w;
  }
}

}  // namespace

int32_t prefill_int8_strided(void* out, const void* q, int64_t q_row, const int8_t* k_cache,
                             const int8_t* v_cache, const uint8_t* k_scales,
                             const uint8_t* v_scales, const int32_t* block_tables,
                             int32_t max_blocks_per_seq, const int32_t* cu_q_lens,
                             const int32_t* past_lens, int32_t num_seqs, int32_t total_q,
                             int32_t max_q_len, int32_t num_heads, int32_t num_kv_heads,
                             int32_t head_dim, int32_t num_blocks, float scale, hipStream_t s) {
  clear_error();
  PA_REQUIRE(num_seqs >= 0 && total_q >= 0 && max_q_len >= 0 && num_heads > 0 &&
                 num_kv_heads > 0 && head_dim > 0 && num_blocks > 0 && max_blocks_per_seq > 0,
             PA_ERR_INVALID_ARG, "pa_prefill_int8: bad sizes");
  PA_REQUIRE(num_heads % num_kv_heads == 0, PA_ERR_INVALID_ARG,
             "pa_prefill_int8: num_heads %d not a multiple of num_kv_heads %d", num_heads,
             num_kv_heads);
  PA_REQUIRE(int8_head_dim(head_dim), PA_ERR_UNSUPPORTED, "pa_prefill_int8: head_dim %d", head_dim);
  if (num_seqs == 0 || total_q == 0 || max_q_len == 0) return PA_OK;
  PA_REQUIRE(out && q && k_cache && v_cache && k_scales && v_scales && block_tables &&
                 cu_q_lens && past_lens,
             PA_ERR_INVALID_ARG, "pa_prefill_int8: null pointer");
  if (q_row == 0) q_row = (int64_t)num_heads * head_dim;
  PA_REQUIRE(q_row >= (int64_t)num_heads * head_dim, PA_ERR_INVALID_ARG,
             "pa_prefill_int8: q row stride %lld below num_heads * head_dim", (long long)q_row);
  PA_REQUIRE(((uintptr_t)k_cache | (uintptr_t)v_cache) % 16 == 0 && (uintptr_t)q % 4 == 0 &&
                 q_row % 2 == 0 && (uintptr_t)out % 8 == 0,
             PA_ERR_INVALID_ARG,
             "pa_prefill_int8: caches not 16-byte, q not 4-byte or out not 8-byte aligned");
  PA_REQUIRE((int64_t)max_blocks_per_seq * kBlock < (1ll << 31) - 4096 && num_heads <= 65535 &&
                 num_seqs <= 65535 && (long long)num_blocks * num_kv_heads < (1ll << 32) &&
                 grid_fits(((int64_t)max_q_len + 63) / 64, 256),
             PA_ERR_UNSUPPORTED, "pa_prefill_int8: launch too large");
  const int rows = 16 * kPrefillWaves;
  const dim3 grid(((int64_t)max_q_len + rows - 1) / rows, num_heads, num_seqs);
  const int G = num_heads / num_kv_heads;
#define PA_LAUNCH_PREFILL_INT8(DD)                                                             \
  prefill_int8_kernel<DD><<<grid, 64 * kPrefillWaves, 0, s>>>(                                 \
      (uint16_t*)out, (const uint16_t*)q, q_row, k_cache, v_cache, k_scales, v_scales,         \
      block_tables, max_blocks_per_seq, cu_q_lens, past_lens, num_heads, num_kv_heads, G,      \
      num_blocks, scale * kInt8Log2e, total_q, max_q_len)
  switch (head_dim) {
    case 32: PA_LAUNCH_PREFILL_INT8(32); break;
    case 64: PA_LAUNCH_PREFILL_INT8(64); break;
    case 96: PA_LAUNCH_PREFILL_INT8(96); break;
    case 128: PA_LAUNCH_PREFILL_INT8(128); break;
    case 192: PA_LAUNCH_PREFILL_INT8(192); break;
    default: PA_LAUNCH_PREFILL_INT8(256); break;
  }
#undef PA_LAUNCH_PREFILL_INT8
  return check_launch("pa_prefill_int8");
}
}  // namespace pa

using namespace pa;

extern "C" int32_t pa_prefill_int8(void* out, const void* q, const int8_t* k_cache,
                                   const int8_t* v_cache, const uint8_t* k_scales,
                                   const uint8_t* v_scales, const int32_t* block_tables,
                                   int32_t max_blocks_per_seq, const int32_t* cu_q_lens,
                                   const int32_t* past_lens, int32_t num_seqs, int32_t total_q,
                                   int32_t max_q_len, int32_t num_heads, int32_t num_kv_heads,
                                   int32_t head_dim, int32_t num_blocks, float scale,
                                   pa_stream_t stream) {
  return prefill_int8_strided(out, q, 0, k_cache, v_cache, k_scales, v_scales, block_tables,
                              max_blocks_per_seq, cu_q_lens, past_lens, num_seqs, total_q,
                              max_q_len, num_heads, num_kv_heads, head_dim, num_blocks, scale,
                              (hipStream_t)stream);
}
