// Single-token attention over the int8 cache (pa_decode_int8).
//
// A workgroup of NW wavefronts takes part_len tokens of one sequence for up to 16
// query heads of one kv head; its wavefronts share them in steps of 64 tokens and
// merge through LDS.  Contexts of several parts leave a result for each in the
// workspace, which a second launch merges.
// Bound by memory: every code is read once, for all heads of its group: 64 x 4096 of
// 32 / 8 heads of 128 87 us, 6.2 TB/s (99 with a wavefront's steps side by side and
// their ids behind the context length).  Few sequences: by the loads' latency, 32 x
// 320-768 of 14 / 2 x 64 6.1 us.
#include <algorithm>
#include <type_traits>

#include "int8_plan.hpp"
#include "int8_wave.hpp"
#include "pa_internal.hpp"

namespace pa {
namespace {

constexpr int kStep = kInt8Step;

// Each wavefront takes every NW-th step of the part, so that its block ids are known
// before the context length is.  The next step's K is loaded where this one's has
// become scores, its V where this one's has been multiplied: a step is always on its
// way, in one set of registers.
template <int D, int NW>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(D == 256 ? 1 : 2))) void
decode_int8_kernel(
    uint16_t* __restrict__ out, const uint16_t* __restrict__ q, int64_t q_row,
    const int8_t* __restrict__ kc, const int8_t* __restrict__ vc, const uint8_t* __restrict__ ks,
    const uint8_t* __restrict__ vs, const int32_t* __restrict__ tables, int mbs,
    const int32_t* __restrict__ context_lens, int Hq, int Hkv, int G, int head_groups,
    int num_blocks, float scale_log2, int num_parts, int part_len, float* __restrict__ ws_o,
    float* __restrict__ ws_ml) {
  constexpr int DT = D / 16;
  const int lane = threadIdx.x & 63, c = lane & 15, j = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int part = blockIdx.x, seq = blockIdx.z;
  const int kvh = blockIdx.y / head_groups, h0 = (blockIdx.y % head_groups) * 16;
  const int heads = min(G - h0, 16);  // query heads of this workgroup
  const int64_t row0 = (int64_t)seq * Hq + kvh * G + h0;
  const int begin = part * part_len;
  const int32_t* tab = tables + (int64_t)seq * mbs;
  // Lane t holds block t % 4 of the wavefront's step t / 4, for 16 steps.
  // (Counted in blocks: tokens so far behind the largest context pass 31 bits.)
  auto load_ids = [&](int step) -> int32_t {
    const int b =
        begin / kBlock + (wave + (step + lane / 4) * NW) * (kStep / kBlock) + lane % 4;
    return b < mbs ? tab[b] : -1;
  };
  int32_t ids = load_ids(0);
  const int ctx = min(context_lens[seq], mbs * kBlock);
  const int end = min(ctx, begin + part_len);
  if (begin >= end && part > 0) return;  // (part 0 of an empty context writes zeros)
  const Int8Blocks<D> blocks{kc, vc, ks, vs, Hkv, kvh};
  const int left = end - begin - wave * kStep;  // tokens from this wavefront's first step on
  const int steps = left > 0 ? (left + NW * kStep - 1) / (NW * kStep) : 0;
  // a step's blocks, in the pool, and how much of block j there is
  struct Place {
    int kid, vid, lim;
    bool whole;
  };
  auto place = [&](int step) -> Place {
    const int at = 4 * (step % 16);
    Place p{__shfl(ids, at + (c >> 2), 64), __shfl(ids, at + j, 64), 0, false};
    const bool ok = p.vid >= 0 && p.vid < num_blocks;
    const int t0 = begin + (wave + step * NW) * kStep + j * kBlock;
    p.lim = ok ? min(max(end - t0, 0), kBlock) : 0;
    p.whole = __builtin_amdgcn_ballot_w64(p.lim < kBlock) == 0;
    if (!ok) p.vid = 0;
    if (p.kid < 0 || p.kid >= num_blocks) p.kid = 0;
    return p;
  };
  Int8Keys<D> k;
  Int8Values<D> v;
  Place now{};
  if (steps > 0) {
    now = place(0);
    blocks.load_keys(now.kid, now.vid, c, j, k);
    blocks.load_values(now.vid, c, v);
  }
  Int8Query<D> qv;
  int8_query<D>(c < heads ? q + (int64_t)seq * q_row + (int64_t)(kvh * G + h0 + c) * D : nullptr,
                j, scale_log2, qv);
  Int8State<D> S;
  S.init();
  int keys = 0;  // whether block j had any
  auto step = [&](int s, auto more) {
    i32x4 a[4];
    bf16x8 p0, p1;
    int8_scores<D>(k, qv, a);
    const uint32_t kscale = k.scale;
    Place next = now;
    if constexpr (decltype(more)::value) {
      if ((s + 1) % 16 == 0) ids = load_ids(s + 1);
      next = place(s + 1);
      blocks.load_keys(next.kid, next.vid, c, j, k);
    }
    __builtin_amdgcn_sched_barrier(0);
    int8_softmax<D>(a, kscale, v.scale, qv, now.whole, now.lim, S, p0, p1);
    keys |= now.lim;
    __builtin_amdgcn_sched_barrier(0);
    int8_output<D>(v, p0, p1, S);
    if constexpr (decltype(more)::value) blocks.load_values(next.vid, c, v);
    now = next;
  };
  for (int s = 0; s + 1 < steps; ++s) step(s, std::true_type{});
  if (steps > 0) step(steps - 1, std::false_type{});
  if (S.m == kInt8NoMax && __builtin_amdgcn_ballot_w64(keys != 0) != 0) S.m = kInt8AllBelow;
  float lsum = S.lsum;
  lsum += __shfl_xor(lsum, 16, 64);
  lsum += __shfl_xor(lsum, 32, 64);
  // The wavefronts' results meet in LDS (rows 4 floats apart in the banks).
  constexpr int P = D + 4;
  __shared__ __attribute__((aligned(16))) float so[NW][16][P];
  __shared__ float sml[NW][16][2];
  if (c < heads) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
      *reinterpret_cast<f32x4*>(&so[wave][c][16 * dt + 4 * j]) = S.o[dt];
    if (j == 0) {
      sml[wave][c][0] = S.m;
      sml[wave][c][1] = lsum;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < heads * D; i += 64 * NW) {
    const int h = i / D, d = i % D;
    float m = kInt8NoMax;
#pragma unroll
    for (int w = 0; w < NW; ++w) m = fmaxf(m, sml[w][h][0]);
    float num = 0.f, den = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float a = __builtin_amdgcn_exp2f(sml[w][h][0] - m);
      num += a * so[w][h][d];
      den += a * sml[w][h][1];
    }
    if (num_parts == 1) {
      out[row0 * D + i] = f32_to_bf16_bits(int8_quotient(num, den, m));
    } else {
      const int64_t at = (row0 + h) * num_parts + part;
      ws_o[at * D + d] = num;
      if (d == 0) {
        ws_ml[2 * at] = m;
        ws_ml[2 * at + 1] = den;
      }
    }
  }
}

// Merges the parts of one (sequence, query head), one wavefront for each: their
// (m, l) a lane each, 64 at a time, then their outputs eight loads at a time.
template <int DL>
__global__ __launch_bounds__(64) void decode_int8_merge_kernel(
    uint16_t* __restrict__ out, const float* __restrict__ ws_o, const float* __restrict__ ws_ml,
    const int32_t* __restrict__ context_lens, int Hq, int D, int num_parts, int part_len,
    int mbs) {
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x;
  const float2* ml = reinterpret_cast<const float2*>(ws_ml) + row * num_parts;
  const float* o = ws_o + row * num_parts * D;
  float2 mine = ml[min(lane, num_parts - 1)];  // (parts without keys are not written)
  const int ctx = min(context_lens[row / Hq], mbs * kBlock);
  // (the part of the last token: ctx + part_len may pass 31 bits)
  const int np = min(num_parts, (max(ctx, 1) - 1) / part_len + 1);
  float M = kInt8NoMax, num[DL], den = 0.f;
#pragma unroll
  for (int x = 0; x < DL; ++x) num[x] = 0.f;
  for (int p0 = 0; p0 < np; p0 += 64) {
    if (p0 > 0) mine = ml[min(p0 + lane, num_parts - 1)];
    const bool on = p0 + lane < np;
    float m = on ? mine.x : kInt8NoMax;
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) m = fmaxf(m, __shfl_xor(m, s, 64));
    m = fmaxf(m, M);
    const float keep = __builtin_amdgcn_exp2f(M - m);
    M = m;
    const float w = on ? __builtin_amdgcn_exp2f(mine.x - m) : 0.f;
    float l = on ? w * mine.y : 0.f;
#pragma unroll
    for (int s = 32; s > 0; s >>= 1) l += __shfl_xor(l, s, 64);
    den = den * keep + l;
#pragma unroll
    for (int x = 0; x < DL; ++x) num[x] *= keep;
    const int n = min(64, np - p0);
    for (int p = 0; p < n; p += 8) {
      float v[8][DL];
#pragma unroll
      for (int u = 0; u < 8; ++u)
#pragma unroll
        for (int x = 0; x < DL; ++x)
          v[u][x] = lane + 64 * x < D ? o[(int64_t)(p0 + min(p + u, n - 1)) * D + lane + 64 * x]
                                      : 0.f;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        if (p + u < n) {
          const float a = __builtin_bit_cast(
              float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), p + u));
#pragma unroll
          for (int x = 0; x < DL; ++x) num[x] += a * v[u][x];
        }
      }
    }
  }
#pragma unroll
  for (int x = 0; x < DL; ++x)
    if (lane + 64 * x < D)
      out[row * D + lane + 64 * x] = f32_to_bf16_bits(int8_quotient(num[x], den, M));
}

}  // namespace
}  // namespace pa

using namespace pa;

extern "C" size_t pa_decode_int8_workspace_size(int32_t num_seqs, int32_t num_heads,
                                                int32_t num_kv_heads, int32_t head_dim,
                                                int32_t max_context_len) {
  if (num_seqs <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads ||
      head_dim <= 0 || max_context_len <= 0)
    return 0;
  return (size_t)int8_most_parts(num_seqs, num_heads, num_kv_heads, head_dim, max_context_len) *
         num_heads * (head_dim + 2) * sizeof(float);
}

namespace pa {
int32_t decode_int8_strided(void* out, const void* q, int64_t q_row, const int8_t* k_cache,
                            const int8_t* v_cache, const uint8_t* k_scales,
                            const uint8_t* v_scales, const int32_t* block_tables,
                            int32_t max_blocks_per_seq, const int32_t* context_lens,
                            int32_t max_context_len, int32_t num_seqs, int32_t num_heads,
                            int32_t num_kv_heads, int32_t head_dim, int32_t num_blocks, float scale,
                            void* workspace, size_t workspace_bytes, hipStream_t s) {
  clear_error();
  PA_REQUIRE(num_seqs >= 0 && num_heads > 0 && num_kv_heads > 0 && head_dim > 0 &&
                 num_blocks > 0 && max_blocks_per_seq > 0 && max_context_len >= 0,
             PA_ERR_INVALID_ARG, "pa_decode_int8: bad sizes");
  PA_REQUIRE(num_heads % num_kv_heads == 0, PA_ERR_INVALID_ARG,
             "pa_decode_int8: num_heads %d not a multiple of num_kv_heads %d", num_heads,
             num_kv_heads);
  PA_REQUIRE((int64_t)max_blocks_per_seq * kBlock >= max_context_len &&
                 (int64_t)max_blocks_per_seq * kBlock < (1ll << 31) - 4096,
             PA_ERR_OUT_OF_BOUNDS,
             "pa_decode_int8: max_context_len %d, block table of %d blocks", max_context_len,
             max_blocks_per_seq);
  PA_REQUIRE(int8_head_dim(head_dim), PA_ERR_UNSUPPORTED, "pa_decode_int8: head_dim %d", head_dim);
  if (num_seqs == 0 || max_context_len == 0) return PA_OK;
  PA_REQUIRE(out && q && k_cache && v_cache && k_scales && v_scales && block_tables &&
                 context_lens,
             PA_ERR_INVALID_ARG, "pa_decode_int8: null pointer");
  if (q_row == 0) q_row = (int64_t)num_heads * head_dim;
  PA_REQUIRE(q_row >= (int64_t)num_heads * head_dim, PA_ERR_INVALID_ARG,
             "pa_decode_int8: q row stride %lld below num_heads * head_dim", (long long)q_row);
  PA_REQUIRE(((uintptr_t)k_cache | (uintptr_t)v_cache) % 16 == 0 && (uintptr_t)q % 4 == 0 &&
                 q_row % 2 == 0 && (uintptr_t)out % 2 == 0,
             PA_ERR_INVALID_ARG, "pa_decode_int8: caches not 16-byte or q not 4-byte aligned");
  const int G = num_heads / num_kv_heads, head_groups = (G + 15) / 16;
  const Int8Plan plan = int8_plan(num_seqs, num_heads, num_kv_heads, head_dim, max_context_len);
  const int np = plan.parts;
  PA_REQUIRE(num_seqs <= 65535 && (long long)num_kv_heads * head_groups <= 65535 &&
                 (long long)num_blocks * num_kv_heads < (1ll << 32) && grid_fits(np, 512) &&
                 grid_fits((int64_t)num_seqs * num_heads, 256),
             PA_ERR_UNSUPPORTED, "pa_decode_int8: launch too large");
  float* ws_o = nullptr;
  float* ws_ml = nullptr;
  if (np > 1) {
    const size_t rows = (size_t)num_seqs * num_heads * np;
    const size_t need = rows * (head_dim + 2) * sizeof(float);
    PA_REQUIRE(workspace && workspace_bytes >= need && (uintptr_t)workspace % 8 == 0,
               PA_ERR_WORKSPACE, "pa_decode_int8: workspace of %zu bytes needed, %zu given", need,
               workspace ? workspace_bytes : 0);
    ws_o = (float*)workspace;
    ws_ml = ws_o + rows * head_dim;
  }
  const dim3 grid(np, num_kv_heads * head_groups, num_seqs);
#define PA_LAUNCH_DECODE_INT8_NW(DD, NW)                                                       \
  decode_int8_kernel<DD, NW><<<grid, 64 * NW, 0, s>>>(                                         \
      (uint16_t*)out, (const uint16_t*)q, q_row, k_cache, v_cache, k_scales, v_scales,         \
      block_tables, max_blocks_per_seq, context_lens, num_heads, num_kv_heads, G, head_groups, \
      num_blocks, scale * kInt8Log2e, np, plan.part_len, ws_o, ws_ml)
#define PA_LAUNCH_DECODE_INT8(DD)                         \
  do {                                                    \
    if (plan.waves == 4)                                  \
      PA_LAUNCH_DECODE_INT8_NW(DD, 4);                    \
    else                                                  \
      PA_LAUNCH_DECODE_INT8_NW(DD, (DD == 256 ? 4 : 8));  \
  } while (0)
  switch (head_dim) {
    case 32: PA_LAUNCH_DECODE_INT8(32); break;
    case 64: PA_LAUNCH_DECODE_INT8(64); break;
    case 96: PA_LAUNCH_DECODE_INT8(96); break;
    case 128: PA_LAUNCH_DECODE_INT8(128); break;
    case 192: PA_LAUNCH_DECODE_INT8(192); break;
    default: PA_LAUNCH_DECODE_INT8(256); break;
  }
#undef PA_LAUNCH_DECODE_INT8
#undef PA_LAUNCH_DECODE_INT8_NW
  int32_t rc = check_launch("pa_decode_int8");
  if (rc != PA_OK || np == 1) return rc;
  auto merge = [&](auto kernel) {
    kernel<<<num_seqs * num_heads, 64, 0, s>>>((uint16_t*)out, ws_o, ws_ml, context_lens,
                                               num_heads, head_dim, np, plan.part_len,
                                               max_blocks_per_seq);
  };
  if (head_dim <= 64)
    merge(decode_int8_merge_kernel<1>);
  else if (head_dim <= 128)
    merge(decode_int8_merge_kernel<2>);
  else
    merge(decode_int8_merge_kernel<4>);
  return check_launch("pa_decode_int8 merge");
}
}  // namespace pa

extern "C" int32_t pa_decode_int8(void* out, const void* q, const int8_t* k_cache,
                                  const int8_t* v_cache, const uint8_t* k_scales,
                                  const uint8_t* v_scales, const int32_t* block_tables,
                                  int32_t max_blocks_per_seq, const int32_t* context_lens,
                                  int32_t max_context_len, int32_t num_seqs, int32_t num_heads,
                                  int32_t num_kv_heads, int32_t head_dim, int32_t num_blocks,
                                  float scale, void* workspace, size_t workspace_bytes,
                                  pa_stream_t stream) {
  return decode_int8_strided(out, q, 0, k_cache, v_cache, k_scales, v_scales, block_tables,
                             max_blocks_per_seq, context_lens, max_context_len, num_seqs,
                             num_heads, num_kv_heads, head_dim, num_blocks, scale, workspace,
                             workspace_bytes, (hipStream_t)stream);
}
