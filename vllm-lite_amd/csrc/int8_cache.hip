// Writing and reading the int8 cache (pa_append_int8, pa_read_kv_int8).
//
// Quantising a block of 16 tokens and one kv head to int8 with a power-of-two
// scale:
//   a = max |x| of the call's values, e = the least integer >= -126 with
//   a <= 127 2^e, code = rint(x 2^-e).
// Every step is exact but the one rounding to a code: a scale's product or
// quotient only moves the exponent.  A block that grows over several calls keeps
// its scale while the new tokens fit it; where they do not, the codes that are
// there move down by a power of two, with one more rounding.  (A scale a / 127
// would be half a bit finer on average, but a block appended to token by token
// outgrows it three times as often, each time with such a rounding.)
#include <algorithm>

#include "int8_common.hpp"

namespace pa {
namespace {

// The scale's exponent for a largest magnitude a (finite, >= 0): a <= 127 2^e.
// a = m 2^x with 1 <= m < 2 (from its bits; below the normal floats x < -126, and
// the bound -126 holds anyway): 127 = (127 / 64) 2^6, so e = x - 6, one more where
// m > 127 / 64.
__device__ inline int scale_exponent(float a) {
  const uint32_t u = __builtin_bit_cast(uint32_t, a);
  const int x = (int)(u >> 23) - 127;
  const int e = x - 6 + ((u & 0x7FFFFFu) > 0x7E0000u ? 1 : 0);
  return e < -126 ? -126 : e;
}

// x 2^-e to the nearest integer, ties to even, as the low byte: x 2^-e + 1.5 2^23 rounds
// once, to an integer.  For |x| <= 127 2^e (`down` is 2^-e).
__device__ inline uint32_t encode(float x, float down) {
  return __builtin_bit_cast(uint32_t, __builtin_fmaf(x, down, 0x1.8p23f));
}
// The low bytes of four words.
__device__ inline uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0C0C0400u),
                               __builtin_amdgcn_perm(b, a, 0x0C0C0400u), 0x05040100u);
}

struct Eight {
  float v[8];
};

// What the launch works on.
struct AppendArgs {
  int8_t* k_cache;
  int8_t* v_cache;
  uint8_t* k_scales;
  uint8_t* v_scales;
  const void* key;
  const void* value;
  void* q;
  int64_t key_stride, value_stride, q_stride;
  const float* inv_freq;
  const int32_t* tables;
  const int32_t* cu;
  const int32_t* ctx;
  int mbs, num_tokens, max_tokens, chunks, Hq, Hkv, D, num_blocks;
};

// One wavefront for each (sequence, chunk of its touched blocks, column): column
// h < Hkv writes kv head h of K, Hkv + h of V, 2 Hkv + h rotates query head h.  A
// block goes through it whole: its tokens' values in registers, the largest by lane
// shuffles, so no launch reads the tokens twice and the blocks need no order.
// A lane has 8 values of each of TPL neighbouring tokens: 16-byte loads of bf16 rows
// where ALIGNED, and V's codes meet in LDS as words of neighbouring tokens.  ROPE
// (K and q are rotated) is apart for its registers.
// Bound by its chain of loads (offsets, table, old scale and codes) for a decode
// step: 4.2 us for 32 tokens; by memory for prompts: 9434 tokens of 8 x 128 bf16 15.6
// us, 3.7 TB/s (22 with 4 values a lane and codes by compares and conversions).
template <typename T, int D, bool ALIGNED, bool ROPE>
__global__ __launch_bounds__(64) void append_int8_kernel(const AppendArgs a) {
  constexpr int LPR = D / 8;  // lanes a row
  constexpr int SUBS = 64 / LPR >= 16 ? 16 : 64 / LPR >= 8 ? 8 : 64 / LPR >= 4 ? 4 : 2;
  constexpr int TPL = kBlock / SUBS;  // tokens a lane
  // V's codes, [dim][token]; rows of 5 words, to spread the lanes over the banks
  constexpr int PITCH = kBlock + 4;
  __shared__ __attribute__((aligned(16))) uint8_t tile[PITCH * D];
  const int lane = threadIdx.x, sub = lane / LPR, u = lane % LPR;
  const bool on = sub < SUBS;
  const int seq = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
  const int col = blockIdx.y;
  const int part = col < a.Hkv ? 0 : col < 2 * a.Hkv ? 1 : 2;  // K, V, q
  const int head = part == 2 ? col - 2 * a.Hkv : col - part * a.Hkv;
  const int begin = min(max(a.cu[seq], 0), a.num_tokens);
  const int end = min(max(a.cu[seq + 1], begin), a.num_tokens);
  const int n = min(end - begin, a.max_tokens);
  const int start = a.ctx[seq] - (end - begin);  // position of the first new token
  if (n <= 0 || start < 0) return;
  const int64_t row_stride = part == 0 ? a.key_stride : part == 1 ? a.value_stride : a.q_stride;
  const T* src = (const T*)(part == 0 ? a.key : part == 1 ? a.value : a.q) +
                 (int64_t)begin * row_stride + head * D;
  const int b0 = start / kBlock, nb = (int)(((int64_t)start + n - 1) / kBlock) - b0 + 1;
  auto load = [&](const T* p) -> Eight {
    Eight r;
    if constexpr (ALIGNED) {
      struct __attribute__((aligned(16))) V {
        T v[8];
      };
      const V w = *reinterpret_cast<const V*>(p);
#pragma unroll
      for (int i = 0; i < 8; ++i) r.v[i] = Elem<T>::load(w.v + i);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) r.v[i] = Elem<T>::load(p + i);
    }
    return r;
  };
  for (int bi = chunk; bi < nb; bi += a.chunks) {
    const int b = b0 + bi;
    const int first = bi == 0 ? start % kBlock : 0;
    const int last = min(kBlock, start + n - b * kBlock);  // one past the block's last new token
    int32_t id = -1;
    if (part != 2) {
      if (b < a.mbs) id = a.tables[(int64_t)seq * a.mbs + b];
      if (id < 0 || id >= a.num_blocks) continue;
    }
    // token `at` of the block is row at - first of this block's rows
    const T* rows = src + (int64_t)(b * kBlock - start) * row_stride;
    Eight x[TPL];
    uint32_t most = 0;  // the largest magnitude's bits
#pragma unroll
    for (int p = 0; p < TPL; ++p) {
      const int at = sub * TPL + p;
      const bool mine = on && at >= first && at < last;
      x[p] = Eight{{0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}};
      if (mine) x[p] = load(rows + (int64_t)at * row_stride + 8 * u);
    }
#pragma unroll
    for (int p = 0; p < TPL; ++p) {
      const int at = sub * TPL + p;
      if (on && at >= first && at < last) {
        const T* row = rows + (int64_t)at * row_stride;
        if (ROPE && part != 1) {
          // dims i < D / 2 and i + D / 2 form a pair
          const bool low = u < LPR / 2;
          const int i0 = 8 * (low ? u : u - LPR / 2);
          const Eight y = load(row + (low ? 8 * u + D / 2 : 8 * u - D / 2));
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float s, c;
            sincosf((float)(b * kBlock + at) * a.inv_freq[i0 + i], &s, &c);
            x[p].v[i] = low ? __builtin_fmaf(x[p].v[i], c, -(y.v[i] * s))
                            : __builtin_fmaf(x[p].v[i], c, y.v[i] * s);
          }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
          most = max(most, __builtin_bit_cast(uint32_t, x[p].v[i]) & 0x7FFFFFFFu);
      }
    }
    if (part == 2) {
      T* dst = const_cast<T*>(rows);
#pragma unroll
      for (int p = 0; p < TPL; ++p) {
        const int at = sub * TPL + p;
        if (!on || at < first || at >= last) continue;
        T* to = dst + (int64_t)at * row_stride + 8 * u;
        if constexpr (ALIGNED) {
          struct __attribute__((aligned(16))) V {
            T v[8];
          } w;
#pragma unroll
          for (int i = 0; i < 8; ++i) Elem<T>::store(w.v + i, x[p].v[i]);
          *reinterpret_cast<V*>(to) = w;
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) Elem<T>::store(to + i, x[p].v[i]);
        }
      }
      continue;
    }
    auto wave_max = [](uint32_t v) -> uint32_t {
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o, 64));
      return v;
    };
    constexpr uint32_t kInf = 0x7F800000u;
    most = wave_max(most);
    const bool odd = most >= kInf;  // infinities or NaN: of the finite values, then
    if (odd) {
      most = 0;
#pragma unroll
      for (int p = 0; p < TPL; ++p)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t m = __builtin_bit_cast(uint32_t, x[p].v[i]) & 0x7FFFFFFFu;
          most = max(most, m < kInf ? m : 0);
        }
      most = wave_max(most);
    }
    const int64_t slice = (int64_t)id * a.Hkv + head;
    uint8_t* scale = (part == 0 ? a.k_scales : a.v_scales) + slice;
    int8_t* codes = (part == 0 ? a.k_cache : a.v_cache) + slice * (kBlock * D);
    int e = scale_exponent(__builtin_bit_cast(float, most));
    int drop = 0;  // the kept codes move down by 2^drop
    if (first > 0) {
      const int old = (int)*scale - 127;
      e = max(e, old);
      drop = e - old;
    }
    if (lane == 0) *scale = (uint8_t)(e + 127);
    float down = ldexpf(1.f, -e);
    if (odd) {  // in units of 2^e: NaN as 0, infinities as the largest codes
#pragma unroll
      for (int p = 0; p < TPL; ++p)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float v = x[p].v[i] * down;
          x[p].v[i] = v != v ? 0.f : fminf(fmaxf(v, -127.f), 127.f);
        }
      down = 1.f;
    }
    // four of the codes that were there
    auto kept = [&](uint32_t w) -> uint32_t {
      const float by = ldexpf(1.f, -drop);
      return low_bytes(encode((float)(int8_t)w, by), encode((float)(int8_t)(w >> 8), by),
                       encode((float)(int8_t)(w >> 16), by), encode((float)(int8_t)(w >> 24), by));
    };
    if (part == 0) {
      if (drop) {
        uint32_t* words = reinterpret_cast<uint32_t*>(codes);
#pragma unroll 1
        for (int i = lane; i < first * D / 4; i += 64) {
          words[i] = kept(words[i]);
        }
      }
#pragma unroll
      for (int p = 0; p < TPL; ++p) {
        const int at = sub * TPL + p;
        if (!on || at < first || at >= last) continue;
        uint32_t c[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = encode(x[p].v[i], down);
        *reinterpret_cast<uint2*>(codes + at * D + 8 * u) =
            uint2{low_bytes(c[0], c[1], c[2], c[3]), low_bytes(c[4], c[5], c[6], c[7])};
      }
    } else {
      __syncthreads();  // the last block's rows have been read
      if (on) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          uint8_t* to = tile + (8 * u + i) * PITCH + sub * TPL;
          uint32_t c[TPL < 4 ? 4 : TPL] = {};
#pragma unroll
          for (int p = 0; p < TPL; ++p) c[p] = encode(x[p].v[i], down);
          const uint32_t w = low_bytes(c[0], c[1], c[2], c[3]);
          if constexpr (TPL == 1) *to = (uint8_t)w;
          if constexpr (TPL == 2) *reinterpret_cast<uint16_t*>(to) = (uint16_t)w;
          if constexpr (TPL >= 4) *reinterpret_cast<uint32_t*>(to) = w;
          if constexpr (TPL == 8)
            reinterpret_cast<uint32_t*>(to)[1] = low_bytes(c[4], c[5], c[6], c[7]);
        }
      }
      __syncthreads();
      // the bytes of word i that are tokens before t
      auto before = [](int i, int t) -> uint32_t {
        const int n = min(max(t - 4 * i, 0), 4);
        return n == 4 ? 0xFFFFFFFFu : (1u << (8 * n)) - 1;
      };
#pragma unroll 1
      for (int d = lane; d < D; d += 64) {
        struct __attribute__((aligned(16))) Row {
          uint32_t w[kBlock / 4];
        } r;
        Row* to = reinterpret_cast<Row*>(codes + d * kBlock);
#pragma unroll
        for (int i = 0; i < kBlock / 4; ++i)
          r.w[i] = *reinterpret_cast<const uint32_t*>(tile + d * PITCH + 4 * i);
        if (first > 0 || last < kBlock) {
          Row was = *to;
#pragma unroll
          for (int i = 0; i < kBlock / 4; ++i) {
            const uint32_t old = before(i, first), fresh = before(i, last) & ~old;
            if (drop) was.w[i] = (was.w[i] & ~old) | (kept(was.w[i]) & old);
            r.w[i] = (r.w[i] & fresh) | (was.w[i] & ~fresh);
          }
        }
        *to = r;
      }
    }
  }
}

// out[t][h][d] = code * scale, a workgroup for each (block, kv head).
__global__ __launch_bounds__(256) void read_kv_int8_kernel(
    const int8_t* __restrict__ k_cache, const int8_t* __restrict__ v_cache,
    const uint8_t* __restrict__ k_scales, const uint8_t* __restrict__ v_scales,
    const int32_t* __restrict__ ids, int seq_len, int Hkv, int D, int num_blocks,
    float* __restrict__ out_k, float* __restrict__ out_v) {
  const int b = blockIdx.x, h = blockIdx.y;
  const int32_t id = ids[b];
  const bool ok = id >= 0 && id < num_blocks;
  const int64_t slice = (int64_t)(ok ? id : 0) * Hkv + h;
  const float ks = ok ? scale_of(k_scales[slice]) : 0.f;
  const float vs = ok ? scale_of(v_scales[slice]) : 0.f;
  const int8_t* k = k_cache + slice * (kBlock * D);
  const int8_t* v = v_cache + slice * (kBlock * D);
  const int n = min(kBlock, seq_len - b * kBlock);
  for (int i = threadIdx.x; i < n * D; i += 256) {
    const int t = i / D, d = i % D;
    const int64_t at = ((int64_t)(b * kBlock + t) * Hkv + h) * D + d;
    out_k[at] = ok ? (float)k[t * D + d] * ks : 0.f;
    out_v[at] = ok ? (float)v[d * kBlock + t] * vs : 0.f;
  }
}

}  // namespace
}  // namespace pa

using namespace pa;

extern "C" int32_t pa_append_int8(int8_t* k_cache, int8_t* v_cache, uint8_t* k_scales,
                                  uint8_t* v_scales, const void* key, int64_t key_stride,
                                  const void* value, int64_t value_stride, void* q,
                                  int64_t q_stride, const float* inv_freq,
                                  const int32_t* block_tables, int32_t max_blocks_per_seq,
                                  const int32_t* cu_seq_tokens, const int32_t* context_lens,
                                  int32_t num_seqs, int32_t num_tokens, int32_t max_tokens,
                                  int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                                  int32_t num_blocks, int32_t dtype, pa_stream_t stream) {
  clear_error();
  PA_REQUIRE(dtype_ok(dtype), PA_ERR_INVALID_ARG, "pa_append_int8: unknown dtype %d", dtype);
  PA_REQUIRE(num_seqs >= 0 && num_tokens >= 0 && max_tokens >= 0 && num_kv_heads > 0 &&
                 head_dim > 0 && num_blocks > 0 && max_blocks_per_seq > 0,
             PA_ERR_INVALID_ARG, "pa_append_int8: bad sizes");
  PA_REQUIRE(!q || num_heads > 0, PA_ERR_INVALID_ARG, "pa_append_int8: num_heads %d", num_heads);
  PA_REQUIRE(!q == !inv_freq, PA_ERR_INVALID_ARG,
             "pa_append_int8: q is rotated with inv_freq: both or neither");
  PA_REQUIRE(int8_head_dim(head_dim), PA_ERR_UNSUPPORTED, "pa_append_int8: head_dim %d", head_dim);
  if (num_seqs == 0 || num_tokens == 0 || max_tokens == 0) return PA_OK;
  PA_REQUIRE(k_cache && v_cache && k_scales && v_scales && key && value && block_tables &&
                 cu_seq_tokens && context_lens,
             PA_ERR_INVALID_ARG, "pa_append_int8: null pointer");
  PA_REQUIRE(((uintptr_t)k_cache | (uintptr_t)v_cache) % 16 == 0, PA_ERR_INVALID_ARG,
             "pa_append_int8: caches not 16-byte aligned");
  const int64_t row = (int64_t)num_kv_heads * head_dim, q_row = (int64_t)num_heads * head_dim;
  if (key_stride == 0) key_stride = row;
  if (value_stride == 0) value_stride = row;
  if (q_stride == 0) q_stride = q_row;
  PA_REQUIRE(key_stride >= row && value_stride >= row && (!q || q_stride >= q_row),
             PA_ERR_INVALID_ARG, "pa_append_int8: token strides below a row");
  // Wavefronts: a sequence's touched blocks among `chunks` of them, as many as
  // it may touch up to about 16384 in all.
  const int columns = 2 * num_kv_heads + (q ? num_heads : 0);
  const int most = std::min(max_tokens, num_tokens);
  const int64_t blocks = ((int64_t)most + kBlock - 2) / kBlock + 1;
  const int chunks =
      (int)std::max<int64_t>(1, std::min<int64_t>(blocks, 16384 / ((int64_t)num_seqs * columns)));
  PA_REQUIRE(columns <= 65535 && grid_fits((int64_t)num_seqs * chunks, 64), PA_ERR_UNSUPPORTED,
             "pa_append_int8: %d sequences, %d heads", num_seqs, columns);
  const AppendArgs a{k_cache, v_cache, k_scales, v_scales, key, value, q, key_stride, value_stride,
                     q_stride, inv_freq, block_tables, cu_seq_tokens, context_lens,
                     max_blocks_per_seq, num_tokens, max_tokens, chunks, num_heads, num_kv_heads,
                     head_dim, num_blocks};
  const int es = dtype == PA_DTYPE_BF16 ? 2 : 4;
  const bool aligned = ((uintptr_t)key | (uintptr_t)value | (uintptr_t)q) % 16 == 0 &&
                       (key_stride | value_stride | (q ? q_stride : 0)) * es % 16 == 0;
  const dim3 grid(num_seqs * chunks, columns);
  hipStream_t s = (hipStream_t)stream;
#define PA_LAUNCH_APPEND_T(T, DD)                                                       \
  (q ? (aligned ? append_int8_kernel<T, DD, true, true><<<grid, 64, 0, s>>>(a)          \
                : append_int8_kernel<T, DD, false, true><<<grid, 64, 0, s>>>(a))        \
     : (aligned ? append_int8_kernel<T, DD, true, false><<<grid, 64, 0, s>>>(a)         \
                : append_int8_kernel<T, DD, false, false><<<grid, 64, 0, s>>>(a)))
#define PA_LAUNCH_APPEND(DD) \
  (dtype == PA_DTYPE_BF16 ? PA_LAUNCH_APPEND_T(uint16_t, DD) : PA_LAUNCH_APPEND_T(float, DD))
  switch (head_dim) {
    case 32: PA_LAUNCH_APPEND(32); break;
    case 64: PA_LAUNCH_APPEND(64); break;
    case 96: PA_LAUNCH_APPEND(96); break;
    case 128: PA_LAUNCH_APPEND(128); break;
    case 192: PA_LAUNCH_APPEND(192); break;
    default: PA_LAUNCH_APPEND(256); break;
  }
#undef PA_LAUNCH_APPEND
#undef PA_LAUNCH_APPEND_T
  return check_launch("pa_append_int8");
}

extern "C" int32_t pa_read_kv_int8(const int8_t* k_cache, const int8_t* v_cache,
                                   const uint8_t* k_scales, const uint8_t* v_scales,
                                   const int32_t* block_ids, int32_t n_ids, int32_t seq_len,
                                   int32_t num_kv_heads, int32_t head_dim, int32_t num_blocks,
                                   float* out_k, float* out_v, pa_stream_t stream) {
  clear_error();
  PA_REQUIRE(n_ids >= 0 && seq_len >= 0 && num_kv_heads > 0 && head_dim > 0 && num_blocks > 0,
             PA_ERR_INVALID_ARG, "pa_read_kv_int8: bad sizes");
  PA_REQUIRE((int64_t)n_ids * kBlock >= seq_len, PA_ERR_OUT_OF_BOUNDS,
             "pa_read_kv_int8: %d block ids cannot hold %d tokens", n_ids, seq_len);
  PA_REQUIRE(num_kv_heads <= 65535 && head_dim <= 1 << 20, PA_ERR_UNSUPPORTED,
             "pa_read_kv_int8: %d heads x %d", num_kv_heads, head_dim);
  if (seq_len == 0) return PA_OK;
  PA_REQUIRE(k_cache && v_cache && k_scales && v_scales && block_ids && out_k && out_v,
             PA_ERR_INVALID_ARG, "pa_read_kv_int8: null pointer");
  const int blocks = (int)(((int64_t)seq_len + kBlock - 1) / kBlock);
  PA_REQUIRE_GRID("pa_read_kv_int8", (int64_t)blocks);
  read_kv_int8_kernel<<<dim3(blocks, num_kv_heads), 256, 0, (hipStream_t)stream>>>(
      k_cache, v_cache, k_scales, v_scales, block_ids, seq_len, num_kv_heads, head_dim, num_blocks,
      out_k, out_v);
  return check_launch("pa_read_kv_int8");
}
