// Attention of one wavefront over an int8 cache: 16 query rows (the columns of the
// matrix instructions) against a run of 16-token blocks, four blocks a step.
//
// Lanes (lane = 16 j + c):
//   Sᵀ = K·Qᵀ on v_mfma_i32_16x16x64_i8, the codes as they lie in memory.  The
//     query row is a fixed-point number of 15 bits, 2^e (128 hi + lo), hi and lo
//     int8, so a score is 128 K·hi + K·lo in exact 32-bit integers; what is rounded
//     is q alone, by at most 2^-14 of the row's largest (bf16 would round the scaled
//     q by 2^-9 of each value).  Tile kk's row 4 g + r is token 4 kk + r of block g: the
//     lane (c, j) receives query c's scores of block j, token 4 kk + r in x[4 kk + r],
//     and the block's K scale is one factor a lane.
//   Oᵀ += Vᵀ·Pᵀ on v_mfma_f32_16x16x32_bf16: a lane loads the 16 tokens of dim
//     16 dt + c of block j (16 bytes of the token-minor block), and holds their
//     probabilities already.  The codes become bf16 exactly; the V scale goes into
//     the probability, which is rounded to bf16 with it (2^-9 of each).
// All loads are 16 bytes a lane.
#pragma once

#include "int8_common.hpp"

namespace pa {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));

constexpr float kInt8Log2e = 1.4426950408889634f;
// "No maximum yet": below any score, and m - m is 0.  And where there were keys, all of
// whose scores are -inf: no maximum either, but a row of only such is no row without keys.
constexpr float kInt8NoMax = -3.0e38f;
constexpr float kInt8AllBelow = -2.9e38f;
// A row's output from its numerator, denominator and maximum: 0 for one without keys; NaN
// goes through.
__device__ inline float int8_quotient(float num, float den, float m) {
  return den != 0.f ? num / den : m == kInt8AllBelow ? __builtin_nanf("") : 0.f;
}

// Four int8 codes of w as floats, and pairs of those as bf16 (exact: the low half
// of such a float is 0).
__device__ inline uint32_t codes_bf16x2(uint32_t w, int at) {
  const float a = (float)(int8_t)(w >> (8 * at));
  const float b = (float)(int8_t)(w >> (8 * at + 8));
  return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, a),
                               0x07060302u);
}
__device__ inline void codes_bf16x16(i32x4 w, bf16x8& lo, bf16x8& hi) {
  // the words as they are: the compiler would carry bytes in registers of their own
  // from the loads to here
  asm("" : "+v"(w));
  typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
  lo = __builtin_bit_cast(bf16x8, u32x4_t{codes_bf16x2(w[0], 0), codes_bf16x2(w[0], 2),
                                          codes_bf16x2(w[1], 0), codes_bf16x2(w[1], 2)});
  hi = __builtin_bit_cast(bf16x8, u32x4_t{codes_bf16x2(w[2], 0), codes_bf16x2(w[2], 2),
                                          codes_bf16x2(w[3], 0), codes_bf16x2(w[3], 2)});
}

template <int D>
struct Int8Query {
  static constexpr int KS = (D + 63) / 64;  // reduction steps of 64 dims
  i32x4 hi[KS], lo[KS];
  // Of a score: factor 2^e, scale * log2(e) by the row's unit; NaN for a row that is not
  // finite.  (Apart, as the product may be below the floats and a score not.)
  float factor;
  int e;
};

// The 16-byte chunk of a K row that reduction step s reads in lane group j; a chunk
// past the row (dims not a multiple of 64) reads another, against zeros.
template <int D>
__device__ inline int int8_chunk(int s, int j) {
  const int ch = 4 * s + j;
  return D % 64 == 0 || ch < D / 16 ? ch : ch - 2;
}

// Splits the query row at `row` (null: zeros), dims as int8_chunk says; the lanes
// of a column hold the row's parts.
template <int D>
__device__ inline void int8_query(const uint16_t* row, int j, float scale_log2, Int8Query<D>& q) {
  constexpr int KS = Int8Query<D>::KS;
  uint32_t raw[KS][8];  // pairs of bf16
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    const bool on = row && (D % 64 == 0 || 4 * s + j < D / 16);
    struct __attribute__((aligned(4))) Half {  // rows of any 4-byte alignment
      uint32_t v[8];
    };
    Half h{};
    if (on) h = *reinterpret_cast<const Half*>(row + 16 * (4 * s + j));
#pragma unroll
    for (int i = 0; i < 8; ++i) raw[s][i] = h.v[i];
  }
  // the largest of |x| as integers: NaN and infinities are above the rest
  uint32_t top = 0;
#pragma unroll
  for (int s = 0; s < KS; ++s)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      top = max(top, max(raw[s][i] & 0x7FFFu, (raw[s][i] >> 16) & 0x7FFFu));
  top = max(top, (uint32_t)__shfl_xor((int)top, 16, 64));
  top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
  const bool worse = top >= 0x7F80u;
  const float amax = bf16_bits_to_f32((uint16_t)top);
  // |x| 2^-e < 2^14, the largest being m 2^b, m < 2, and e = b - 13.  (Subnormal rows are
  // multiples of 2^-133: exact at e = -140.)
  const uint32_t u = __builtin_bit_cast(uint32_t, amax);
  const int e = (int)(u >> 23) - 127 - 13;
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    uint32_t hw[4], lw[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) hw[i] = lw[i] = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float x = bf16_bits_to_f32((uint16_t)(raw[s][i / 2] >> (16 * (i & 1))));
      const int n = worse ? 0 : (int)rintf(ldexpf(x, -e));
      // |n| <= 2^14 - 64 (8 bits of the largest): hi from -128 to 127, lo from -63 to 64
      const int hi = (n + 63) >> 7, lo = n - 128 * hi;
      hw[i / 4] |= (uint32_t)(uint8_t)hi << (8 * (i & 3));
      lw[i / 4] |= (uint32_t)(uint8_t)lo << (8 * (i & 3));
    }
    q.hi[s] = i32x4{(int)hw[0], (int)hw[1], (int)hw[2], (int)hw[3]};
    q.lo[s] = i32x4{(int)lw[0], (int)lw[1], (int)lw[2], (int)lw[3]};
  }
  q.factor = worse ? __builtin_nanf("") : scale_log2;
  q.e = e;
}

// A wavefront's online softmax: o unnormalised, m in the log2 domain, lsum this
// lane's share of the denominator.
template <int D>
struct Int8State {
  f32x4 o[D / 16];
  float m, lsum;
  __device__ void init() {
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    m = kInt8NoMax;
    lsum = 0.f;
  }
};

// A step of four blocks: this lane's rows of K and V, and block j's scale bytes.
template <int D>
struct Int8Keys {
  static constexpr int KS = Int8Query<D>::KS;
  i32x4 k[4][KS];
  uint32_t scale;
};
template <int D>
struct Int8Values {
  i32x4 v[D / 16];
  uint32_t scale;
};

template <int D>
struct Int8Blocks {
  const int8_t* kc;
  const int8_t* vc;
  const uint8_t* ks;
  const uint8_t* vs;
  int Hkv, kvh;
  // Load a step: kid the id of block c / 4 (whose K rows this lane loads), vid that
  // of block j, both in the pool.
  __device__ inline void load_keys(int kid, int vid, int c, int j, Int8Keys<D>& st) const {
    const uint32_t slice = (uint32_t)kid * (uint32_t)Hkv + kvh;
    const int8_t* kr = kc + (uint64_t)slice * (kBlock * D) + (c & 3) * D;
    st.scale = ks[(uint32_t)vid * (uint32_t)Hkv + kvh];
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
#pragma unroll
      for (int s = 0; s < Int8Keys<D>::KS; ++s)
        st.k[kk][s] = __builtin_nontemporal_load(
            reinterpret_cast<const i32x4*>(kr + 4 * kk * D + 16 * int8_chunk<D>(s, j)));
  }
  __device__ inline void load_values(int vid, int c, Int8Values<D>& st) const {
    const uint32_t slice = (uint32_t)vid * (uint32_t)Hkv + kvh;
    const int8_t* vr = vc + (uint64_t)slice * (kBlock * D) + c * kBlock;
    st.scale = vs[slice];
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt)
      st.v[dt] = __builtin_nontemporal_load(reinterpret_cast<const i32x4*>(vr + dt * 16 * kBlock));
  }
};

// The step's scores as integers.
template <int D>
__device__ inline void int8_scores(const Int8Keys<D>& st, const Int8Query<D>& q, i32x4 (&a)[4]) {
  constexpr int KS = Int8Query<D>::KS;
#pragma unroll
  for (int kk = 0; kk < 4; ++kk) a[kk] = i32x4{0, 0, 0, 0};
#pragma unroll
  for (int s = 0; s < KS; ++s)
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
      a[kk] = __builtin_amdgcn_mfma_i32_16x16x64_i8(st.k[kk][s], q.hi[s], a[kk], 0, 0, 0);
#pragma unroll
  for (int kk = 0; kk < 4; ++kk)
#pragma unroll
    for (int r = 0; r < 4; ++r) a[kk][r] <<= 7;
#pragma unroll
  for (int s = 0; s < KS; ++s)
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
      a[kk] = __builtin_amdgcn_mfma_i32_16x16x64_i8(st.k[kk][s], q.lo[s], a[kk], 0, 0, 0);
}

// The scores into the softmax: the probabilities times the V scale, in bf16.  lim:
// tokens of block j (this lane's scores) that query c attends, 16 where `whole`
// (wavefront-uniform).
template <int D>
__device__ inline void int8_softmax(const i32x4 (&a)[4], uint32_t kscale, uint32_t vscale,
                                    const Int8Query<D>& q, bool whole, int lim, Int8State<D>& S,
                                    bf16x8& p0, bf16x8& p1) {
  // blocks that are not attended may hold any bytes
  const bool none = !whole && lim <= 0;
  // (a factor of 2^-1000 is 0, NaN stays)
  const float f = ldexpf(q.factor, none ? 0 : kscale ? q.e + (int)kscale - 127 : -1000);
  const float fv = scale_of(none ? 127 : vscale);
  float x[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = (float)a[i >> 2][i & 3] * f;
  if (!whole) {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (i >= lim) x[i] = -INFINITY;
  }
  float bm = x[0];
#pragma unroll
  for (int i = 1; i < 16; ++i) bm = fmaxf(bm, x[i]);
  // the maximum stays until a score passes it by 2^8
  if (__builtin_amdgcn_ballot_w64(bm > S.m + 8.0f)) {
    bm = fmaxf(bm, __shfl_xor(bm, 16, 64));
    bm = fmaxf(bm, __shfl_xor(bm, 32, 64));
    const float mn = fmaxf(S.m, bm);
    const float r = __builtin_amdgcn_exp2f(S.m - mn);
    S.m = mn;
    S.lsum *= r;
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) S.o[dt] *= r;
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float p = __builtin_amdgcn_exp2f(x[i] - S.m);
    S.lsum += p;
    if (i < 8)
      p0[i] = (__bf16)(p * fv);
    else
      p1[i - 8] = (__bf16)(p * fv);
  }
}

// The probabilities' product with the values.
template <int D>
__device__ inline void int8_output(const Int8Values<D>& st, const bf16x8& p0, const bf16x8& p1,
                                   Int8State<D>& S) {
#pragma unroll
  for (int dt = 0; dt < D / 16; ++dt) {
    bf16x8 lo, hi;
    codes_bf16x16(st.v[dt], lo, hi);
    S.o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(lo, p0, S.o[dt], 0, 0, 0);
    S.o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hi, p1, S.o[dt], 0, 0, 0);
    // (all the conversions first would take four times the values' registers)
    __builtin_amdgcn_sched_barrier(0);
  }
}

}  // namespace pa
