// Chunked causal attention over the int8 cache (pa_prefill_int8).
//
// A workgroup takes ROWS query rows of one sequence and kv head, a row being one
// (token, query head of the group), numbered token by token, so any group fills it.
// Keys come in tiles of KT (whole blocks).  Their codes are copied HBM -> LDS four
// tiles ahead; two tiles ahead every wavefront writes the pieces that it copied itself
// (so no barrier stands between) as bf16, exact, into one of three buffers of matrix
// operands, once for all wavefronts.
//   Sᵀ = K·Qᵀ on v_mfma_f32_16x16x32_bf16, codes by the query as it is: exact
//     products.  A lane's eight scores of a step of 32 keys are of one block: the
//     softmax's and the block's scale and the row's running maximum are one
//     multiply-add of a score.
//   Oᵀ += Vᵀ·Pᵀ, codes by probabilities that carry the V scale: its exponent goes
//     into the exponential's argument (what is below 2^-32 of it into the operands,
//     once they are written).  The denominators are one more product, of the same
//     probabilities (as rounded) by 2^-exponent, exact.
// The maximum is kept until a score passes it by 2^8.
// Bound by vector instructions (softmax, conversions) beside the products: 4 x
// 1055-2048 on 360-4096, 32 / 8 heads of 128, 360 us, 825 TFLOP/s; without the writes
// of operands 305, and a bf16 cache's kernel, which has no conversions, 306.
// KG = 2: half the wavefronts take the first 32 keys of each tile, half the second,
// for launches of few rows; their results meet in LDS.
#include <algorithm>
#include <type_traits>

#include "int8_wave.hpp"
#include "lds_copy.hpp"
#include "pa_internal.hpp"

namespace pa {
namespace {

// Rows of sequence s in q, clamped to what the caller's arrays hold.
struct Rows {
  int begin, len, past;
};
__device__ inline Rows rows_of(const int32_t* __restrict__ cu_q,
                               const int32_t* __restrict__ past_lens, int s, int total_q,
                               int max_q) {
  const int begin = min(max(cu_q[s], 0), total_q);
  const int end = min(max(cu_q[s + 1], begin), total_q);
  return {begin, min(end - begin, max_q), max(past_lens[s], 0)};
}

template <int V>
using IC = std::integral_constant<int, V>;

__device__ inline float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

struct PrefillArgs {
  uint16_t* out;
  const uint16_t* q;
  int64_t q_row;
  const int8_t* kc;
  const int8_t* vc;
  const uint8_t* ks;
  const uint8_t* vs;
  const int32_t* tables;
  const int32_t* cu_q;
  const int32_t* past_lens;
  int mbs, Hq, Hkv, G, num_blocks, B, total_q, max_q, tiles_per_seq;
  float scale_log2;
};

// The least exponent of a V scale that the probabilities carry.  They are bf16 and the
// denominators are theirs, so a weight below 2^(-126 - e) of the row's largest is lost:
// with all of e (-126 in a block of zeros) every weight below 1.  What is below goes
// into the values, which stay normal numbers (2^-126 is the least scale).
constexpr int kLeast = -32;

template <int D>
constexpr int key_tile() {  // keys a tile: three buffers of K and V fit LDS
  return D <= 128 ? 64 : 32;
}

template <int D>
constexpr int max_seqs() {  // whose tiles a launch numbers through, beside the tiles in LDS
  return D <= 192 ? 256 : 128;
}

template <int D, int NT, int W, int KG>
__global__ __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(W / 4))) void
prefill_int8_kernel(const PrefillArgs a) {
  constexpr int KS = D / 32;  // reduction steps of the scores
  constexpr int DT = D / 16;  // tiles of the output
  constexpr int KT = key_tile<D>(), NB = KT / kBlock;
  constexpr int SPT = KT / 32 / KG;  // a wavefront's steps a tile
  static_assert(SPT >= 1, "a step for every group of wavefronts");
  // EARLY: K's operands are read two steps ahead, where the tile is there.
  constexpr bool EARLY = SPT == 2;
  constexpr int NBUF = 3;  // operand buffers; tile kt + 2 is written during tile kt
  constexpr int ROWS = 16 * NT * (W / KG);
  constexpr int T = 64 * W;
  // LDS rows of 2 mod 4 16-byte chunks: an operand read (16 rows, 4 chunks of each)
  // runs at 248 bytes a clock, at 128 with an odd number and at 32 with rows of 256
  // bytes
  constexpr int KROW = D * 2 + 32, VROW = KT * 2 + 32;
  static_assert(KROW / 16 % 4 == 2 && VROW / 16 % 4 == 2, "LDS rows");
  constexpr int PIECES = 2 * KT * D / 16;  // 16-byte pieces of a tile, K's then V's
  constexpr int CHUNKS = PIECES / 64;      // of a wavefront's copy instruction
  constexpr int PPT = (CHUNKS + W - 1) / W;
  constexpr int GT = 64 / NB;  // tiles whose blocks' ids and scales 64 lanes hold
  struct Tiles {
    uint8_t k[NBUF][KT * KROW], v[NBUF][D * VROW];
  };
  __shared__ __attribute__((aligned(16))) Tiles lds;
  __shared__ __attribute__((aligned(1024))) uint8_t stage[2][PIECES * 16];
  constexpr int kMaxSeqs = max_seqs<D>();
  __shared__ int rank_seq[kMaxSeqs], rank_begin[kMaxSeqs], rank_len[kMaxSeqs],
      rank_past[kMaxSeqs], rank_tile0[kMaxSeqs], rank_of[kMaxSeqs], tile0_of[kMaxSeqs];
  __shared__ int tiles_in_all;
  __shared__ float rest_of[64];  // see apply_rest

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, j = lane >> 4;
  const int G = a.G, B = a.B;
  auto tiles_of = [&](int len) -> int { return (len * G + ROWS - 1) / ROWS; };

  // Work items: ROWS rows of a sequence for one kv head.  The sequences' tiles are
  // numbered through, those with the most keys first and within one the later
  // (longer) tiles first, by ranks and prefix sums formed in LDS (up to kMaxSeqs
  // sequences; beyond, tiles_per_seq for each in index order).  A kv head's items go
  // to one XCD, or to its share of them, whose L2 then holds its K and V; an XCD's
  // workgroups take its items in rounds, forth and back, which pairs long and short
  // ones.
  const bool compact = B <= kMaxSeqs;
  if (compact) {
    for (int b = tid; b < B; b += T) rank_of[b] = tile0_of[b] = 0;
    __syncthreads();
    for (int o0 = 0; o0 < B; o0 += 64) {
      const Rows ro = rows_of(a.cu_q, a.past_lens, min(o0 + lane, B - 1), a.total_q, a.max_q);
      const int okey = ro.past + ro.len, otiles = tiles_of(ro.len), n = min(B - o0, 64);
      for (int b0 = 0; b0 < B; b0 += 64) {
        const int b = b0 + lane;
        int key = okey;
        if (b0 != o0) {
          const Rows r = rows_of(a.cu_q, a.past_lens, min(b, B - 1), a.total_q, a.max_q);
          key = r.past + r.len;
        }
        int rank = 0, before = 0;
        for (int i = wave; i < n; i += W) {
          const int ko = __builtin_amdgcn_readlane(okey, i);
          const bool first = ko > key || (ko == key && o0 + i < b);
          rank += first;
          before += first ? __builtin_amdgcn_readlane(otiles, i) : 0;
        }
        if (b < B && rank > 0) {
          atomicAdd(&rank_of[b], rank);
          atomicAdd(&tile0_of[b], before);
        }
      }
    }
    __syncthreads();
    for (int b = tid; b < B; b += T) {
      const Rows r = rows_of(a.cu_q, a.past_lens, b, a.total_q, a.max_q);
      const int rank = rank_of[b], before = tile0_of[b];
      rank_seq[rank] = b;
      rank_begin[rank] = r.begin;
      rank_len[rank] = r.len;
      rank_past[rank] = r.past;
      rank_tile0[rank] = before;
      if (rank == B - 1) tiles_in_all = before + tiles_of(r.len);
    }
    __syncthreads();
  }
  const int nq = compact ? tiles_in_all : B * a.tiles_per_seq;  // tiles a kv head
  const int xcd = (int)(blockIdx.x % 8), nslot = (int)(gridDim.x / 8), slot = (int)(blockIdx.x / 8);
  // the XCD's item i is tile (t0 + i * dt) % nq of head g0 + (t0 + i * dt) / nq
  int g0 = 0, t0 = 0, dt_items = 1, items;
  const int Hkv = a.Hkv;
  if (Hkv == 1 || Hkv == 2 || Hkv == 4 || Hkv == 8) {
    const int sh = Hkv == 1 ? 3 : Hkv == 2 ? 2 : Hkv == 4 ? 1 : 0;
    dt_items = 1 << sh;
    g0 = xcd >> sh;
    t0 = xcd & (dt_items - 1);
    items = t0 < nq ? (nq - t0 + dt_items - 1) >> sh : 0;
  } else {
    const int total = Hkv * nq, per_xcd = (total + 7) / 8;
    t0 = min(total, xcd * per_xcd);
    items = min(total, t0 + per_xcd) - t0;
  }

  auto process = [&](int item) {
    int kvh = g0, qt = t0 + item * dt_items;
    if (qt >= nq) {
      kvh += qt / nq;
      qt %= nq;
    }
    __syncthreads();  // every wavefront is done with the previous item's LDS
    int seq, tile;
    Rows qr;
    if (compact) {
      int r = -1;  // the last rank whose tiles begin at or before this one
      for (int b0 = 0; b0 < B; b0 += 64)
        r += __builtin_popcountll(__builtin_amdgcn_ballot_w64(
            b0 + lane < B && rank_tile0[min(b0 + lane, B - 1)] <= qt));
      seq = __builtin_amdgcn_readfirstlane(rank_seq[r]);
      qr.begin = __builtin_amdgcn_readfirstlane(rank_begin[r]);
      qr.len = __builtin_amdgcn_readfirstlane(rank_len[r]);
      qr.past = __builtin_amdgcn_readfirstlane(rank_past[r]);
      tile = tiles_of(qr.len) - 1 - (qt - __builtin_amdgcn_readfirstlane(rank_tile0[r]));
    } else {
      seq = qt / a.tiles_per_seq;
      tile = a.tiles_per_seq - 1 - qt % a.tiles_per_seq;
      qr = rows_of(a.cu_q, a.past_lens, seq, a.total_q, a.max_q);
    }
    const int rows = qr.len * G, past = qr.past;
    if (tile * ROWS >= rows) return;  // uniform over the workgroup
    const int last_token = (min(rows, (tile + 1) * ROWS) - 1) / G;
    const int64_t cap = (int64_t)a.mbs * kBlock;
    const int key_end = (int)min((int64_t)past + last_token + 1, cap);
    const int n_kt = (key_end + KT - 1) / KT;
    const int nblk = (key_end + kBlock - 1) / kBlock;
    const int32_t* tab = a.tables + (int64_t)seq * a.mbs;

    // KG = 2: wavefronts W / 2 .. take the second 32 keys of every tile
    const int kgrp = KG == 2 ? wave / (W / 2) : 0, wt = KG == 2 ? wave % (W / 2) : wave;
    const int r0 = tile * ROWS + wt * 16 * NT;  // first row of this wavefront
    const bool active = r0 < rows;

    // ---- the blocks' places and scales: lane t holds those of block t of a group of GT
    // tiles.  Blocks behind the last read the last, ids outside the pool block 0.
    const float scale = fabsf(a.scale_log2);
    auto load_ids = [&](int group) -> int32_t {
      return tab[min(group * 64 + lane, nblk - 1)];
    };
    auto place_of = [&](int32_t id) -> uint32_t {
      return (uint32_t)(id >= 0 && id < a.num_blocks ? id : 0) * (uint32_t)Hkv + kvh;
    };
    uint32_t places = place_of(load_ids(0));  // of the tiles copied
    int32_t ids_next = load_ids(1);
    // K's scale bytes, V's << 8, of the next group
    uint32_t bytes_next = (uint32_t)a.ks[places] | (uint32_t)a.vs[places] << 8;
    // of the tiles computed: the scores' factor, and 2^-e twice in bf16, e being the V
    // scale's exponent as far as the probabilities carry it: kLeast to 126, whose 2^-e is
    // a normal number
    float factors;
    uint32_t units;
    auto carried = [&](uint32_t v) -> uint32_t {  // e + 127
      return min(max(v, 127u + kLeast), 253u);
    };
    auto next_scales = [&]() {
      factors = scale * scale_of(bytes_next & 255);
      units = (254 - carried(bytes_next >> 8)) * 0x00800080u;
    };
    next_scales();
    // ---- staging: wavefront w copies and writes pieces 64 (w + n W) + lane.  Piece
    // i < KT D / 16 is chunk i % (D / 16) of key i / (D / 16); the others are dim i' % D
    // of block i' / D.
    auto copy_tile = [&](int kt) {
      if (kt % GT == 0 && kt > 0) {
        places = place_of(ids_next);
        ids_next = load_ids(kt / GT + 1);
        bytes_next = (uint32_t)a.ks[places] | (uint32_t)a.vs[places] << 8;
      }
#pragma unroll
      for (int n = 0; n < PPT; ++n) {
        const int ch = wave + n * W;
        if (CHUNKS % W != 0 && ch >= CHUNKS) continue;
        const bool is_k = ch < CHUNKS / 2;
        const int i = (is_k ? ch : ch - CHUNKS / 2) * 64 + lane;
        const uint64_t off = (uint64_t)(uint32_t)__shfl((int)places, kt % GT * NB + i / D, 64) *
                                 (kBlock * D) +
                             (uint32_t)(i % D) * 16;
        const uint32_t to = (uint32_t)(uintptr_t)(
            __attribute__((address_space(3))) uint8_t*)&stage[kt & 1][ch * 1024];
        lds_copy16((const uint8_t*)(is_k ? a.kc : a.vc), off,
                   __builtin_amdgcn_readfirstlane(to));
      }
    };
    // Waits for this wavefront's copies of a tile, those of the next one (`more`) in
    // flight, and writes the tile's operands.
    auto write_tile = [&](int kt, int buf, bool more) {
      if (!more)
        wait_vm<0>();
      else if (CHUNKS % W == 0 || wave + (PPT - 1) * W < CHUNKS)
        wait_vm<PPT>();
      else
        wait_vm<PPT - 1>();
      asm volatile("" ::: "memory");
#pragma unroll
      for (int n = 0; n < PPT; ++n) {
        const int ch = wave + n * W;
        if (CHUNKS % W != 0 && ch >= CHUNKS) continue;
        const bool is_k = ch < CHUNKS / 2;
        const int i = (is_k ? ch : ch - CHUNKS / 2) * 64 + lane;
        const i32x4 raw = *reinterpret_cast<const i32x4*>(&stage[kt & 1][ch * 1024 + lane * 16]);
        uint8_t* to;
        if (is_k) {
          // key 32 s + 8 g + 4 kk + r sits at row 32 s + 16 kk + 4 g + r: the lanes of
          // an operand read take consecutive rows
          const int key = i / (D / 16), x = i % (D / 16);
          const int r = (key & ~31) + ((key >> 2) & 1) * 16 + ((key >> 3) & 3) * 4 + (key & 3);
          to = &lds.k[buf][r * KROW + x * 32];
        } else {
          to = &lds.v[buf][(i % D) * VROW + (i / D) * 32];
        }
        bf16x8 first, second;
        codes_bf16x16(raw, first, second);
        reinterpret_cast<bf16x8*>(to)[0] = first;
        reinterpret_cast<bf16x8*>(to)[1] = second;
      }
    };
    // What V's scales leave for the operands: this wavefront's pieces of a tile that it has
    // written (they are its own until the next barrier) times the rest, 0 for scale byte 0.
    // Apart from write_tile, word by word and from LDS, for the time and registers of
    // tiles without.
    int rest_at = 0;  // the next tile that may have a rest
    auto apply_rest = [&](int kt, int buf) {
      if (kt % GT == 0) {  // (its group's bytes are the last loaded)
        const uint32_t v = bytes_next >> 8, r = v ? 127 + v - carried(v) : 0;
        const bool any = __builtin_amdgcn_ballot_w64(r != 127) != 0;
        rest_at = any ? kt : kt + GT;
        if (!any) return;
        rest_of[lane] = scale_of(r);  // (every wavefront writes the same)
      }
#pragma unroll 1
      for (int ch = wave; ch < CHUNKS; ch += W) {
        if (ch < CHUNKS / 2) continue;
        const int i = (ch - CHUNKS / 2) * 64 + lane;
        const float by = rest_of[kt % GT * NB + i / D];
        uint32_t* at = reinterpret_cast<uint32_t*>(&lds.v[buf][(i % D) * VROW + (i / D) * 32]);
#pragma unroll 1
        for (int m = 0; m < 8; ++m) {
          const uint32_t w = at[m];
          const float lo = __builtin_bit_cast(float, w << 16) * by;
          const float hi = __builtin_bit_cast(float, w & 0xFFFF0000u) * by;
          at[m] = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, hi),
                                        __builtin_bit_cast(uint32_t, lo), 0x07060302u);
        }
      }
    };
    // LDS writes done, then a barrier; loads to registers stay in flight.
    auto barrier = [&]() __attribute__((always_inline)) {
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
    };

    // ---- the query rows, and the table's ids
    copy_tile(0);
    if (n_kt > 1) copy_tile(1);
    bf16x8 qv[NT][KS];
    int pos[NT];  // the lane's rows' positions
    const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0;  // a negative scale, by the query
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = r0 + 16 * nt + c, rc = min(row, rows - 1);
      const int token = rc / G, h = rc - token * G;
      pos[nt] = past + token;
      const uint16_t* qp =
          a.q + (int64_t)(qr.begin + token) * a.q_row + (int64_t)(kvh * G + h) * D + 8 * j;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        struct __attribute__((aligned(4))) Piece {  // rows of any 4-byte alignment
          uint32_t v[4];
        };
        const Piece p = *reinterpret_cast<const Piece*>(qp + 32 * s);
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = row < rows ? p.v[i] ^ flip : 0;
        typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
        qv[nt][s] = __builtin_bit_cast(bf16x8, u32x4_t{w[0], w[1], w[2], w[3]});
      }
    }
    int bad = 0;
    for (int b = tid; b < nblk; b += T) {
      const int32_t id = tab[b];
      bad |= id < 0 || id >= a.num_blocks ? 1 : 0;
    }
    const bool bad_ids = __syncthreads_or(bad) != 0;
    f32x4 o[NT][DT];
    f32x4 lacc[NT];  // denominators
    float nm[NT];    // minus the rows' maxima; kNone: none yet
    constexpr float kNone = 3.0e38f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      nm[nt] = kNone;
      lacc[nt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[nt][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    // the first two tiles' operands, the next two on their way
    write_tile(0, 0, n_kt > 1);
    if (n_kt > 2) copy_tile(2);
    if (n_kt > 1) {
      write_tile(1, 1, n_kt > 2);
      if (n_kt > 3) copy_tile(3);
    }
    apply_rest(0, 0);
    if (n_kt > 1 && rest_at <= 1) apply_rest(1, 1);
    barrier();

    f32x4 S[NT][2];
    bf16x8 ka[2][KS], va[DT], pb[NT];
    auto qk_load = [&](int buf, int st) __attribute__((always_inline)) {
      const uint8_t* p = &lds.k[buf][(st * 32 + c) * KROW + j * 16];
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int s = 0; s < KS; ++s)
          ka[kk][s] = *reinterpret_cast<const bf16x8*>(p + kk * 16 * KROW + s * 64);
    };
    auto v_load = [&](int buf, int st) __attribute__((always_inline)) {
      const uint8_t* p = &lds.v[buf][c * VROW + st * 64 + j * 16];
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        va[dt] = *reinterpret_cast<const bf16x8*>(p + dt * 16 * VROW);
    };
    auto scores = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int kk = 0; kk < 2; ++kk)
            S[nt][kk] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                ka[kk][s], qv[nt][s], s == 0 ? f32x4{0.f, 0.f, 0.f, 0.f} : S[nt][kk], 0, 0, 0);
    };
    auto next_buf = [](int buf, int n) -> int { return buf + n >= NBUF ? buf + n - NBUF : buf + n; };
    qk_load(0, kgrp);
    scores();
    if constexpr (EARLY) qk_load(0, 1);
    const int last_pos = past + (min(rows, r0 + 16 * NT) - 1) / G;  // of this wavefront's rows

    // During tile kt: this wavefront's share of the tile two on, and the copies of the
    // one four on.
    auto prepare = [&](int kt, int buf) __attribute__((always_inline)) {
      if (kt + 2 >= n_kt) return;
      write_tile(kt + 2, next_buf(buf, 2), kt + 3 < n_kt);
      if (__builtin_expect(kt + 2 >= rest_at, 0)) apply_rest(kt + 2, next_buf(buf, 2));
      if (kt + 4 < n_kt) copy_tile(kt + 4);
    };
    // A step of 32 keys, step `st` of tile kt (in buffer buf): probabilities of S, the
    // next S, the products with V, the operands of the steps after.  A tile's first
    // step begins with a barrier: behind it the next tile is in LDS, written during the
    // one before, and the buffer of that one is free.
    auto step = [&](int buf, int st, auto first_, int kt) {
      constexpr bool FIRST = decltype(first_)::value;
      const int kb = kt * KT + st * 32;
      const bool live = active && kb <= last_pos;
      if (FIRST && kt > 0) {
        if (kt % GT == 0) next_scales();
        barrier();
      }
      if (live) {
        if constexpr (!EARLY) qk_load(next_buf(buf, 1), kgrp);
        // the scales of the lane's block
        const int at = 4 * (kt % GT * NB + 2 * st) + 4 * (j >> 1);
        float f = __builtin_bit_cast(
            float, __builtin_amdgcn_ds_bpermute(at, __builtin_bit_cast(int, factors)));
        const uint32_t one = __builtin_amdgcn_ds_bpermute(at, (int)units);
        const float e = (float)(127 - (int)(one >> 23));
        const bool tail = kt * KT + KT > key_end || bad_ids;
        if (tail || kb + 31 > past + r0 / G) {
          // keys behind the last, in blocks outside the pool or above a row's diagonal
          int end = key_end;
          if (bad_ids) {
            const int b = kt * NB + 2 * st + (j >> 1);
            const int32_t id = b < nblk ? tab[b] : -1;
            end = id >= 0 && id < a.num_blocks ? key_end : 0;
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int key = kb + 8 * j + i;
              const float x = S[nt][i >> 2][i & 3] * f;
              S[nt][i >> 2][i & 3] = key >= end || key > pos[nt] ? -INFINITY : x;
            }
          f = 1.f;
        }
        float lm[NT];
        bool need = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float m0 = max3(S[nt][0][0], S[nt][0][1], S[nt][0][2]);
          const float m1 = max3(S[nt][0][3], S[nt][1][0], S[nt][1][1]);
          lm[nt] = max3(m0, m1, max3(S[nt][1][2], S[nt][1][3], S[nt][1][3])) * f;
          // (a row without keys so far: any score passes, and -inf + kNone does not)
          need |= lm[nt] + nm[nt] > 8.0f;
        }
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(need) != 0, 0)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float top = fmaxf(lm[nt], -nm[nt]);
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            const float r = __builtin_amdgcn_exp2f(-nm[nt] - top);
            nm[nt] = -top;
            lacc[nt] *= r;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[nt][dt] *= r;
          }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float shift = nm[nt] + e;
#pragma unroll
          for (int i = 0; i < 8; ++i)
            pb[nt][i] = (__bf16)__builtin_amdgcn_exp2f(
                __builtin_fmaf(S[nt][i >> 2][i & 3], f, shift));
        }
        // between the softmax and the products, which the other wavefront of this SIMD
        // runs meanwhile (4 x 1100-2048 tokens on 100-4096, 32 / 8 heads of 128: 24 us
        // less than at the step's end, 50 less than behind the scores)
        if constexpr (FIRST) prepare(kt, buf);
        scores();
        // (where K's operands are of no use any more: with both at once, head_dim 256
        // keeps 68 registers in scratch and takes 149 us for 90, 128 keeps 12 and 368
        // for 357)
        v_load(buf, st);
        // (past the last tile what is read here is never used)
        if constexpr (EARLY) qk_load(next_buf(buf, 1), st);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            o[nt][dt] =
                __builtin_amdgcn_mfma_f32_16x16x32_bf16(va[dt], pb[nt], o[nt][dt], 0, 0, 0);
        typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
        const bf16x8 ones = __builtin_bit_cast(bf16x8, u32x4_t{one, one, one, one});
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          lacc[nt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, pb[nt], lacc[nt], 0, 0, 0);
      }
      if (FIRST && !live) prepare(kt, buf);
    };

    for (int kt = 0, buf = 0; kt < n_kt; ++kt, buf = next_buf(buf, 1)) {
      step(buf, SPT == 2 ? 0 : kgrp, std::true_type{}, kt);
      if constexpr (SPT == 2) step(buf, 1, std::false_type{}, kt);
    }

    if constexpr (KG == 2) {
      // The two groups' results, in the tiles' space.  A group that saw no key of a
      // row (nm = kNone) drops out.
      static_assert(W / 2 * NT * (DT * 1024 + 512) <= (int)sizeof(Tiles), "space");
      float* mo = reinterpret_cast<float*>(&lds);
      float* mml = mo + W / 2 * NT * DT * 256;
      __syncthreads();
      if (kgrp == 1) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int dt = 0; dt < DT; ++dt)
            *reinterpret_cast<f32x4*>(mo + ((wt * NT + nt) * DT + dt) * 256 + lane * 4) =
                o[nt][dt];
          *reinterpret_cast<float2*>(mml + ((wt * NT + nt) * 64 + lane) * 2) =
              float2{-nm[nt], lacc[nt][0]};
        }
      }
      __syncthreads();
      if (kgrp == 1) return;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float2 ml = *reinterpret_cast<const float2*>(mml + ((wt * NT + nt) * 64 + lane) * 2);
        const float m = -nm[nt], mx = fmaxf(m, ml.x);
        const float fa = __builtin_amdgcn_exp2f(m - mx), fb = __builtin_amdgcn_exp2f(ml.x - mx);
        // (a row of NaN has no maximum, but sums of NaN)
        lacc[nt][0] = lacc[nt][0] * fa + ml.y * fb;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
          o[nt][dt] = o[nt][dt] * fa + *reinterpret_cast<const f32x4*>(
                                           mo + ((wt * NT + nt) * DT + dt) * 256 + lane * 4) * fb;
      }
    }

    if (!active) return;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = r0 + 16 * nt + c;
      if (row >= rows) continue;
      const int token = row / G, h = row - token * G;
      const float l = lacc[nt][0];
      float inv = 1.f / l;
      if (l == 0.f) {
        // no keys, or all its scores are -inf (an infinity in q, against codes of one
        // sign): 0 or, as other rows of infinities have it, NaN
        bool keys = !bad_ids;
        for (int b = 0; !keys && b <= min(pos[nt], key_end - 1) / kBlock; ++b)
          keys = (uint32_t)tab[b] < (uint32_t)a.num_blocks;
        inv = keys ? __builtin_nanf("") : 0.f;
      }
      uint16_t* to = a.out + ((int64_t)(qr.begin + token) * a.Hq + kvh * G + h) * D + 4 * j;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        struct __attribute__((aligned(8))) Four {
          uint16_t v[4];
        } w;
#pragma unroll
        for (int r = 0; r < 4; ++r) w.v[r] = f32_to_bf16_bits(o[nt][dt][r] * inv);
        *reinterpret_cast<Four*>(to + 16 * dt) = w;
      }
    }
  };
  for (int r = 0; r * nslot < items; ++r) {
    const int item = r * nslot + ((r & 1) ? nslot - 1 - slot : slot);
    if (item < items) process(item);
  }
}

int compute_units() {
  static const int cus = [] {
    int dev = 0, n = 0;
    if (hipGetDevice(&dev) != hipSuccess ||
        hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess)
      n = 256;
    return std::max(n, 8);
  }();
  return cus;
}

template <int D, int NT, int W, int KG>
int32_t launch(const PrefillArgs& args, int num_seqs, hipStream_t s) {
  PrefillArgs a = args;
  constexpr int ROWS = 16 * NT * (W / KG);
  a.tiles_per_seq = (int)(((int64_t)a.max_q * a.G + ROWS - 1) / ROWS);
  const long long total = (long long)num_seqs * a.Hkv * a.tiles_per_seq;
  PA_REQUIRE(total < (1ll << 31) / 8 && (int64_t)a.max_q * a.G < (1ll << 31) - ROWS,
             PA_ERR_UNSUPPORTED, "pa_prefill_int8: launch too large");
  const int per_xcd = (int)((total + 7) / 8);
  // a multiple of the 8 XCDs, about one workgroup per CU
  const dim3 grid(8 * std::max(1, std::min(per_xcd, compute_units() / 8)));
  prefill_int8_kernel<D, NT, W, KG><<<grid, 64 * W, 0, s>>>(a);
  return PA_OK;
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
  PA_REQUIRE((int64_t)max_blocks_per_seq * kBlock < (1ll << 31) - 4096 &&
                 (long long)num_blocks * num_kv_heads < (1ll << 32),
             PA_ERR_UNSUPPORTED, "pa_prefill_int8: launch too large");
  const int G = num_heads / num_kv_heads;
  const PrefillArgs a{(uint16_t*)out, (const uint16_t*)q, q_row, k_cache, v_cache, k_scales,
                      v_scales, block_tables, cu_q_lens, past_lens, max_blocks_per_seq, num_heads,
                      num_kv_heads, G, num_blocks, num_seqs, total_q, max_q_len, 0,
                      scale * kInt8Log2e};
  // Rows a workgroup: an item's time is its keys times the time a tile takes, and a
  // launch's items share the CUs; the lengths are on the device, so the items are
  // counted from the totals.  us for 256 / 128 / 64 rows: 4 prompts of 2048, 32 / 8
  // heads of 128, 182 / 245 / 397; one of 2048 79 / 65 / 102; one of 512 on 1024
  // 61 / 45 / 40; 64 x 16 on 500 48 / 38 / 39; 1624 tokens of two, 24 / 4 heads of 96,
  // 100 / 74 / 94; one of 333, 14 / 2 heads of 64, 16 / 12 / 10.  (128 rows as two groups of keys,
  // 72, 48 and 47 where 65, 45 and 38; 64 rows of one group 135, 51 and 45.)
  auto cost = [&](int rows, double per_tile) -> double {
    const double tiles = std::max((double)num_seqs, (double)total_q * G / rows + 0.5 * num_seqs);
    return per_tile * std::max(1., 0.65 / 256 * tiles * num_kv_heads);
  };
  const double c256 = cost(256, 1.), c128 = cost(128, 0.72), c64 = cost(64, 0.62);
  auto narrow = [&](auto dc) -> int32_t {
    constexpr int DD = decltype(dc)::value;
    if (c256 <= c128 && c256 <= c64) return launch<DD, 2, 8, 1>(a, num_seqs, s);
    if (c128 <= c64) return launch<DD, 1, 8, 1>(a, num_seqs, s);
    return launch<DD, 1, 8, 2>(a, num_seqs, s);
  };
  // (the registers of the wide heads hold 16 rows a wavefront: 134 us where four
  // wavefronts of 32 rows took 199, 700 tokens on 1000 and 300, 16 / 4 heads of 256)
  auto wide = [&](auto dc) -> int32_t {
    constexpr int DD = decltype(dc)::value;
    return launch<DD, 1, 8, 1>(a, num_seqs, s);
  };
  int32_t rc;
  switch (head_dim) {
    case 32: rc = narrow(IC<32>{}); break;
    case 64: rc = narrow(IC<64>{}); break;
    case 96: rc = narrow(IC<96>{}); break;
    case 128: rc = narrow(IC<128>{}); break;
    case 192: rc = wide(IC<192>{}); break;
    default: rc = wide(IC<256>{}); break;
  }
  if (rc != PA_OK) return rc;
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
