// pa_linear_mx: Y[M, N] = X[M, K] · W[N, K]ᵀ on MXFP8 rows and weights
// (layouts: include/pa_dense.h), a tiled GEMM on the scaled matrix
// instructions.  Times here are a call's on the device, calls in a row, over sets
// of operands that together pass the last-level cache (large products: three
// sets).
#include <algorithm>
#include <type_traits>

#include "lds_copy.hpp"
#include "mx_common.hpp"
#include "mx_tiling.hpp"
#include "pa_common.hpp"
#include "pa_internal.hpp"
#include "../../include/pa_dense.h"

namespace pa {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
// at the alignment of a row of bf16 (the memory takes it whole)
typedef int i32x4u __attribute__((ext_vector_type(4), aligned(2)));
typedef uint64_t u64u __attribute__((aligned(2)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

struct MxLinear {
  void* out;
  uint8_t* out_scales;
  const uint8_t *x, *xs, *w, *ws;
  const uint16_t *bias, *residual;
  int M, N;
  int steps;      // of 128 columns
  int64_t pad_m;  // rows of a scale column of x (and of the output)
};

// Workgroup = KG groups of WM x WN wavefronts.  Wavefront (wm, wn) of a group
// computes TM x TN tiles of 32 x 32 (v_mfma_scale_f32_32x32x64_f8f6f4), so the
// workgroup tile is BM = 32 WM TM rows of X by BN = 32 WN TN rows of W.  Group
// kg takes the K steps (128 columns) kg, KG + kg, ..., and the groups' sums
// meet in LDS at the end.  A stage is one step of every group, copied HBM ->
// LDS into one of S buffers, S - 1 stages ahead of use, one barrier per stage.
//
// LDS, per step: X rows of 128 bytes with their 16-byte chunks XOR-swizzled by
// the row (the 16 rows that an operand read serves at once hit distinct bank
// slots), W fragments as they lie in memory, one scale dword per row of each.
// Operands of a product over 64 columns: lane (n, g) = (lane % 32, lane / 32)
// holds columns 16 g .. + 15 and 32 + 16 g .. + 15 of row n, and the scale
// byte of columns 32 g .. + 31.  The products compute the transposed tile (A =
// W, B = X): lane (n, g) holds X row n and, in register r, output column
// 8 (r / 4) + 4 g + r % 4.
//
// SILU: the tile's BN weight rows are BN/2 gate rows, then the matching up
// rows; a wavefront takes TN/2 gate tiles and their up tiles.
//
// 256 x 256 tiles read the fewest operand bytes per product, and their four
// wavefronts, one per SIMD, hold the accumulators in 256 registers each (and
// three that only the epilogues read in scratch).  Times and rates (normal
// values): 7569 x 4096 x 4096 112 us, 2270 TFLOP/s, with the residual 123, in
// place 117; 8192^3 412 us, 2670; gate|up 2048 x 24576 x 4096 with its codes 166
// us, 2480, in bf16 169 (a library's product alone, one scale per matrix: 103, 381
// and 143 us).  Bound by the matrix units' power: on zeros 8192^3 takes 375 us
// (without the copies 280), on normal values products alone reach 3590 TFLOP/s of the 4700 on
// zeros.  Fetching lines into L2 ahead of the copies took zeros to 318 us and
// normal values to 409, at the first two sizes nothing, and is left out.  Fewer
// tiles than fill the chip: the copies' latency, see mx_tiling.hpp.
template <bool SILU, int WM, int WN, int TM, int TN, int KG, int S>
__global__ __launch_bounds__(64 * WM * WN * KG) void mx_gemm_kernel(const MxLinear p, int ntm,
                                                                    int ntn) {
  constexpr int GW = WM * WN, NT = 64 * GW * KG;
  constexpr int BM = 32 * WM * TM, BN = 32 * WN * TN, BNO = SILU ? BN / 2 : BN;
  constexpr int CA = BM / 8 / GW, CB = BN / 8 / GW;         // 1 KB copies per wavefront
  constexpr int BS = (BN + 63) / 64 * 64;                 // scales of W: 64 rows a copy
  constexpr int SC = (BM + BS) / 64, CS = (SC + GW - 1) / GW;  // 256 B copies of scales
  constexpr int PER = CA + CB + CS;
  static_assert(CA * GW * 8 == BM && CB * GW * 8 == BN && BM % 64 == 0 &&
                    (!SILU || (TN % 2 == 0 && BN % 64 == 0)),
                "tiles");
  constexpr int STEP = (BM + BN) * 128 + (BM + BS) * 4;  // codes, then scale dwords
  constexpr int STAGE = KG * STEP;
  constexpr int SX = (BM + BN) * 128, SW = SX + BM * 4;
  constexpr int ORB = BNO * 2 + 16;  // bytes per row of the staged output tile
  constexpr int RED = BM * BN * 4 * (KG - 1);
  constexpr int SM0 = S * STAGE > BM * ORB ? S * STAGE : BM * ORB;
  constexpr int SM = SM0 > RED ? SM0 : RED;
  static_assert(SM + 4 * BN + 16 <= 160 * 1024, "LDS");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[SM];
  __shared__ __attribute__((aligned(16))) float sbias[SILU ? 4 : BN];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kg = wave / GW, wt = wave % GW;
  const int wm = wt / WN, wn = wt % WN;
  const int n = lane & 31, g = lane >> 5;
  const int M = p.M, N = p.N, nk = p.steps;
  // Tile order: workgroups are dealt round-robin to the 8 XCDs; XCD i takes
  // the i-th contiguous range of an order that goes through groups of row
  // tiles (up to 8, so that W is streamed once), column tiles outer within a
  // group, so the tiles in flight on an XCD share X and W rows in its L2.
  const uint32_t group_m = min(ntm, 8), group = group_m * (uint32_t)ntn;
  const uint32_t total = (uint32_t)ntm * ntn, per_xcd = (total + 7) / 8;
  const uint32_t tile = blockIdx.x % 8 * per_xcd + blockIdx.x / 8;
  if (blockIdx.x / 8 >= per_xcd || tile >= total) return;
  const uint32_t first_m = tile / group * group_m, in_grp = tile % group;
  const uint32_t gsz = min(group_m, ntm - first_m);
  const int m0 = (int)(first_m + in_grp % gsz) * BM;
  const int c0 = (int)(in_grp / gsz) * BNO;  // first output column
  const int tiles_n = (int)((uint32_t)(N + 15) >> 4);  // 16-row fragments of W (of its gate half)
  auto swz = [](int r) -> int { return (r / 2) % 8; };

  // This wavefront's copies of a step: scalar bases, 32-bit lane offsets.
  const uint8_t* xb = p.x + (int64_t)m0 * nk * 128;
  uint32_t xo[CA];
#pragma unroll
  for (int u = 0; u < CA; ++u) {
    const int r = (CA * wt + u) * 8 + lane / 8;
    xo[u] = (uint32_t)min(r, M - 1 - m0) * (uint32_t)(nk * 128) + ((lane % 8) ^ swz(r)) * 16;
  }
  // the fragment of W that holds row r of the tile
  auto frag = [&](int r) __attribute__((always_inline)) -> int {
    const bool up = SILU && r >= BN / 2;
    return min((c0 + (up ? r - BN / 2 : r)) >> 4, tiles_n - 1) + (up ? tiles_n : 0);
  };
  const uint8_t* wb[CB];  // half a fragment each
#pragma unroll
  for (int u = 0; u < CB; ++u) {
    const int piece = CB * wt + u;
    wb[u] = p.w + (int64_t)frag(piece * 8) * nk * 2048 + piece % 2 * 1024;
  }
  // Scales, 64 rows a copy: first X's, then W's; the last ones twice where
  // the copies do not divide among the wavefronts.
  const uint8_t* sb[CS];
  uint32_t so[CS], sl[CS];
  int64_t sstep[CS];  // bytes from one step's scales to the next's
  const int f0 = frag(0);
#pragma unroll
  for (int u = 0; u < CS; ++u) {
    const int c = (wt + GW * u) % SC, r = (c * 64 < BM ? 0 : -BM) + c * 64 + lane;
    if (c * 64 < BM) {
      sb[u] = p.xs + (int64_t)m0 * 4;
      so[u] = (uint32_t)min(r, M - 1 - m0) * 4;
      sstep[u] = p.pad_m * 4;
    } else {
      sb[u] = p.ws + (int64_t)f0 * nk * 64;
      so[u] = (uint32_t)(frag(r) - f0) * (uint32_t)(nk * 64) + r % 16 * 4;
      sstep[u] = 64;
    }
    sl[u] = SX + c * 256;
  }
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)lds;
  // copy u of a stage's PER; a group without a step in the last stage copies
  // the last step again
  auto copy = [&](int stage, int buf, int u) __attribute__((always_inline)) {
    const int kt = min(stage * KG + kg, nk - 1);
    const uint32_t l0 = lds0 + buf * STAGE + kg * STEP;
    if (u < CA)
      lds_copy16(xb + (int64_t)kt * 128, xo[u],
                 __builtin_amdgcn_readfirstlane(l0 + (CA * wt + u) * 1024));
    else if (u < CA + CB)
      lds_copy16(wb[u - CA] + (int64_t)kt * 2048, (uint32_t)lane * 16,
                 __builtin_amdgcn_readfirstlane(l0 + BM * 128 + (CB * wt + u - CA) * 1024));
    else
      lds_copy4(sb[u - CA - CB] + kt * sstep[u - CA - CB], so[u - CA - CB],
                __builtin_amdgcn_readfirstlane(l0 + sl[u - CA - CB]));
  };
  // tile rows of this lane's operands (SILU: gate tiles, then their up tiles)
  int arow[TM], brow[TN];
#pragma unroll
  for (int t = 0; t < TM; ++t) arow[t] = (wm * TM + t) * 32 + n;
#pragma unroll
  for (int t = 0; t < TN; ++t)
    brow[t] = SILU ? (t < TN / 2 ? (wn * TN / 2 + t) * 32 + n
                                 : BN / 2 + (wn * TN / 2 + t - TN / 2) * 32 + n)
                   : (wn * TN + t) * 32 + n;
  f32x16 acc[TM][TN];
#pragma unroll
  for (int a = 0; a < TM; ++a)
#pragma unroll
    for (int b = 0; b < TN; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[a][b][i] = 0.f;
  // The operands of half a step (64 columns), read while the half before is
  // multiplied, in 2 (TM + TN) reads.
  struct Half {
    i32x4 a[TM][2], b[TN][2];
  };
  constexpr int READS = 2 * (TM + TN), PRODUCTS = TM * TN;
  auto read = [&](int buf, int h, int u, Half& o) __attribute__((always_inline)) {
    const uint8_t* at = lds + buf * STAGE + kg * STEP;
    const int c = 4 * h + 2 * (u % 2) + g, t = u / 2;
    if (t < TN)
      o.b[t][u % 2] = *reinterpret_cast<const i32x4*>(at + BM * 128 + brow[t] / 16 * 2048 +
                                                      brow[t] % 16 * 16 + c * 256);
    else
      o.a[t - TN][u % 2] = *reinterpret_cast<const i32x4*>(
          at + arow[t - TN] * 128 + (c ^ swz(arow[t - TN])) * 16);
  };
  // This lane's scale bytes: of the first 64 columns in bits 0-7, of the
  // second in 16-23.
  struct Scales {
    int a[TM], b[TN];
  };
  auto read_scales = [&](int st, int buf, Scales& o) __attribute__((always_inline)) {
    const uint8_t* at = lds + buf * STAGE + kg * STEP;
    // a group without a step in the last stage multiplies by 2^-127 twice,
    // which leaves nothing in f32
    const int keep = KG == 1 || st * KG + kg < nk ? -1 : 0;
#pragma unroll
    for (int t = 0; t < TN; ++t)
      o.b[t] = (*reinterpret_cast<const int*>(at + SW + brow[t] * 4) >> (8 * g)) & keep;
#pragma unroll
    for (int t = 0; t < TM; ++t)
      o.a[t] = (*reinterpret_cast<const int*>(at + SX + arow[t] * 4) >> (8 * g)) & keep;
  };
  // Half h's products, with the next half's reads and a stage's copies
  // between them: nothing else of this wavefront would run meanwhile, and
  // a block of reads in front would leave the matrix core waiting.
  auto half = [&](auto hc, const Half& o, const Scales& s, auto&& beside)
                  __attribute__((always_inline)) {
    constexpr int h = decltype(hc)::value;
#pragma unroll
    for (int i = 0; i < PRODUCTS; ++i) {
      const int a = i / TN, b = i % TN;
      acc[a][b] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
          __builtin_shufflevector(o.b[b][0], o.b[b][1], 0, 1, 2, 3, 4, 5, 6, 7),
          __builtin_shufflevector(o.a[a][0], o.a[a][1], 0, 1, 2, 3, 4, 5, 6, 7), acc[a][b], 0, 0,
          2 * h, s.b[b], 2 * h, s.a[a]);
      beside(i);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  const int ns = (nk + KG - 1) / KG;
#pragma unroll
  for (int t = 0; t < S; ++t)
    if (t < ns)
#pragma unroll
      for (int u = 0; u < PER; ++u) copy(t, t, u);
  Half h0, h1;
  Scales sc, sn;
  int buf = 0;
  // piece i of PRODUCTS of n things, the first `early` products taking them
  auto share = [](int i, int n, int early, auto&& f) __attribute__((always_inline)) {
#pragma unroll
    for (int u = min(i, early) * n / early; u < min(i + 1, early) * n / early; ++u) f(u);
  };
  constexpr int EARLY = PRODUCTS > 4 ? PRODUCTS / 2 : PRODUCTS;
  // Stage st and the step to the one after it.  Between the halves this
  // wavefront's copies of the next stage have landed (in_flight: those of the
  // stages behind it), and after the barrier everyone's, and everyone has read
  // all of this stage, whose buffer takes the stage S further on.  No
  // branches: the compiler would move the products behind them.
  auto step = [&](int st, auto in_flight, auto copies) __attribute__((always_inline)) {
    half(std::integral_constant<int, 0>{}, h0, sc, [&](int i) __attribute__((always_inline)) {
      share(i, READS, EARLY, [&](int u) __attribute__((always_inline)) { read(buf, 1, u, h1); });
    });
    wait_copies<decltype(in_flight)::value>();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    const int nb = buf == S - 1 ? 0 : buf + 1;
    read_scales(st + 1, nb, sn);
    half(std::integral_constant<int, 1>{}, h1, sc, [&](int i) __attribute__((always_inline)) {
      share(i, READS, EARLY, [&](int u) __attribute__((always_inline)) { read(nb, 0, u, h0); });
      if constexpr (decltype(copies)::value)
        share(i, PER, PRODUCTS,
              [&](int u) __attribute__((always_inline)) { copy(st + S, buf, u); });
    });
    buf = nb;
    sc = sn;
  };
  if (ns >= S)
    wait_copies<(S - 1) * PER>();
  else
    wait_copies<0>();
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  read_scales(0, 0, sc);
#pragma unroll
  for (int u = 0; u < READS; ++u) read(0, 0, u, h0);
  int st = 0;
  for (; st < ns - S; ++st)
    step(st, std::integral_constant<int, (S - 2) * PER>{}, std::true_type{});
  for (; st < ns - 1; ++st) step(st, std::integral_constant<int, 0>{}, std::false_type{});
  half(std::integral_constant<int, 0>{}, h0, sc, [&](int i) __attribute__((always_inline)) {
    share(i, READS, EARLY, [&](int u) __attribute__((always_inline)) { read(buf, 1, u, h1); });
  });
  half(std::integral_constant<int, 1>{}, h1, sc, [](int) {});
  __syncthreads();
  // the K groups' sums, in group order
  if constexpr (KG > 1) {
    float* red = reinterpret_cast<float*>(lds);
    auto slot = [&](int z, int a, int b, int q) __attribute__((always_inline)) {
      return red + (((z * GW + wt) * TM * TN + a * TN + b) * 4 + q) * 256 + lane * 4;
    };
    if (kg > 0) {
#pragma unroll
      for (int a = 0; a < TM; ++a)
#pragma unroll
        for (int b = 0; b < TN; ++b)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *reinterpret_cast<float4*>(slot(kg - 1, a, b, q)) =
                float4{acc[a][b][4 * q], acc[a][b][4 * q + 1], acc[a][b][4 * q + 2],
                       acc[a][b][4 * q + 3]};
    }
    __syncthreads();
    if (kg == 0) {
#pragma unroll
      for (int z = 0; z < KG - 1; ++z)
#pragma unroll
        for (int a = 0; a < TM; ++a)
#pragma unroll
          for (int b = 0; b < TN; ++b)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const float4 v = *reinterpret_cast<const float4*>(slot(z, a, b, q));
              acc[a][b][4 * q] += v.x;
              acc[a][b][4 * q + 1] += v.y;
              acc[a][b][4 * q + 2] += v.z;
              acc[a][b][4 * q + 3] += v.w;
            }
    }
    __syncthreads();
  }
  // 16 bytes of every rs-th row of a staged tile out, `items` of them (of rows
  // behind M none), in batches of LDS reads, which the asm holds in front of
  // the branches: behind them the compiler reads and stores one by one (43.2 us
  // for 41.6 at 618 x 6144 x 4096 in 256 x 256 tiles).
  auto rows_out = [&](uint8_t* dst, int64_t dst_step, const uint8_t* src, auto src_step, auto items,
                      auto rs, int r0) __attribute__((always_inline)) {
    constexpr int IT = decltype(items)::value, BATCH = IT % 8 == 0 ? 8 : IT;
    constexpr int SRC = decltype(src_step)::value, R = decltype(rs)::value;
#pragma unroll
    for (int i = 0; i < IT; i += BATCH) {
      i32x4 v[BATCH];
#pragma unroll
      for (int u = 0; u < BATCH; ++u) v[u] = *reinterpret_cast<const i32x4*>(src + (i + u) * SRC);
#pragma unroll
      for (int u = 0; u < BATCH; ++u) asm volatile("" : "+v"(v[u]));
#pragma unroll
      for (int u = 0; u < BATCH; ++u, dst += dst_step)
        if (r0 + (i + u) * R < M - m0) *reinterpret_cast<i32x4u*>(dst) = v[u];
    }
  };
  if constexpr (SILU) {
    constexpr int TB = TN / 2;
    // silu(g) u, 0 in the columns behind the last (an MXFP8 output's padding)
    if (KG == 1 || kg == 0) {
#pragma unroll
      for (int a = 0; a < TM; ++a)
#pragma unroll
        for (int b = 0; b < TB; ++b) {
          const bool real = c0 + (wn * TB + b) * 32 < N;  // N is a multiple of 32
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float y = mx_silu_mul(acc[a][b][i], acc[a][b + TB][i]);
            acc[a][b][i] = real ? y : 0.f;
          }
        }
    }
    if (p.out_scales) {
      constexpr int CRB = BNO + 16, NBLK = BNO / 32;  // bytes per staged row, blocks per row
      static_assert(BM * (CRB + NBLK) <= SM, "staged codes");
      if (KG == 1 || kg == 0) {
#pragma unroll
        for (int a = 0; a < TM; ++a)
#pragma unroll
          for (int b = 0; b < TB; ++b) {
            // a block's 32 columns are this lane's 16 and those of lane ^ 32
            float y[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) y[i] = acc[a][b][i];
            uint32_t top = mx_top(y);
            top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
            const uint32_t byte = mx_scale_byte(top);
            const float inv = mx_inverse(byte);
            const int blk = wn * TB + b;
#pragma unroll
            for (int q = 0; q < 4; ++q)
              *reinterpret_cast<uint32_t*>(lds + arow[a] * CRB + blk * 32 + 8 * q + 4 * g) =
                  mx_codes4(y[4 * q], y[4 * q + 1], y[4 * q + 2], y[4 * q + 3], inv);
            if (g == 0) lds[BM * CRB + arow[a] * NBLK + blk] = (uint8_t)byte;
          }
      }
      __syncthreads();
      const int pitch = (N + 127) / 128 * 128;
      constexpr int CPR = BNO / 16, RS = NT / CPR;  // threads of a row, rows per pass
      constexpr int ITEMS = BM > RS ? BM / RS : 1;
      static_assert(RS * CPR == NT && BM % std::min(BM, RS) == 0, "whole passes");
      const int r0 = threadIdx.x / CPR, cc = threadIdx.x % CPR * 16;
      if (c0 + cc < pitch && r0 < BM)
        rows_out(static_cast<uint8_t*>(p.out) + (int64_t)(m0 + r0) * pitch + c0 + cc,
                 (int64_t)RS * pitch, lds + r0 * CRB + cc, std::integral_constant<int, RS * CRB>{},
                 std::integral_constant<int, ITEMS>{}, std::integral_constant<int, RS>{}, r0);
      // the blocks of one scale column at once
      using Bytes = std::conditional_t<NBLK == 4, uint32_t,
                                       std::conditional_t<NBLK == 2, uint16_t, uint8_t>>;
      static_assert(sizeof(Bytes) == NBLK, "scale bytes of a tile's row");
      if (c0 < pitch)
        for (int r = threadIdx.x; r < min(BM, M - m0); r += NT)
          *reinterpret_cast<Bytes*>(p.out_scales + ((c0 / 128) * p.pad_m + m0 + r) * 4 +
                                    c0 / 32 % 4) =
              *reinterpret_cast<const Bytes*>(lds + BM * CRB + r * NBLK);
      return;
    }
  }
  // bf16 output.  The residual rows and the bias into LDS ...
  uint16_t* out = static_cast<uint16_t*>(p.out);
  // 8 columns a thread at a time, which stay, and RS rows a pass
  constexpr int CPRO = BNO / 8, RS = NT / CPRO, ITEMS = BM > RS ? BM / RS : 1;
  static_assert(RS * CPRO == NT && BM % std::min(BM, RS) == 0, "whole passes");
  const int r0 = threadIdx.x / CPRO, cc = threadIdx.x % CPRO * 8;
  if constexpr (!SILU) {
    if (p.residual && N >= 8) {
      // several loads in flight per thread (one at a time took 17 us of a
      // 256 x 256 tile); those outside the output read its last row or piece
      constexpr int BATCH = ITEMS % 16 == 0 ? 16 : ITEMS;
      const int col = min(c0 + cc, N - 8);
      const uint16_t* src = p.residual + col;
      // a piece that ends behind the row: its columns are the last of the 8
      // that end with it
      const int shift = min(c0 + cc - col, 7) * 16;
#pragma unroll
      for (int i = 0; i < ITEMS; i += BATCH) {
        i32x4 v[BATCH];
#pragma unroll
        for (int u = 0; u < BATCH; ++u)
          v[u] = *reinterpret_cast<const i32x4u*>(
              src + (int64_t)(m0 + min(r0 + (i + u) * RS, M - 1 - m0)) * N);
        if (c0 + BNO > N) {
#pragma unroll
          for (int u = 0; u < BATCH; ++u) {
            typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));
            u64x2 w = __builtin_bit_cast(u64x2, v[u]);
            w = shift < 64 ? u64x2{w.x >> shift | (shift ? w.y << (64 - shift) : 0), w.y >> shift}
                           : u64x2{w.y >> (shift - 64), 0};
            v[u] = __builtin_bit_cast(i32x4, w);
          }
        }
#pragma unroll
        for (int u = 0; u < BATCH; ++u)
          if (RS <= BM || r0 < BM)
            *reinterpret_cast<i32x4*>(lds + (r0 + (i + u) * RS) * ORB + cc * 2) = v[u];
      }
    } else if (p.residual) {
      for (int i = threadIdx.x; i < min(BM, M - m0) * N; i += NT)
        *reinterpret_cast<uint16_t*>(lds + i / N * ORB + i % N * 2) =
            p.residual[(int64_t)m0 * N + i];
    }
    if (p.bias)
      for (int i = threadIdx.x; i < BN; i += NT)
        sbias[i] = c0 + i < N ? bf16_bits_to_f32(p.bias[c0 + i]) : 0.f;
    if (p.bias || p.residual) __syncthreads();
  }
  // ... the results beside them, rounded once ...
  if (KG == 1 || kg == 0) {
    constexpr int TB = SILU ? TN / 2 : TN;
    auto stage = [&](auto bias, auto residual) __attribute__((always_inline)) {
#pragma unroll
      for (int b = 0; b < TB; ++b) {
        const int col = (wn * TB + b) * 32 + 4 * g;
        f32x4 add[4];
        if constexpr (decltype(bias)::value)
#pragma unroll
          for (int q = 0; q < 4; ++q) add[q] = *reinterpret_cast<const f32x4*>(sbias + col + 8 * q);
        // the LDS reads of two tiles, then their results (with a wait for each
        // read a 256 x 256 tile took 1 us longer)
        constexpr int AB = TM < 2 ? 1 : 2;
#pragma unroll
        for (int a0 = 0; a0 < TM; a0 += AB) {
          uint64_t prev[AB][4];
          if constexpr (decltype(residual)::value) {
#pragma unroll
            for (int u = 0; u < AB * 4; ++u)
              prev[u / 4][u % 4] = *reinterpret_cast<const uint64_t*>(
                  lds + arow[a0 + u / 4] * ORB + (col + 8 * (u % 4)) * 2);
            __builtin_amdgcn_sched_barrier(0);
          }
#pragma unroll
          for (int u = 0; u < AB * 4; ++u) {
            const int a = a0 + u / 4, q = u % 4;
            f32x4 y = {acc[a][b][4 * q], acc[a][b][4 * q + 1], acc[a][b][4 * q + 2],
                       acc[a][b][4 * q + 3]};
            if constexpr (decltype(bias)::value) y += add[q];
            if constexpr (decltype(residual)::value)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                y[e] += bf16_bits_to_f32((uint16_t)(prev[u / 4][q] >> (16 * e)));
            *reinterpret_cast<uint64_t*>(lds + arow[a] * ORB + (col + 8 * q) * 2) =
                __builtin_bit_cast(uint64_t, __builtin_convertvector(y, bf16x4));
          }
        }
      }
    };
    using yes = std::true_type;
    using no = std::false_type;
    if constexpr (SILU) {
      stage(no{}, no{});
    } else if (!p.residual) {
      p.bias ? stage(yes{}, no{}) : stage(no{}, no{});
    } else {
      p.bias ? stage(yes{}, yes{}) : stage(no{}, yes{});
    }
  }
  __syncthreads();
  // ... and the rows out
  if (c0 + cc >= N || r0 >= BM) return;
  uint16_t* dst = out + (int64_t)(m0 + r0) * N + c0 + cc;
  if (c0 + cc + 8 <= N) {
    rows_out(reinterpret_cast<uint8_t*>(dst), (int64_t)RS * N * 2, lds + r0 * ORB + cc * 2,
             std::integral_constant<int, RS * ORB>{}, std::integral_constant<int, ITEMS>{},
             std::integral_constant<int, RS>{}, r0);
  } else {  // the row's last piece
    for (int r = r0; r < min(BM, M - m0); r += RS, dst += (int64_t)RS * N) {
      uint16_t v[8];
      *reinterpret_cast<i32x4*>(v) = *reinterpret_cast<const i32x4*>(lds + r * ORB + cc * 2);
#pragma unroll
      for (int e = 0; e < 7; ++e)
        if (c0 + cc + e < N) dst[e] = v[e];
    }
  }
}

template <bool SILU, int WM, int WN, int TM, int TN, int KG, int S>
int32_t launch(const MxLinear& p, hipStream_t stream) {
  constexpr int BM = 32 * WM * TM, BN = 32 * WN * TN, NT = 64 * WM * WN * KG;
  constexpr int BNO = SILU ? BN / 2 : BN;
  // an MXFP8 output's padding is written too
  const int64_t cols = p.out_scales ? mx_steps(p.N) * 128 : p.N;
  const int64_t ntm = ((int64_t)p.M + BM - 1) / BM, ntn = (cols + BNO - 1) / BNO;
  PA_REQUIRE(ntm * ntn < (1ll << 30) && grid_fits(ntm * ntn + 7, NT), PA_ERR_UNSUPPORTED,
             "pa_linear_mx: %d x %d outputs", p.M, p.N);
  const dim3 grid(8 * (uint32_t)((ntm * ntn + 7) / 8));
  mx_gemm_kernel<SILU, WM, WN, TM, TN, KG, S><<<grid, NT, 0, stream>>>(p, (int)ntm, (int)ntn);
  return check_launch("pa_linear_mx");
}

// Few rows (decode steps): the weights' bytes bound the call, so they stream
// from memory straight to registers.  Yᵀ tiles on
// v_mfma_scale_f32_16x16x128_f8f6f4: A = a fragment of W (16 rows), B = 16 rows
// of X; lane (c, j) = (lane % 16, lane / 16) holds columns 16 j .. + 15 and
// 64 + 16 j .. + 15 of row c of both and the scale byte of columns 32 j .. + 31,
// and of a product Yᵀ[W row 4 j + r][X row c].  A workgroup computes TG NT W
// tiles x MT X tiles: TG groups of kw wavefronts, which take NT tiles and an
// equal share of the K steps each and sum in LDS, from where every thread
// finishes four columns of one row.  SILU: one group takes two gate tiles, the
// other their up tiles, so that a workgroup holds whole blocks of 32 output
// columns.  (Up to KW wavefronts a group: short rows have fewer steps.)
// A wavefront has the step at hand and the next in flight.  X goes through LDS
// of the wavefront's own, copied in whole 128-byte lines (loaded as the
// operands need it, half a line per row and load, L2 served it at half its
// rate, and 32 rows took 4 us longer than 1 at 896 x 4864).
// Bound by the weights' bytes where they are many (1 x 151936 x 896 22.9 us, 6.1
// TB/s), and by X's, which every workgroup reads (4096 x 12288: 1 row 11.7 us, 4.4
// TB/s, 17 rows 14.1, 32 rows 17.2; three steps in flight 3% less for 1 row, 8%
// more for 17 and 32; 32 x 151936 x 896 30.4, 64 rows 44.8); else by a launch and a
// few steps' latency (32 x 1152 x 896 3.4 us, with the bias 3.7).
template <bool SILU, int MT, int NT, int KW>
__global__ __launch_bounds__(64 * KW * (SILU ? 2 : 1), MT == 4 ? 2 : 4) void mx_skinny_kernel(
    const MxLinear p, int kw, int share, int more) {
  static_assert(!SILU || NT == 2, "two gate and two up tiles");
  constexpr int TG = SILU ? 2 : 1, TILES = TG * NT, NO = NT;  // NO: output tiles
  constexpr int XB = MT * 2048;                               // a step's rows of X
  constexpr int PART = KW * TILES * MT * 1024;
  constexpr int SM = KW * TG * 2 * XB > PART ? KW * TG * 2 * XB : PART;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[SM];
  f32x4* part = reinterpret_cast<f32x4*>(lds);  // [kw][TILES][MT][64], behind the products
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, j = lane >> 4;
  const int M = p.M, N = p.N, nk = p.steps;
  const int tiles_n = (int)((uint32_t)(N + 15) >> 4);  // of W (of its gate half)
  const int tg = TG == 1 || wave < kw ? 0 : 1, kp = wave - tg * kw;
  // `share` steps each, the first `more` one more (a division here costs as
  // much as a step)
  const int s0 = kp * share + min(kp, more), s1 = s0 + share + (kp < more ? 1 : 0);
  const uint8_t *wp[NT], *sp[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    // tiles behind the last read it again
    const int f = min((int)blockIdx.x * NO + t, tiles_n - 1) + (SILU ? tg * tiles_n : 0);
    wp[t] = p.w + (int64_t)f * nk * 2048 + lane * 16;
    sp[t] = p.ws + (int64_t)f * nk * 64 + c * 4;
  }
  // rows behind the last are the last again; 16-byte chunks swizzled by the row
  auto swz = [](int r) -> int { return (r / 2) % 8; };
  uint32_t xo[2 * MT];
#pragma unroll
  for (int u = 0; u < 2 * MT; ++u) {
    const int r = u * 8 + lane / 8;
    xo[u] = (uint32_t)min(r, M - 1) * (uint32_t)(nk * 128) + ((lane % 8) ^ swz(r)) * 16;
  }
  const uint32_t x0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)lds +
                      wave * 2 * XB;
  f32x4 acc[NT][MT];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int q = 0; q < MT; ++q) acc[t][q] = f32x4{0.f, 0.f, 0.f, 0.f};
  struct Stage {
    i32x4 w[NT][2];
    int ws[NT], xs[MT];
  };
  constexpr int FETCHED = 2 * MT + 3 * NT + MT;  // copies and loads of a step
  auto fetch = [&](int s, int buf, Stage& o) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < 2 * MT; ++u)
      lds_copy16(p.x + (int64_t)s * 128, xo[u],
                 __builtin_amdgcn_readfirstlane(x0 + buf * XB + u * 1024));
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const uint8_t* at = wp[t] + (int64_t)s * 2048;
      o.w[t][0] = __builtin_nontemporal_load(reinterpret_cast<const i32x4*>(at));
      o.w[t][1] = __builtin_nontemporal_load(reinterpret_cast<const i32x4*>(at + 1024));
      o.ws[t] = *reinterpret_cast<const int*>(sp[t] + (int64_t)s * 64);
    }
#pragma unroll
    for (int t = 0; t < MT; ++t)
      o.xs[t] = *reinterpret_cast<const int*>(
          p.xs + ((int64_t)s * p.pad_m + min(16 * t + c, M - 1)) * 4);
  };
  // newer: the copies and loads issued after the step's own, all of which have
  // to be in flight still or done
  auto multiply = [&](int buf, const Stage& o, auto newer) __attribute__((always_inline)) {
    wait_vm<decltype(newer)::value>();
    asm volatile("" ::: "memory");
    // The scales are used behind the wait only: the compiler moved their
    // shifts to the loop's head, and waited there for the loads.
    int ws[NT], xs[MT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      ws[t] = o.ws[t];
      asm volatile("" : "+v"(ws[t]));
    }
#pragma unroll
    for (int q = 0; q < MT; ++q) {
      xs[q] = o.xs[q];
      asm volatile("" : "+v"(xs[q]));
    }
#pragma unroll
    for (int q = 0; q < MT; ++q) {
      const uint8_t* row = lds + wave * 2 * XB + buf * XB + (16 * q + c) * 128;
      const i32x4 lo = *reinterpret_cast<const i32x4*>(row + (j ^ swz(16 * q + c)) * 16);
      const i32x4 hi = *reinterpret_cast<const i32x4*>(row + ((4 + j) ^ swz(16 * q + c)) * 16);
#pragma unroll
      for (int t = 0; t < NT; ++t)
        acc[t][q] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
            __builtin_shufflevector(o.w[t][0], o.w[t][1], 0, 1, 2, 3, 4, 5, 6, 7),
            __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7), acc[t][q], 0, 0, 0,
            ws[t] >> (8 * j), 0, xs[q] >> (8 * j));
    }
    wait_copies<63>();  // the reads are done before the buffer is copied into again
    asm volatile("" ::: "memory");
  };
  // No load under a branch that ends before its step is multiplied: the
  // compiler would wait for all loads in front of every product.
  using Next = std::integral_constant<int, FETCHED>;
  using None = std::integral_constant<int, 0>;
  Stage a, b;
  if (s0 < s1) {
    fetch(s0, 0, a);
    int s = s0;
    for (; s + 2 < s1; s += 2) {
      fetch(s + 1, 1, b);
      multiply(0, a, Next{});
      fetch(s + 2, 0, a);
      multiply(1, b, Next{});
    }
    if (s + 1 < s1) {
      fetch(s + 1, 1, b);
      multiply(0, a, Next{});
      multiply(1, b, None{});
    } else {
      multiply(0, a, None{});
    }
  }
  __syncthreads();  // everyone is done with X
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int q = 0; q < MT; ++q)
      part[((kp * TILES + tg * NT + t) * MT + q) * 64 + lane] = acc[t][q];
  __syncthreads();
  // columns 4 i % (4 NO) .. + 3 of row i / (4 NO), partial sums in K order
  const int rows = min(M, 16 * MT);
  auto total = [&](int tile, int row, int quad) __attribute__((always_inline)) {
    f32x4 v = part[(tile * MT + row / 16) * 64 + row % 16 + 16 * quad];
    for (int w = 1; w < kw; ++w)
      v += part[((w * TILES + tile) * MT + row / 16) * 64 + row % 16 + 16 * quad];
    return v;
  };
  for (int i = threadIdx.x; i < 16 * MT * 4 * NO; i += 64 * TG * kw) {
    const int row = i / (4 * NO), quad = i % (4 * NO);
    if (row >= rows) break;  // whole rows: the shuffles below stay within one
    const int col = ((int)blockIdx.x * 4 * NO + quad) * 4;
    f32x4 y = total(quad / 4, row, quad % 4);
    if constexpr (SILU) {
      const f32x4 up = total(NO + quad / 4, row, quad % 4);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        y[e] = col < N ? mx_silu_mul(y[e], up[e]) : 0.f;  // N: a multiple of 32
      if (p.out_scales) {
        // a block is eight consecutive threads' columns
        const float four[4] = {y[0], y[1], y[2], y[3]};
        uint32_t top = mx_top(four);
        top = max(top, dpp<kDppXor1>(top));
        top = max(top, dpp<kDppXor2>(top));
        top = max(top, dpp<kDppHalfMirror>(top));
        const uint32_t byte = mx_scale_byte(top);
        const int pitch = (N + 127) / 128 * 128;
        *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(p.out) + (int64_t)row * pitch + col) =
            mx_codes4(y[0], y[1], y[2], y[3], mx_inverse(byte));
        if (quad % 8 == 0)
          p.out_scales[((int64_t)(col / 128) * p.pad_m + row) * 4 + col / 32 % 4] = (uint8_t)byte;
        continue;
      }
    }
    const int64_t at = (int64_t)row * N + col;
    uint16_t* out = static_cast<uint16_t*>(p.out) + at;
    uint16_t prev[4] = {0, 0, 0, 0}, v[4];
    if (col >= N) continue;
    const bool wide = col + 4 <= N;
    if (!SILU && p.residual) {
      if (wide)
        *reinterpret_cast<uint64_t*>(prev) = *reinterpret_cast<const u64u*>(p.residual + at);
      else
        for (int e = 0; e < 4 && col + e < N; ++e) prev[e] = p.residual[at + e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float f = y[e];
      if (!SILU && p.bias && col + e < N) f += bf16_bits_to_f32(p.bias[col + e]);
      if (!SILU) f += bf16_bits_to_f32(prev[e]);
      v[e] = f32_to_bf16_bits(f);
    }
    if (wide)
      *reinterpret_cast<u64u*>(out) = *reinterpret_cast<const uint64_t*>(v);
    else
      for (int e = 0; e < 4 && col + e < N; ++e) out[e] = v[e];
  }
}

template <bool SILU, int MT, int NT, int KW>
int32_t launch_skinny(const MxLinear& p, hipStream_t stream) {
  const int kw = std::min(KW, p.steps);
  // an MXFP8 output's padding is written too
  const int64_t cols = p.out_scales ? mx_steps(p.N) * 128 : p.N;
  const dim3 grid((uint32_t)((cols + 16 * NT - 1) / (16 * NT)));
  mx_skinny_kernel<SILU, MT, NT, KW><<<grid, 64 * (SILU ? 2 : 1) * kw, 0, stream>>>(
      p, kw, p.steps / kw, p.steps % kw);
  return check_launch("pa_linear_mx");
}

}  // namespace
}  // namespace pa

using namespace pa;

extern "C" int32_t pa_linear_mx(void* out, uint8_t* out_scales, const uint8_t* x,
                                const uint8_t* x_scales, const uint8_t* weight,
                                const uint8_t* weight_scales, const void* bias,
                                const void* residual, int32_t rows, int32_t out_features,
                                int32_t in_features, int32_t act, pa_stream_t stream) {
  clear_error();
  const bool silu = act == PA_ACT_SILU_MUL;
  PA_REQUIRE(act == PA_ACT_NONE || silu, PA_ERR_INVALID_ARG, "pa_linear_mx: unknown activation %d",
             act);
  PA_REQUIRE(rows >= 0 && out_features > 0 && in_features > 0, PA_ERR_INVALID_ARG,
             "pa_linear_mx: bad sizes");
  PA_REQUIRE(!silu || (!bias && !residual), PA_ERR_INVALID_ARG,
             "pa_linear_mx: bias or residual with the SwiGLU epilogue");
  PA_REQUIRE(silu || !out_scales, PA_ERR_INVALID_ARG,
             "pa_linear_mx: an MXFP8 output needs the SwiGLU epilogue");
  PA_REQUIRE(!silu || out_features % 32 == 0, PA_ERR_UNSUPPORTED,
             "pa_linear_mx: SwiGLU over %d columns (a multiple of 32)", out_features);
  // 32-bit lane offsets: 255 rows of codes, and the scales from a gate row to
  // its up row
  PA_REQUIRE(in_features <= kMxMaxCols && mx_pad_rows(out_features) / 16 * mx_steps(in_features) *
                                                  64 < (1ll << 31),
             PA_ERR_UNSUPPORTED, "pa_linear_mx: a weight of %d x %d", out_features, in_features);
  if (rows == 0) return PA_OK;
  PA_REQUIRE(out && x && x_scales && weight && weight_scales, PA_ERR_INVALID_ARG,
             "pa_linear_mx: null pointer");
  PA_REQUIRE(((uintptr_t)out | (uintptr_t)x | (uintptr_t)weight) % 16 == 0, PA_ERR_INVALID_ARG,
             "pa_linear_mx: out, x and weight must be 16-byte aligned");
  PA_REQUIRE(((uintptr_t)x_scales | (uintptr_t)weight_scales | (uintptr_t)out_scales) % 4 == 0,
             PA_ERR_INVALID_ARG, "pa_linear_mx: scales must be 4-byte aligned");
  PA_REQUIRE((uintptr_t)bias % 2 == 0 && (uintptr_t)residual % 16 == 0, PA_ERR_INVALID_ARG,
             "pa_linear_mx: the residual must be 16-byte aligned, the bias to its elements");
  {
    const int64_t wrows = silu ? 2 * (int64_t)out_features : out_features;
    const int64_t kp = mx_steps(in_features) * 128, nb = (int64_t)rows * out_features * 2;
    const int64_t no = out_scales ? rows * mx_steps(out_features) * 128 : nb;
    const int64_t ns = out_scales ? mx_scale_bytes(rows, out_features) : 0;
    auto meets = [&](const void* q, int64_t n) {
      return mx_overlap(q, n, x, rows * kp) ||
             mx_overlap(q, n, x_scales, mx_scale_bytes(rows, in_features)) ||
             mx_overlap(q, n, weight, mx_pad_rows(wrows) * kp) ||
             mx_overlap(q, n, weight_scales, mx_scale_bytes(wrows, in_features)) ||
             mx_overlap(q, n, bias, 2 * (int64_t)out_features);
    };
    PA_REQUIRE(!meets(out, no) && !meets(out_scales, ns) && !mx_overlap(out, no, out_scales, ns) &&
                   (residual == out || !mx_overlap(out, no, residual, nb)),
               PA_ERR_INVALID_ARG, "pa_linear_mx: out overlaps another array");
  }
  const MxLinear p{out,      out_scales,
                   x,        x_scales,
                   weight,   weight_scales,
                   (const uint16_t*)bias, (const uint16_t*)residual,
                   rows,     out_features,
                   (int)mx_steps(in_features), mx_pad_rows(rows)};
  hipStream_t s = (hipStream_t)stream;
  if (const MxSkinny k = choose_mx_skinny(rows, out_features, in_features, silu); k.kw) {
    const int tiles = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;  // of X rows
    if (silu)  // four share K up to 16 rows only
      return k.kw == 4    ? launch_skinny<true, 1, 2, 4>(p, s)
             : tiles == 1 ? launch_skinny<true, 1, 2, 2>(p, s)
                          : launch_skinny<true, 2, 2, 2>(p, s);
    if (k.nt == 2)
      return tiles == 1   ? launch_skinny<false, 1, 2, 4>(p, s)
             : tiles == 2 ? launch_skinny<false, 2, 2, 4>(p, s)
                          : launch_skinny<false, 4, 2, 4>(p, s);
    return tiles == 1   ? launch_skinny<false, 1, 1, 8>(p, s)
           : tiles == 2 ? launch_skinny<false, 2, 1, 8>(p, s)
                        : launch_skinny<false, 4, 1, 8>(p, s);
  }
  if (silu) switch (choose_mx_tiling(rows, 2 * (int64_t)out_features, in_features, true)) {
      case kMx256x256: return launch<true, 2, 2, 4, 4, 1, 2>(p, s);
      case kMx256x128: return launch<true, 4, 2, 2, 2, 1, 3>(p, s);
      case kMx128x128Pair: return launch<true, 2, 2, 2, 2, 1, 2>(p, s);
      case kMx128x128: return launch<true, 4, 2, 1, 2, 1, 3>(p, s);
      case kMx128x64: return launch<true, 4, 1, 1, 2, 1, 4>(p, s);
      default: return launch<true, 2, 1, 1, 2, 2, 4>(p, s);
    }
  switch (choose_mx_tiling(rows, out_features, in_features, false)) {
    case kMx256x256: return launch<false, 2, 2, 4, 4, 1, 2>(p, s);
    case kMx256x128: return launch<false, 4, 2, 2, 2, 1, 3>(p, s);
    case kMx128x128Pair: return launch<false, 2, 2, 2, 2, 1, 2>(p, s);
    case kMx128x128: return launch<false, 4, 2, 1, 2, 1, 3>(p, s);
    case kMx128x64: return launch<false, 4, 1, 1, 2, 1, 4>(p, s);
    case kMx64x64: return launch<false, 2, 2, 1, 1, 2, 4>(p, s);
    default: return launch<false, 2, 1, 1, 1, 2, 4>(p, s);
  }
}
