// fk_fp8_gemm.h — C = A Bᵀ of 8-bit matrices with a scale for each block of
// 128 (include/fkrocm_fp8.h: fk_fp8_gemm).
//
// v_mfma_scale_f32_16x16x128_f8f6f4 and 32x32x64 (D = A B + C, both operands
// e4m3): a lane holds 32 elements of a row, 32 bytes, and a scale for them, a
// power of two, which the operation applies.  All 32 lie in one block of 128,
// whose scale is the same for every lane of the row, so which of k a lane
// holds does not matter as long as it is the same for both operands: pieces of
// 16 elements, 16 lanes the 16 rows of a tile, so that an operand is a 1 KB
// load or LDS read of 16 bytes a lane from where the matrix holds it.  The
// weights are the first operand, so a lane has four consecutive columns of
// one row of C.
//
// The 8-bit operations add eight products of consecutive k of an operand as
// whole numbers of 2^-14 of the largest one's power of two (measured: a product
// below that is lost beside it, one of the next eight is not), so a sum is off
// by up to 7 2^-14 of such a largest product: 1 to 6 10^-5 of C for normal
// rows, with some columns 20 times as large.  CUT: C of 16 bits whose caller asked
// for that, for up to twice the rate.  Otherwise the operands are widened to bf16,
// scales and all, which is exact from 2^-126 on, and go to
// v_mfma_f32_16x16x32_bf16 and 32x32x16, whose sums are binary32's.
#pragma once

#include "fk_fp8.h"
#include "fk_mx4_gemm.h"

typedef __bf16 fk_fp8_bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t fk_fp8_u32x8 __attribute__((ext_vector_type(8)));

namespace fk {

__device__ __forceinline__ fk_fp8_u32x8 fp8_join(u32x4 lo, u32x4 hi) {
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}
__device__ __forceinline__ fk_float4v fp8_mfma(fk_fp8_u32x8 b, uint32_t bs, fk_fp8_u32x8 a, uint32_t as, fk_float4v c) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(__builtin_bit_cast(fk_mx4_int8, b),
                                                          __builtin_bit_cast(fk_mx4_int8, a), c, 0, 0, 0, (int)bs, 0,
                                                          (int)as);
}
__device__ __forceinline__ fk_float16v fp8_mfma32(fk_fp8_u32x8 b, uint32_t bs, fk_fp8_u32x8 a, uint32_t as,
                                                  fk_float16v c) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(__builtin_bit_cast(fk_mx4_int8, b),
                                                         __builtin_bit_cast(fk_mx4_int8, a), c, 0, 0, 0, (int)bs, 0,
                                                         (int)as);
}

// Elements 8 i .. + 7 of a lane's 32, widened, times their scale.
__device__ __forceinline__ fk_fp8_bf16x8 fp8_widen(fk_fp8_u32x8 x, uint32_t i, uint32_t byte) {
  const float scale = e4m3_scale(byte);
  const u32x4 w = {__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[2 * i], scale, false)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[2 * i], scale, true)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[2 * i + 1], scale, false)),
                   __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[2 * i + 1], scale, true))};
  return __builtin_bit_cast(fk_fp8_bf16x8, w);
}

// acc[i][j] += A's block i times B's block j, over the 32 elements a lane holds
// of each, for A's blocks I0 .. I1 - 1.
template <bool CUT, uint32_t I0, uint32_t I1, uint32_t M, uint32_t N, typename Acc>
__device__ __forceinline__ void fp8_multiply(Acc (&acc)[M][N], const fk_fp8_u32x8 (&fb)[N], const uint32_t (&sb)[N],
                                             const fk_fp8_u32x8 (&fa)[M], const uint32_t (&sa)[M]) {
  constexpr bool WIDE = sizeof(Acc) == sizeof(fk_float16v);
  if constexpr (CUT) {
#pragma unroll
    for (uint32_t i = I0; i < I1; i++)
#pragma unroll
      for (uint32_t j = 0; j < N; j++) {
        if constexpr (WIDE) acc[i][j] = fp8_mfma32(fb[j], sb[j], fa[i], sa[i], acc[i][j]);
        else acc[i][j] = fp8_mfma(fb[j], sb[j], fa[i], sa[i], acc[i][j]);
      }
  } else {
#pragma unroll
    for (uint32_t q = 0; q < 4; q++) {
      fk_fp8_bf16x8 b[N];
#pragma unroll
      for (uint32_t j = 0; j < N; j++) b[j] = fp8_widen(fb[j], q, sb[j]);
#pragma unroll
      for (uint32_t i = I0; i < I1; i++) {
        const fk_fp8_bf16x8 x = fp8_widen(fa[i], q, sa[i]);
#pragma unroll
        for (uint32_t j = 0; j < N; j++) {
          if constexpr (WIDE) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(b[j], x, acc[i][j], 0, 0, 0);
          else acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[j], x, acc[i][j], 0, 0, 0);
        }
      }
    }
  }
}

// Few rows: a threadgroup takes MB × NB blocks of 16 × 16, its W wavefronts
// every W-th block of k, the operands straight from memory, two blocks in
// flight; the wavefronts' sums are added in their order in LDS.  Bound by the
// weights' stream where there are many of them (8 rows by 16384, k 8192: 23 µs,
// 5.8 TB/s), else by what each CU takes in (306 KB of 100 rows by 5000, k 3080, in a
// kernel of 9.4 µs): twice the wavefronts, and so loads in flight, gained nothing.  So
// a block is as wide as leaves all CUs one: 100 rows by 5000, k 8192, f32 in blocks of
// 4 x 2 31.6 µs, of 4 x 3, 210 of them, 22.6; 8 rows in 313 of 1 x 1 12.0, in 157 of
// 1 x 2 10.6.
template <uint32_t MB, uint32_t NB, uint32_t W, int T, bool CUT>
__device__ __forceinline__ void fp8_gemm_few(const fk_fp8_gemm_args &a) {
  __shared__ fk_float4v sums[W][MB * NB][FK_WAVE];
  const uint32_t lane = threadIdx.x % FK_WAVE;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / FK_WAVE);
  const uint32_t blocks = fp8_blocks(a.k), quads = fp8_quads(a.k);
  const uint32_t rows_a = fp8_row_tiles(a.m), rows_b = fp8_row_tiles(a.n);
  const uint32_t tiles_m = (rows_a + MB - 1) / MB;
  const uint32_t tm = blockIdx.x % tiles_m * MB, tn = blockIdx.x / tiles_m * NB;
  fk_float4v acc[MB][NB];
#pragma unroll
  for (uint32_t i = 0; i < MB; i++)
#pragma unroll
    for (uint32_t j = 0; j < NB; j++) acc[i][j] = fk_float4v{0.0f, 0.0f, 0.0f, 0.0f};
  // (tiles past the last repeat it; nothing of theirs is stored)
  uint64_t ac[MB], bc[NB], as[MB], bs[NB];
  // A's lanes of rows past the last take it again, whose lines are there (8 rows
  // by 2048, k 8192 7.4 µs without that, 6.5 so; the tallest blocks have no
  // registers for it).
  uint32_t a_lane[MB];
#pragma unroll
  for (uint32_t i = 0; i < MB; i++) {
    const uint64_t t = min(tm + i, rows_a - 1);
    ac[i] = a.a_codes + t * blocks * 2048;
    as[i] = a.a_scales + t * quads * 64;
    a_lane[i] = MB < 8 ? lane / 16 * 16 + min(lane % 16, a.m - 16 * (uint32_t)t - 1) : lane;
  }
#pragma unroll
  for (uint32_t j = 0; j < NB; j++) {
    const uint64_t t = min(tn + j, rows_b - 1);
    bc[j] = a.b_codes + t * blocks * 2048;
    bs[j] = a.b_scales + t * quads * 64;
  }
  struct Block {
    fk_fp8_u32x8 a[MB], b[NB];
    uint32_t as[MB], bs[NB];
  };
  auto load = [&](uint32_t p) {
    Block x;
    const uint64_t codes = (uint64_t)p * 2048, scale = (uint64_t)(p / 4) * 64 + p % 4;
#pragma unroll
    for (uint32_t j = 0; j < NB; j++) {
      const auto from = global_at<const u32x4>(bc[j] + codes);
      x.b[j] = fp8_join(__builtin_nontemporal_load(&from[lane]), __builtin_nontemporal_load(&from[64 + lane]));
      x.bs[j] = global_at<const uint8_t>(bs[j] + scale)[lane % 16 * 4];
    }
#pragma unroll
    for (uint32_t i = 0; i < MB; i++) {
      const auto from = global_at<const u32x4>(ac[i] + codes);
      x.a[i] = fp8_join(from[a_lane[i]], from[64 + a_lane[i]]);
      x.as[i] = global_at<const uint8_t>(as[i] + scale)[lane % 16 * 4];
    }
    return x;
  };
  auto multiply = [&](const Block &x) { fp8_multiply<CUT, 0, MB>(acc, x.b, x.bs, x.a, x.as); };
  // (nothing moves past where loads have gone out)
#define FK_FP8_OUT() __builtin_amdgcn_sched_barrier(0)
  if constexpr (!CUT && MB == 8) {  // (no registers for two blocks and what the widening holds)
    for (uint32_t p = wave; p < blocks; p += W) multiply(load(p));
  } else if (wave + W < blocks) {
    Block x = load(wave), y = load(wave + W);
    FK_FP8_OUT();
    uint32_t p = wave + 2 * W;
    for (; p + W < blocks; p += 2 * W) {
      multiply(x);
      x = load(p);
      FK_FP8_OUT();
      multiply(y);
      y = load(p + W);
      FK_FP8_OUT();
    }
    multiply(x);
    if (p < blocks) {
      x = load(p);
      FK_FP8_OUT();
      multiply(y);
      multiply(x);
    } else {
      multiply(y);
    }
  } else if (wave < blocks) {
    const Block x = load(wave);
    FK_FP8_OUT();
    multiply(x);
  }
#undef FK_FP8_OUT
#pragma unroll
  for (uint32_t i = 0; i < MB; i++)
#pragma unroll
    for (uint32_t j = 0; j < NB; j++) sums[wave][i * NB + j][lane] = acc[i][j];
  __syncthreads();
  for (uint32_t b = wave; b < MB * NB; b += W) {
    fk_float4v v = sums[0][b][lane];
#pragma unroll
    for (uint32_t w = 1; w < W; w++) v += sums[w][b][lane];
    mx4_store_c<T>(a, 16 * (tm + b / NB) + lane % 16, 16 * (tn + b % NB) + 4 * (lane / 16), v);
  }
}

// More rows, in 32 × 32 blocks: lane l holds 32 elements of row l mod 32, and
// D[8 (r div 4) + 4 (l div 32) + r mod 4][l mod 32] as register r.  A
// threadgroup of 4 wavefronts, two by two, takes a tile of 64 GM rows and 64 GN
// columns, each wavefront GM × GN blocks.  A step is one tile of k (64): the
// operands' 1 KB tiles go straight into a ring of LDS stages and are read back
// 16 bytes a lane, no bank twice.  The scales come to registers ahead of their
// blocks, a byte or four blocks' bytes a lane.  Two kernels, by what hides what:
//
// - fp8_gemm_mid: a ring of as many stages as the tile wants.  Three, and three
//   threadgroups a CU, one's loads, reads and stores under another's matrix
//   operations; or, where the tiles do not fill the CUs that often, as many as
//   the LDS holds for one threadgroup, so that a step's loads have the time of
//   seven others to land: 400 rows by 5000, k 8192, 62 µs by three stages, 58 by
//   eight (cut 52 and 36); 200 rows 61, and 41 in tiles of 64 rows (51 and 29).
//   The widening bounds it there, and with cut sums what a CU takes in.
// - fp8_gemm_many: 256 × 256 tiles whose sums take half the register file, one
//   threadgroup a CU, four stages, the next step's operands read and a later
//   step's loaded between a step's matrix operations, and tile after tile with
//   the next one's first loads under the stores.  8192 by 8192 to f16, k 2048: 205
//   to 214 µs (1.3 PFLOP/s; the library's bf16 product 1.37), cut 119 to 124 (2.2 to
//   2.3; from registers alone, random data, 3.0 to 3.4), of which C's stores take
//   8 µs a turn of tiles.
#define FK_FP8_STAGES 4
constexpr uint32_t fp8_many_side = 16;  // row tiles of a tile's side
constexpr uint32_t fp8_many_lds = FK_FP8_STAGES * 2 * fp8_many_side * 1024;
template <uint32_t GM, uint32_t GN, uint32_t STAGES>
constexpr uint32_t fp8_mid_lds() {
  return STAGES * 4 * (GM + GN) * 1024;
}

// An operand's source: up to ROWS row tiles from `tile` on, as buffers of codes
// and of scales.
struct Fp8Source {
  __amdgpu_buffer_rsrc_t codes, scales;
  uint32_t have;
};
__device__ __forceinline__ Fp8Source fp8_source(uint64_t codes, uint64_t scales, uint32_t tile, uint32_t rows,
                                                uint32_t most, uint32_t blocks, uint32_t quads) {
  Fp8Source s;
  s.have = min(rows - tile, most);
  s.codes = buffer((const void *)(codes + (uint64_t)tile * blocks * 2048), (size_t)s.have * blocks * 2048);
  s.scales = buffer((const void *)(scales + (uint64_t)tile * quads * 64), (size_t)s.have * quads * 64);
  return s;
}

template <uint32_t GM, uint32_t GN, uint32_t STAGES, int T, bool CUT>
__device__ __forceinline__ void fp8_gemm_mid(const fk_fp8_gemm_args &a) {
  static_assert(GN >= 2, "the stores' rows of a wavefront are of 128 bytes at least");
  extern __shared__ u32x4 fp8_lds[];
  constexpr uint32_t RA = 4 * GM, RN = 4 * GN;     // row tiles of the slabs
  constexpr uint32_t SLAB = RA * 1024, STAGE = (RA + RN) * 1024;
  const uint32_t lane = threadIdx.x % FK_WAVE;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / FK_WAVE);
  const uint32_t wm = wave & 1, wn = wave >> 1;
  const uint32_t blocks = fp8_blocks(a.k), quads = fp8_quads(a.k);
  const uint32_t rows_a = fp8_row_tiles(a.m), rows_b = fp8_row_tiles(a.n);
  const uint32_t tiles_m = (rows_a + RA - 1) / RA;
  const uint32_t tm = blockIdx.x % tiles_m * RA, tn = blockIdx.x / tiles_m * RN;
  const uint32_t half = lane % 32 / 16, place = lane / 32 * 16 + lane % 16;
  const Fp8Source as = fp8_source(a.a_codes, a.a_scales, tm, rows_a, RA, blocks, quads);
  const Fp8Source bs = fp8_source(a.b_codes, a.b_scales, tn, rows_b, RN, blocks, quads);
  uint32_t a_at[GM], b_at[GN], as_at[GM], bs_at[GN];
#pragma unroll
  for (uint32_t i = 0; i < GM; i++) {
    a_at[i] = min(wave * GM + i, as.have - 1) * blocks * 2048 + lane * 16;
    as_at[i] = min(2 * (wm * GM + i) + half, as.have - 1) * quads * 64 + lane % 16 * 4;
  }
#pragma unroll
  for (uint32_t i = 0; i < GN; i++) {
    b_at[i] = min(wave * GN + i, bs.have - 1) * blocks * 2048 + lane * 16;
    bs_at[i] = min(2 * (wn * GN + i) + half, bs.have - 1) * quads * 64 + lane % 16 * 4;
  }
  FK_MX4_LDS char *const a_to = (FK_MX4_LDS char *)fp8_lds + wave * GM * 1024;
  FK_MX4_LDS char *const b_to = (FK_MX4_LDS char *)fp8_lds + SLAB + wave * GN * 1024;
  const uint32_t ra = (2 * wm * GM + half) * 64 + place, rb = SLAB / 16 + (2 * wn * GN + half) * 64 + place;
  fk_float16v acc[GM][GN];
#pragma unroll
  for (uint32_t i = 0; i < GM; i++)
#pragma unroll
    for (uint32_t j = 0; j < GN; j++)
#pragma unroll
      for (int r = 0; r < 16; r++) acc[i][j][r] = 0.0f;
  const uint32_t last = 2 * blocks - 1;
  auto codes = [&](uint32_t step, uint32_t stage) __attribute__((always_inline)) {
    const uint32_t so = min(step, last) * 1024;
#pragma unroll
    for (uint32_t q = 0; q < GM; q++)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(as.codes, a_to + stage * STAGE + q * 1024, 16, a_at[q], so, 0, 0);
#pragma unroll
    for (uint32_t q = 0; q < GN; q++)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(bs.codes, b_to + stage * STAGE + q * 1024, 16, b_at[q], so, 0, 0);
  };
  // Four blocks' scales, a byte each.
  auto scales = [&](uint32_t (&s)[GM], uint32_t (&t)[GN], uint32_t quad) __attribute__((always_inline)) {
#pragma unroll
    for (uint32_t i = 0; i < GM; i++) s[i] = __builtin_amdgcn_raw_buffer_load_b32(as.scales, as_at[i], quad * 64, 0);
#pragma unroll
    for (uint32_t i = 0; i < GN; i++) t[i] = __builtin_amdgcn_raw_buffer_load_b32(bs.scales, bs_at[i], quad * 64, 0);
  };
  uint32_t sa[GM], sb[GN], next_a[GM], next_b[GN];
  scales(sa, sb, 0);
#pragma unroll
  for (uint32_t t = 0; t + 1 < STAGES; t++) codes(t, t);
  uint32_t at = 0, to = STAGES - 1;   // the stage a step reads, and the one it loads
  // A step loads the stage that the step before it read, so a wavefront comes
  // to its barrier with its reads done (their products may follow).  Its own
  // stage has landed once no more than the loads behind it are in flight (the
  // scales' among them make that early, never late).
  auto step = [&](uint32_t s, uint32_t byte) __attribute__((always_inline)) {
    FK_MX4_VMCNT((STAGES - 2) * (GM + GN));
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    FK_MX4_BARRIER();
    __builtin_amdgcn_sched_barrier(0);
    codes(s + STAGES - 1, to);
    const u32x4 *from = fp8_lds + at * (STAGE / 16);
    fk_fp8_u32x8 fa[GM], fb[GN];
    uint32_t xa[GM], xb[GN];
#pragma unroll
    for (uint32_t j = 0; j < GN; j++) {
      fb[j] = fp8_join(from[rb + 128 * j], from[rb + 128 * j + 32]);
      xb[j] = sb[j] >> (8 * byte) & 255u;
    }
#pragma unroll
    for (uint32_t i = 0; i < GM; i++) {
      fa[i] = fp8_join(from[ra + 128 * i], from[ra + 128 * i + 32]);
      xa[i] = sa[i] >> (8 * byte) & 255u;
    }
    fp8_multiply<CUT, 0, GM>(acc, fb, xb, fa, xa);
    at = at == STAGES - 1 ? 0 : at + 1;
    to = to == STAGES - 1 ? 0 : to + 1;
  };
  auto turn = [&] __attribute__((always_inline)) {
#pragma unroll
    for (uint32_t i = 0; i < GM; i++) sa[i] = next_a[i];
#pragma unroll
    for (uint32_t j = 0; j < GN; j++) sb[j] = next_b[j];
  };
  // Whole fours of blocks, their scales loaded a four ahead: waited for nearer,
  // the counter would hold the codes' loads behind them too.
  uint32_t p = 0;
  for (; p + 4 <= blocks; p += 4) {
    scales(next_a, next_b, min(p / 4 + 1, quads - 1));
#pragma unroll
    for (uint32_t b = 0; b < 4; b++) {
      step(2 * (p + b), b);
      step(2 * (p + b) + 1, b);
    }
    turn();
  }
#pragma unroll
  for (uint32_t b = 0; b < 3; b++)
    if (p + b < blocks) {
      step(2 * (p + b), b);
      step(2 * (p + b) + 1, b);
    }
  __builtin_amdgcn_s_waitcnt(0);
  FK_MX4_BARRIER();
  mx4_store_many<GM, GN, false, T>(a, 16 * tm + 32 * wm * GM, 16 * tn + 32 * wn * GN, acc,
                                   reinterpret_cast<char *>(fp8_lds) + wave * GN * 2048);
}

template <int T, bool CUT>
__device__ __forceinline__ void fp8_gemm_many(const fk_fp8_gemm_args &a) {
  extern __shared__ u32x4 fp8_lds[];
  constexpr uint32_t GB = fp8_many_side / 4;       // a wavefront's blocks of 32, each way
  constexpr uint32_t ROWS = fp8_many_side;         // row tiles of an operand's slab
  constexpr uint32_t SLAB = ROWS * 1024;           // its bytes a step
  constexpr uint32_t STAGE = 2 * SLAB;             // A's, then B's
  constexpr uint32_t Q = ROWS / 4;                 // loads of an operand a wavefront makes a step
  constexpr uint32_t H = GB / 2;                   // A's blocks of half a step
  const uint32_t lane = threadIdx.x % FK_WAVE;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / FK_WAVE);
  const uint32_t wm = wave & 1, wn = wave >> 1;
  const uint32_t blocks = fp8_blocks(a.k), quads = fp8_quads(a.k);
  const uint32_t rows_a = fp8_row_tiles(a.m), rows_b = fp8_row_tiles(a.n);
  const uint32_t tiles_m = (rows_a + ROWS - 1) / ROWS, tiles = tiles_m * ((rows_b + ROWS - 1) / ROWS);

  // A tile's sources.  A wavefront's loads: row tiles Q wave + q of each slab
  // (past the last: the last again, whose blocks are not stored), a lane's 16
  // bytes in their place; the scales of its blocks: of row l mod 32.
  const uint32_t half = lane % 32 / 16, place = lane / 32 * 16 + lane % 16;
  uint32_t tm, tn;
  Fp8Source as, bs;
  uint32_t a_at[Q], b_at[Q], as_at[GB], bs_at[GB];
  auto sources = [&](uint32_t tile) {
    tm = tile % tiles_m * ROWS;
    tn = tile / tiles_m * ROWS;
    as = fp8_source(a.a_codes, a.a_scales, tm, rows_a, ROWS, blocks, quads);
    bs = fp8_source(a.b_codes, a.b_scales, tn, rows_b, ROWS, blocks, quads);
#pragma unroll
    for (uint32_t q = 0; q < Q; q++) {
      a_at[q] = min(wave * Q + q, as.have - 1) * blocks * 2048 + lane * 16;
      b_at[q] = min(wave * Q + q, bs.have - 1) * blocks * 2048 + lane * 16;
    }
#pragma unroll
    for (uint32_t i = 0; i < GB; i++) {
      as_at[i] = min(2 * (wm * GB + i) + half, as.have - 1) * quads * 64 + lane % 16 * 4;
      bs_at[i] = min(2 * (wn * GB + i) + half, bs.have - 1) * quads * 64 + lane % 16 * 4;
    }
  };
  FK_MX4_LDS char *const stage0 = (FK_MX4_LDS char *)fp8_lds + wave * Q * 1024;
  const uint32_t ra = (2 * wm * GB + half) * 64 + place, rb = SLAB / 16 + (2 * wn * GB + half) * 64 + place;

  fk_float16v acc[GB][GB];
  fk_fp8_u32x8 fa0[GB], fb0[GB], fa1[GB], fb1[GB];
  uint32_t sa0[GB], sb0[GB], sa1[GB], sb1[GB];
#define FK_FP8_PIN(X) asm volatile("" : "+v"(X))
#define FK_FP8_PIN_ACC()                                                    \
  _Pragma("unroll") for (uint32_t i_ = 0; i_ < GB; i_++)                    \
  _Pragma("unroll") for (uint32_t j_ = 0; j_ < GB; j_++) asm volatile("" : "+a"(acc[i_][j_]))
#define FK_FP8_SCALES(SA, SB, P)                                                                              \
  _Pragma("unroll") for (uint32_t i_ = 0; i_ < GB; i_++) {                                                    \
    const uint32_t so_ = __builtin_amdgcn_readfirstlane((P) / 4 * 64 + (P) % 4);                              \
    SA[i_] = __builtin_amdgcn_raw_buffer_load_b8(as.scales, as_at[i_], so_, 0);                               \
    SB[i_] = __builtin_amdgcn_raw_buffer_load_b8(bs.scales, bs_at[i_], so_, 0);                               \
  }
  // One step in two halves, A's blocks 0 .. H - 1 then the rest against all
  // of B's.  The first half issues the loads of A's part of step LOAD (and, in a
  // block's first step, those of the next block's scales before them), and reads
  // the next step's B blocks and A blocks 0 .. H - 1; the second B's loads and
  // the next step's other A blocks.  WAIT: the loads that may still be in
  // flight when the step begins.
#define FK_FP8_STEP(FIRST, FA, FB, NA, NB, WAIT, NEXT, LOAD, ST_LOAD, ST_READ)                                \
  do {                                                                                                        \
    if (under && p == 0) FK_MX4_VMCNT(FK_FP8_UNDER(WAIT));                                                    \
    else FK_MX4_VMCNT(WAIT);                                                                                  \
    FK_MX4_BARRIER();                                                                                         \
    __builtin_amdgcn_sched_barrier(0);                                                                        \
    const uint32_t so_ = (LOAD) * 1024;                                                                       \
    FK_MX4_LDS char *d_ = stage0 + (ST_LOAD) * STAGE;                                                         \
    const u32x4 *s_ = fp8_lds + (ST_READ) * (STAGE / 16);                                                     \
    if (FIRST) FK_FP8_SCALES(sa1, sb1, NEXT)                                                                  \
    _Pragma("unroll") for (uint32_t q = 0; q < Q; q++)                                                        \
        __builtin_amdgcn_raw_ptr_buffer_load_lds(as.codes, d_ + q * 1024, 16, a_at[q], so_, 0, 0);            \
    _Pragma("unroll") for (uint32_t j = 0; j < GB; j++) NB[j] = fp8_join(s_[rb + 128 * j], s_[rb + 128 * j + 32]); \
    _Pragma("unroll") for (uint32_t i = 0; i < H; i++) NA[i] = fp8_join(s_[ra + 128 * i], s_[ra + 128 * i + 32]); \
    fp8_multiply<CUT, 0, H>(acc, FB, sb0, FA, sa0);                                                             \
    _Pragma("unroll") for (uint32_t g_ = 0; g_ < H * GB; g_++) {                                              \
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                                                      \
      __builtin_amdgcn_sched_group_barrier(0x020, 2, 0);                                                      \
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);                                                      \
    }                                                                                                         \
    __builtin_amdgcn_sched_barrier(0);                                                                        \
    _Pragma("unroll") for (uint32_t i = H; i < GB; i++) FK_FP8_PIN(FA[i]);                                    \
    _Pragma("unroll") for (uint32_t q = 0; q < Q; q++)                                                        \
        __builtin_amdgcn_raw_ptr_buffer_load_lds(bs.codes, d_ + SLAB + q * 1024, 16, b_at[q], so_, 0, 0);     \
    _Pragma("unroll") for (uint32_t i = H; i < GB; i++) NA[i] = fp8_join(s_[ra + 128 * i], s_[ra + 128 * i + 32]); \
    fp8_multiply<CUT, H, GB>(acc, FB, sb0, FA, sa0);                                                            \
    _Pragma("unroll") for (uint32_t g_ = 0; g_ < H * GB; g_++) {                                              \
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                                                      \
      __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);                                                      \
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);                                                      \
    }                                                                                                         \
    __builtin_amdgcn_sched_barrier(0);                                                                        \
    _Pragma("unroll") for (uint32_t j = 0; j < GB; j++) FK_FP8_PIN(NB[j]);                                    \
    _Pragma("unroll") for (uint32_t i = 0; i < H; i++) FK_FP8_PIN(NA[i]);                                     \
    FK_FP8_PIN_ACC();                                                                                         \
  } while (0)

  // At step s (after its barrier) step s's blocks are in registers but for
  // A's second half, on its way from stage s mod 4, and steps s + 1 and s + 2
  // are in their stages or on their way there.  Loads past the last step
  // repeat it into stages that no step reads, so every wait counts the same
  // loads.
  const uint32_t steps = 2 * blocks, last = steps - 1;
#define FK_FP8_T(X) ((X) < last ? (X) : last)
  // The first three steps of a tile, and its first scales, on their way.
#define FK_FP8_FIRST()                                                                                        \
  do {                                                                                                        \
    FK_FP8_SCALES(sa0, sb0, 0)                                                                                \
    _Pragma("unroll") for (uint32_t t_ = 0; t_ + 1 < FK_FP8_STAGES; t_++) {                                   \
      const uint32_t so_ = FK_FP8_T(t_) * 1024;                                                               \
      FK_MX4_LDS char *d_ = stage0 + t_ * STAGE;                                                              \
      _Pragma("unroll") for (uint32_t q = 0; q < Q; q++) {                                                    \
        __builtin_amdgcn_raw_ptr_buffer_load_lds(as.codes, d_ + q * 1024, 16, a_at[q], so_, 0, 0);            \
        __builtin_amdgcn_raw_ptr_buffer_load_lds(bs.codes, d_ + SLAB + q * 1024, 16, b_at[q], so_, 0, 0);     \
      }                                                                                                       \
    }                                                                                                         \
  } while (0)
  // Tile after tile, the next one's first loads under this one's stores (which
  // go by way of the fourth stage; step 0 loads it).  The counter that a wait
  // looks at has loads and stores in their order, so the waits of a tile's
  // first block leave out the stores that went out behind its first loads,
  // whose number is known where the tile before was whole.
  constexpr uint32_t STORES = 32 * GB * 32 * GB * mx4_bytes_of(T) / (16 * FK_WAVE);  // of a whole tile, a wavefront's
#define FK_FP8_UNDER(N) ((N) + STORES < 63 ? (N) + STORES : 63)
  bool under = false;
  sources(blockIdx.x);
  FK_FP8_FIRST();
  for (uint32_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
#pragma unroll
    for (uint32_t i = 0; i < GB; i++)
#pragma unroll
      for (uint32_t j = 0; j < GB; j++)
#pragma unroll
        for (int r = 0; r < 16; r++) acc[i][j][r] = 0.0f;
    // step 0 landed
    if (under) FK_MX4_VMCNT(FK_FP8_UNDER(2 * Q * (FK_FP8_STAGES - 2)));
    else FK_MX4_VMCNT(2 * Q * (FK_FP8_STAGES - 2));
    FK_MX4_BARRIER();
#pragma unroll
    for (uint32_t i = 0; i < GB; i++) {
      fb0[i] = fp8_join(fp8_lds[rb + 128 * i], fp8_lds[rb + 128 * i + 32]);
      fa0[i] = fp8_join(fp8_lds[ra + 128 * i], fp8_lds[ra + 128 * i + 32]);
    }
#pragma unroll
    for (uint32_t i = 0; i < GB; i++) {
      FK_FP8_PIN(fb0[i]);
      if (i < H) FK_FP8_PIN(fa0[i]);
    }
    for (uint32_t p = 0; p < blocks; p++) {
      const uint32_t s = 2 * p, next = p + 1 < blocks ? p + 1 : p;
      FK_FP8_STEP(true, fa0, fb0, fa1, fb1, 2 * Q, next, FK_FP8_T(s + 3), (s + 3) % 4, (s + 1) % 4);
      FK_FP8_STEP(false, fa1, fb1, fa0, fb0, 2 * Q + 2 * GB, next, FK_FP8_T(s + 4), s % 4, (s + 2) % 4);
#pragma unroll
      for (uint32_t i = 0; i < GB; i++) sa0[i] = sa1[i], sb0[i] = sb1[i];
    }
    // Nothing lands in LDS any more, and no wavefront reads it.
    __builtin_amdgcn_s_waitcnt(0);
    FK_MX4_BARRIER();
    const uint32_t m = 16 * tm + 32 * wm * GB, n = 16 * tn + 32 * wn * GB;
    under = 16 * tm + 64 * GB <= a.m && 16 * tn + 64 * GB <= a.n;
    if (tile + gridDim.x < tiles) {
      sources(tile + gridDim.x);
      FK_FP8_FIRST();
    }
    mx4_store_many<GB, GB, true, T>(a, m, n, acc,
                                    reinterpret_cast<char *>(fp8_lds) + 3 * STAGE + wave * (STAGE / 4));
  }
#undef FK_FP8_PIN
#undef FK_FP8_PIN_ACC
#undef FK_FP8_SCALES
#undef FK_FP8_STEP
#undef FK_FP8_FIRST
#undef FK_FP8_UNDER
#undef FK_FP8_T
}

}  // namespace fk
