// fk_mx4_gemm.h — C = A Bᵀ of 4-bit microscaled matrices (include/
// fkrocm_mx4.h: fk_mx4_gemm).
//
// v_mfma_scale_f32_16x16x128_f8f6f4 (D = A B + C, both operands e2m1): lane l
// holds 32 elements of row l mod 16, k 32 (l div 16) .. + 31 — one block of
// the format, 16 bytes, and its scale a byte of another register — and D[4 (l
// div 16) + r][l mod 16] as register r.  The matrices are held in that order,
// so an operand is one 1 KB load of 16 bytes a lane.  The weights are the
// first operand, so a lane has four consecutive columns of one row of C.
#pragma once

#include "fk_mfma.h"
#include "fk_mx4.h"

typedef int fk_mx4_int8 __attribute__((ext_vector_type(8)));

namespace fk {

// The operand registers: the operation reads the first four of the eight.
__device__ __forceinline__ fk_mx4_int8 mx4_operand(u32x4 w) {
  return fk_mx4_int8{(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
}
// TILE: which of a pair of tiles, so which byte of the scales.
template <int TILE>
__device__ __forceinline__ fk_float4v mx4_mfma(u32x4 b, uint32_t bs, u32x4 a, uint32_t as, fk_float4v c) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx4_operand(b), mx4_operand(a), c, 4, 4, TILE, (int)bs, TILE,
                                                          (int)as);
}

// Four consecutive columns n .. n + 3 of row m of C (of a call's arguments).
template <int T, typename Args>
__device__ __forceinline__ void mx4_store_c(const Args &a, uint32_t m, uint32_t n, fk_float4v v) {
  if (m >= a.m || n >= a.n) return;
  const uint64_t at = a.c + ((uint64_t)m * a.c_stride + n) * mx4_bytes_of(T);
  if (n + 4 <= a.n) {
    if constexpr (T == FK_T_F32) {
      *global_at<mx4_float4>(at) = v;
    } else if constexpr (T == FK_T_F16) {
      typedef _Float16 half4 __attribute__((ext_vector_type(4), aligned(2)));
      *global_at<half4>(at) = half4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
    } else {
      typedef __bf16 bf4 __attribute__((ext_vector_type(4), aligned(2)));
      *global_at<bf4>(at) = bf4{(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
    }
  } else {
#pragma unroll
    for (uint32_t r = 0; r < 3; r++)
      if (n + r < a.n) mx4_store<T>(at, r, v[r]);
  }
}

// Few rows: a threadgroup takes MB × NB blocks of 16 × 16, its W wavefronts
// every W-th pair of tiles along k, the operands straight from memory; the
// wavefronts' sums are added in their order in LDS.  Round trips to memory
// bound it, so a wavefront has two pairs in flight: the compiler alone puts a
// pair's loads right before their products (100 rows by 5000, k 3080 8.3 µs in
// blocks of 8 x 2, so 6.8; 8 by 8192, k 8192 7.2 in 1 x 1, 6.8).
template <uint32_t MB, uint32_t NB, uint32_t W, int T>
__device__ __forceinline__ void mx4_gemm_few(const fk_mx4_gemm_args &a) {
  __shared__ fk_float4v sums[W][MB * NB][FK_WAVE];
  const uint32_t lane = threadIdx.x % FK_WAVE;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / FK_WAVE);
  const uint32_t pairs = mx4_pairs(a.k);
  const uint32_t rows_a = mx4_row_tiles(a.m), rows_b = mx4_row_tiles(a.n);
  const uint32_t tiles_m = (rows_a + MB - 1) / MB;
  const uint32_t tm = blockIdx.x % tiles_m * MB, tn = blockIdx.x / tiles_m * NB;
  fk_float4v acc[MB][NB];
#pragma unroll
  for (uint32_t i = 0; i < MB; i++)
#pragma unroll
    for (uint32_t j = 0; j < NB; j++) acc[i][j] = fk_float4v{0.0f, 0.0f, 0.0f, 0.0f};
  // (blocks past the last repeat it; nothing of theirs is stored)
  uint64_t ac[MB], bc[NB];
#pragma unroll
  for (uint32_t i = 0; i < MB; i++) ac[i] = (uint64_t)min(tm + i, rows_a - 1) * pairs;
#pragma unroll
  for (uint32_t j = 0; j < NB; j++) bc[j] = (uint64_t)min(tn + j, rows_b - 1) * pairs;
  struct Pair {
    u32x4 a[MB][2], b[NB][2];
    uint32_t as[MB], bs[NB];
  };
  auto load = [&](uint32_t p) {
    Pair x;
#pragma unroll
    for (uint32_t j = 0; j < NB; j++) {
      const auto codes = global_at<const u32x4>(a.b_codes + (bc[j] + p) * 2048);
      x.b[j][0] = __builtin_nontemporal_load(&codes[lane]);
      x.b[j][1] = __builtin_nontemporal_load(&codes[64 + lane]);
      x.bs[j] = global_at<const uint16_t>(a.b_scales + (bc[j] + p) * 128)[lane];
    }
#pragma unroll
    for (uint32_t i = 0; i < MB; i++) {
      const auto codes = global_at<const u32x4>(a.a_codes + (ac[i] + p) * 2048);
      x.a[i][0] = codes[lane];
      x.a[i][1] = codes[64 + lane];
      x.as[i] = global_at<const uint16_t>(a.a_scales + (ac[i] + p) * 128)[lane];
    }
    return x;
  };
  auto multiply = [&](const Pair &x) {
#pragma unroll
    for (uint32_t i = 0; i < MB; i++)
#pragma unroll
      for (uint32_t j = 0; j < NB; j++) acc[i][j] = mx4_mfma<0>(x.b[j][0], x.bs[j], x.a[i][0], x.as[i], acc[i][j]);
#pragma unroll
    for (uint32_t i = 0; i < MB; i++)
#pragma unroll
      for (uint32_t j = 0; j < NB; j++) acc[i][j] = mx4_mfma<1>(x.b[j][1], x.bs[j], x.a[i][1], x.as[i], acc[i][j]);
  };
  // (nothing moves past where loads have gone out)
#define FK_MX4_OUT() __builtin_amdgcn_sched_barrier(0)
  if (wave + W < pairs) {
    Pair x = load(wave), y = load(wave + W);
    FK_MX4_OUT();
    uint32_t p = wave + 2 * W;
    for (; p + W < pairs; p += 2 * W) {
      multiply(x);
      x = load(p);
      FK_MX4_OUT();
      multiply(y);
      y = load(p + W);
      FK_MX4_OUT();
    }
    multiply(x);
    if (p < pairs) {
      x = load(p);
      FK_MX4_OUT();
      multiply(y);
      multiply(x);
    } else {
      multiply(y);
    }
  } else if (wave < pairs) {
    const Pair x = load(wave);
    FK_MX4_OUT();
    multiply(x);
  }
#undef FK_MX4_OUT
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

// More rows: v_mfma_scale_f32_32x32x64_f8f6f4, 1.2 times the rate of the 16 ×
// 16 form here on random operands (6.5 and 5.4 PFLOP/s in registers alone,
// where the chip's power holds its clock down; 9.6 and 5.9 on zeros): lane l
// holds a block of row l mod 32, k 32 (l div 32) .. + 31, and D[8 (r div 4) + 4
// (l div 32) + r mod 4][l mod 32] as register r.
//
// A threadgroup of 4 wavefronts, two by two, takes a tile of 64 GM rows and 64
// GN columns, each wavefront GM × GN blocks of 32 × 32.  A step is one tile of
// k (128): the operands' 1 KB blocks go straight into a ring of LDS stages and
// are read back 16 bytes a lane, 16 lanes 256 consecutive bytes, no bank
// twice.  The scales come to registers, two steps' in one load of two bytes a
// lane, a pair of steps ahead.  Two kernels, by what hides what:
//
// - mx4_gemm_mid: three stages, the operands read as they are needed, and
//   three threadgroups a CU, one's loads, reads and stores under another's
//   matrix operations.  For what few 256 x 256 tiles would leave to few CUs.
//   (Before every other step the compiler's waits for the scales drain the loads
//   that the written wait would leave in flight, so the third stage hides less
//   than it could.)
// - mx4_gemm_many: 256 × 256 tiles whose sums take half the register file, so
//   one threadgroup a CU: four stages, the next step's operands read and a
//   later step's loaded between a step's matrix operations, and tile after
//   tile with the next one's first loads under the stores.  Half the traffic
//   for each product: 8192 x 8192 to f16, the same operands each time, k 8192
//   235 to 246 µs (4.5 to 4.7 PFLOP/s; mid 300), k 2048 86 (3.2; mid 91), from
//   memory each time 258 and 85.  With no loads, reads or scales at all its
//   matrix operations take 200 µs of the 235: the clock that the chip's power
//   leaves them (1.9 GHz of 2.4) bounds it.
#define FK_MX4_STAGES 4
#define FK_MX4_LDS __attribute__((address_space(3)))
constexpr uint32_t mx4_many_side = 16;  // row tiles of a tile's side
constexpr uint32_t mx4_many_lds = FK_MX4_STAGES * 2 * mx4_many_side * 1024;
template <uint32_t GM, uint32_t GN>
constexpr uint32_t mx4_mid_lds() {
  return 3 * 4 * (GM + GN) * 1024;
}
// s_waitcnt vmcnt(n), the other counters untouched.
#define FK_MX4_VMCNT(N) __builtin_amdgcn_s_waitcnt(((N) & 15) | (((N) >> 4) << 14) | (0x7 << 4) | (0xf << 8))
// The barrier without __syncthreads' wait for every load in flight.
#define FK_MX4_BARRIER()                  \
  do {                                    \
    asm volatile("" ::: "memory");        \
    __builtin_amdgcn_s_barrier();         \
    asm volatile("" ::: "memory");        \
  } while (0)

template <int TILE>
__device__ __forceinline__ fk_float16v mx4_mfma32(u32x4 b, uint32_t bs, u32x4 a, uint32_t as, fk_float16v c) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx4_operand(b), mx4_operand(a), c, 4, 4, TILE, (int)bs, TILE,
                                                         (int)as);
}

// A wavefront's 32 GM rows of 32 GN columns into C, through its own share of
// an LDS stage: of 32 rows at a time RB bytes each are written as the
// operation left them, a lane 4 columns of a row, and read back a row's
// consecutive 16 bytes a lane, so that stores are RB whole bytes of a row (of the
// many, past the caches: 8192 x 8192, operands from memory, k 2048 97 µs, so 85;
// k 8192 264 and 258).
template <uint32_t GM, uint32_t GN, bool AGPR, int T, typename Args>
__device__ __forceinline__ void mx4_store_many(const Args &a, uint32_t m0, uint32_t n0, fk_float16v (&acc)[GM][GN],
                                               char *stage) {
  constexpr uint32_t RB = GN * 64, BYTES = mx4_bytes_of(T), COLS = RB / BYTES, UNITS = RB / 16, EACH = 16 / BYTES;
  const uint32_t lane = threadIdx.x % FK_WAVE;
  // 16-byte unit u of row m at place u ^ turn(m): no bank twice in 16 lanes
  auto place = [](uint32_t m, uint32_t u) { return m * RB + (u ^ (UNITS == 16 ? m & 15u : (m >> 1) & 7u)) * 16; };
#pragma unroll
  for (uint32_t i = 0; i < GM; i++)
#pragma unroll
    for (uint32_t c = 0; c < 32 * GN / COLS; c++) {
      const uint32_t row = lane % 32;
      // (taken here: rounded further ahead, they would not fit the registers)
#pragma unroll
      for (uint32_t j = 0; j < COLS / 32; j++) {
        if constexpr (AGPR) asm volatile("" : "+a"(acc[i][c * (COLS / 32) + j]));
        else asm volatile("" : "+v"(acc[i][c * (COLS / 32) + j]));
      }
#pragma unroll
      for (uint32_t j = 0; j < COLS / 32; j++)
#pragma unroll
        for (uint32_t q = 0; q < 4; q++) {
          const fk_float16v &v = acc[i][c * (COLS / 32) + j];
          const uint32_t col = 32 * j + 8 * q + 4 * (lane / 32);
          char *const to = stage + place(row, col / EACH) + col % EACH * BYTES;
          if constexpr (T == FK_T_F32) {
            *reinterpret_cast<fk_float4v *>(to) = fk_float4v{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
          } else if constexpr (T == FK_T_F16) {
            typedef _Float16 half4 __attribute__((ext_vector_type(4)));
            *reinterpret_cast<half4 *>(to) =
                half4{(_Float16)v[4 * q], (_Float16)v[4 * q + 1], (_Float16)v[4 * q + 2], (_Float16)v[4 * q + 3]};
          } else {
            typedef __bf16 bf4 __attribute__((ext_vector_type(4)));
            *reinterpret_cast<bf4 *>(to) =
                bf4{(__bf16)v[4 * q], (__bf16)v[4 * q + 1], (__bf16)v[4 * q + 2], (__bf16)v[4 * q + 3]};
          }
        }
      asm volatile("" ::: "memory");
#pragma unroll
      for (uint32_t t = 0; t < 32 * UNITS / FK_WAVE; t++) {
        const uint32_t r = t * (FK_WAVE / UNITS) + lane / UNITS, u = lane % UNITS;
        const u32x4 w = *reinterpret_cast<const u32x4 *>(stage + place(r, u));
        const uint32_t m = m0 + 32 * i + r, n = n0 + c * COLS + u * EACH;
        const uint64_t at = a.c + ((uint64_t)m * a.c_stride + n) * BYTES;
        if (m < a.m && n < a.n) {
          if (n + EACH <= a.n) {
            if constexpr (AGPR) __builtin_nontemporal_store(w, global_at<mx4_u32x4>(at));
            else *global_at<mx4_u32x4>(at) = w;
          } else {
#pragma unroll
            for (uint32_t e = 0; e < EACH - 1; e++)
              if (n + e < a.n) {
                if constexpr (BYTES == 4) global_at<uint32_t>(at)[e] = w[e];
                else global_at<uint16_t>(at)[e] = (uint16_t)(w[e / 2] >> (16 * (e % 2)));
              }
          }
        }
      }
      asm volatile("" ::: "memory");  // read before the next rows are written
    }
}

template <uint32_t GM, uint32_t GN, int T>
__device__ __forceinline__ void mx4_gemm_mid(const fk_mx4_gemm_args &a) {
  extern __shared__ u32x4 mx4_lds[];
  constexpr uint32_t RA = 4 * GM, RN = 4 * GN;     // row tiles of the slabs
  constexpr uint32_t SLAB = RA * 1024, STAGE = (RA + RN) * 1024;
  const uint32_t lane = threadIdx.x % FK_WAVE;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / FK_WAVE);
  const uint32_t wm = wave & 1, wn = wave >> 1;
  const uint32_t pairs = mx4_pairs(a.k), rows_a = mx4_row_tiles(a.m), rows_b = mx4_row_tiles(a.n);
  const uint32_t tiles_m = (rows_a + RA - 1) / RA;
  const uint32_t tm = blockIdx.x % tiles_m * RA, tn = blockIdx.x / tiles_m * RN;
  const uint32_t half = lane % 32 / 16, place = lane / 32 * 16 + lane % 16;
  const uint32_t have_a = min(rows_a - tm, RA), have_b = min(rows_b - tn, RN);
  const auto a_src = buffer((const void *)(a.a_codes + (uint64_t)tm * pairs * 2048), (size_t)have_a * pairs * 2048);
  const auto b_src = buffer((const void *)(a.b_codes + (uint64_t)tn * pairs * 2048), (size_t)have_b * pairs * 2048);
  const auto as_src = buffer((const void *)(a.a_scales + (uint64_t)tm * pairs * 128), (size_t)have_a * pairs * 128);
  const auto bs_src = buffer((const void *)(a.b_scales + (uint64_t)tn * pairs * 128), (size_t)have_b * pairs * 128);
  uint32_t a_at[GM], b_at[GN], as_at[GM], bs_at[GN];
#pragma unroll
  for (uint32_t i = 0; i < GM; i++) {
    a_at[i] = min(wave * GM + i, have_a - 1) * pairs * 2048 + lane * 16;
    as_at[i] = min(2 * (wm * GM + i) + half, have_a - 1) * pairs * 128 + place * 2;
  }
#pragma unroll
  for (uint32_t i = 0; i < GN; i++) {
    b_at[i] = min(wave * GN + i, have_b - 1) * pairs * 2048 + lane * 16;
    bs_at[i] = min(2 * (wn * GN + i) + half, have_b - 1) * pairs * 128 + place * 2;
  }
  FK_MX4_LDS char *const a_to = (FK_MX4_LDS char *)mx4_lds + wave * GM * 1024;
  FK_MX4_LDS char *const b_to = (FK_MX4_LDS char *)mx4_lds + SLAB + wave * GN * 1024;
  const uint32_t ra = (2 * wm * GM + half) * 64 + place, rb = SLAB / 16 + (2 * wn * GN + half) * 64 + place;
  fk_float16v acc[GM][GN];
#pragma unroll
  for (uint32_t i = 0; i < GM; i++)
#pragma unroll
    for (uint32_t j = 0; j < GN; j++)
#pragma unroll
      for (int r = 0; r < 16; r++) acc[i][j][r] = 0.0f;
  uint32_t sa[2][GM][2], sb[2][GN][2];
  const uint32_t steps = 2 * pairs, last = steps - 1;
  auto codes = [&](uint32_t step, uint32_t stage) {
    const uint32_t so = min(step, last) * 1024;
#pragma unroll
    for (uint32_t q = 0; q < GM; q++)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(a_src, a_to + stage * STAGE + q * 1024, 16, a_at[q], so, 0, 0);
#pragma unroll
    for (uint32_t q = 0; q < GN; q++)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(b_src, b_to + stage * STAGE + q * 1024, 16, b_at[q], so, 0, 0);
  };
  auto scales = [&](uint32_t (&s)[GM][2], uint32_t (&t)[GN][2], uint32_t pair) {
#pragma unroll
    for (uint32_t h = 0; h < 2; h++) {
#pragma unroll
      for (uint32_t i = 0; i < GM; i++)
        s[i][h] = __builtin_amdgcn_raw_buffer_load_b16(as_src, as_at[i] + 64 * h, pair * 128, 0);
#pragma unroll
      for (uint32_t i = 0; i < GN; i++)
        t[i][h] = __builtin_amdgcn_raw_buffer_load_b16(bs_src, bs_at[i] + 64 * h, pair * 128, 0);
    }
  };
  scales(sa[0], sb[0], 0);
  codes(0, 0);
  codes(1, 1);
  uint32_t at = 0, to = 2;   // the stage a step reads, and the one it loads
  // A step loads the stage that the step before it read, so a wavefront comes
  // to its barrier with its reads done (their products may follow).
#define FK_MX4_MID(TILE, WAIT, S)                                                                             \
  do {                                                                                                        \
    FK_MX4_VMCNT(WAIT);                                                                                       \
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                                                        \
    FK_MX4_BARRIER();                                                                                         \
    __builtin_amdgcn_sched_barrier(0);                                                                        \
    if (TILE == 0) scales(sa[1], sb[1], min(p + 1, pairs - 1));                                               \
    codes((S) + 2, to);                                                                                       \
    const u32x4 *s_ = mx4_lds + at * (STAGE / 16);                                                            \
    u32x4 fa[GM][2], fb[GN][2];                                                                               \
    _Pragma("unroll") for (uint32_t h = 0; h < 2; h++) {                                                      \
      _Pragma("unroll") for (uint32_t j = 0; j < GN; j++) fb[j][h] = s_[rb + 128 * j + 32 * h];               \
      _Pragma("unroll") for (uint32_t i = 0; i < GM; i++) fa[i][h] = s_[ra + 128 * i + 32 * h];               \
    }                                                                                                         \
    _Pragma("unroll") for (uint32_t h = 0; h < 2; h++)                                                        \
    _Pragma("unroll") for (uint32_t i = 0; i < GM; i++)                                                       \
    _Pragma("unroll") for (uint32_t j = 0; j < GN; j++)                                                       \
        acc[i][j] = mx4_mfma32<TILE>(fb[j][h], sb[0][j][h], fa[i][h], sa[0][i][h], acc[i][j]);                \
    at = at == 2 ? 0 : at + 1;                                                                                \
    to = to == 2 ? 0 : to + 1;                                                                                \
  } while (0)
  for (uint32_t p = 0; p < pairs; p++) {
    FK_MX4_MID(0, GM + GN, 2 * p);
    FK_MX4_MID(1, 3 * (GM + GN), 2 * p + 1);
#pragma unroll
    for (uint32_t h = 0; h < 2; h++) {
#pragma unroll
      for (uint32_t i = 0; i < GM; i++) sa[0][i][h] = sa[1][i][h];
#pragma unroll
      for (uint32_t i = 0; i < GN; i++) sb[0][i][h] = sb[1][i][h];
    }
  }
  __builtin_amdgcn_s_waitcnt(0);
  FK_MX4_BARRIER();
#undef FK_MX4_MID
  mx4_store_many<GM, GN, false, T>(a, 16 * tm + 32 * wm * GM, 16 * tn + 32 * wn * GN, acc,
                                   reinterpret_cast<char *>(mx4_lds) + wave * GN * 2048);
}

template <int T>
__device__ __forceinline__ void mx4_gemm_many(const fk_mx4_gemm_args &a) {
  extern __shared__ u32x4 mx4_lds[];
  constexpr uint32_t GB = mx4_many_side / 4;       // a wavefront's blocks of 32, each way
  constexpr uint32_t ROWS = mx4_many_side;         // row tiles of an operand's slab
  constexpr uint32_t SLAB = ROWS * 1024;           // its bytes a step
  constexpr uint32_t STAGE = 2 * SLAB;             // A's, then B's
  constexpr uint32_t Q = ROWS / 4;                 // loads of an operand a wavefront makes a step
  constexpr uint32_t H = GB / 2;                   // A's blocks of half a step
  const uint32_t lane = threadIdx.x % FK_WAVE;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / FK_WAVE);
  const uint32_t wm = wave & 1, wn = wave >> 1;
  const uint32_t pairs = mx4_pairs(a.k), rows_a = mx4_row_tiles(a.m), rows_b = mx4_row_tiles(a.n);
  const uint32_t tiles_m = (rows_a + ROWS - 1) / ROWS, tiles = tiles_m * ((rows_b + ROWS - 1) / ROWS);

  // A tile's sources.  A wavefront's loads: row tiles Q wave + q of each slab
  // (past the last: the last again, whose blocks are not stored), a lane's 16
  // bytes in their place; the scales of its blocks: of row l mod 32, block 2 h
  // + l div 32.
  const uint32_t half = lane % 32 / 16, place = lane / 32 * 16 + lane % 16;
  uint32_t tm, tn;
  __amdgpu_buffer_rsrc_t a_src, b_src, as_src, bs_src;
  uint32_t a_at[Q], b_at[Q], as_at[GB], bs_at[GB];
  auto sources = [&](uint32_t tile) {
    tm = tile % tiles_m * ROWS;
    tn = tile / tiles_m * ROWS;
    const uint32_t have_a = min(rows_a - tm, ROWS), have_b = min(rows_b - tn, ROWS);
    a_src = buffer((const void *)(a.a_codes + (uint64_t)tm * pairs * 2048), (size_t)have_a * pairs * 2048);
    b_src = buffer((const void *)(a.b_codes + (uint64_t)tn * pairs * 2048), (size_t)have_b * pairs * 2048);
    as_src = buffer((const void *)(a.a_scales + (uint64_t)tm * pairs * 128), (size_t)have_a * pairs * 128);
    bs_src = buffer((const void *)(a.b_scales + (uint64_t)tn * pairs * 128), (size_t)have_b * pairs * 128);
#pragma unroll
    for (uint32_t q = 0; q < Q; q++) {
      a_at[q] = min(wave * Q + q, have_a - 1) * pairs * 2048 + lane * 16;
      b_at[q] = min(wave * Q + q, have_b - 1) * pairs * 2048 + lane * 16;
    }
#pragma unroll
    for (uint32_t i = 0; i < GB; i++) {
      as_at[i] = min(2 * (wm * GB + i) + half, have_a - 1) * pairs * 128 + place * 2;
      bs_at[i] = min(2 * (wn * GB + i) + half, have_b - 1) * pairs * 128 + place * 2;
    }
  };
  FK_MX4_LDS char *const stage0 = (FK_MX4_LDS char *)mx4_lds + wave * Q * 1024;
  const uint32_t ra = (2 * wm * GB + half) * 64 + place, rb = SLAB / 16 + (2 * wn * GB + half) * 64 + place;

  fk_float16v acc[GB][GB];
  u32x4 fa0[GB][2], fb0[GB][2], fa1[GB][2], fb1[GB][2];
  uint32_t sa0[GB][2], sb0[GB][2], sa1[GB][2], sb1[GB][2];
#define FK_MX4_PIN(X) asm volatile("" : "+v"(X))
#define FK_MX4_PIN_ACC()                                                    \
  _Pragma("unroll") for (uint32_t i_ = 0; i_ < GB; i_++)                    \
  _Pragma("unroll") for (uint32_t j_ = 0; j_ < GB; j_++) asm volatile("" : "+a"(acc[i_][j_]))
#define FK_MX4_SCALES(SA, SB, P)                                                                              \
  _Pragma("unroll") for (uint32_t i_ = 0; i_ < GB; i_++)                                                      \
  _Pragma("unroll") for (uint32_t h_ = 0; h_ < 2; h_++) {                                                     \
    SA[i_][h_] = __builtin_amdgcn_raw_buffer_load_b16(as_src, as_at[i_] + 64 * h_, (P) * 128, 0);             \
    SB[i_][h_] = __builtin_amdgcn_raw_buffer_load_b16(bs_src, bs_at[i_] + 64 * h_, (P) * 128, 0);             \
  }
#define FK_MX4_MFMAS(TILE, FA, FB, SA, SB, I0)                                                                \
  _Pragma("unroll") for (uint32_t h = 0; h < 2; h++)                                                          \
  _Pragma("unroll") for (uint32_t i = (I0); i < (I0) + H; i++)                                                \
  _Pragma("unroll") for (uint32_t j = 0; j < GB; j++)                                                         \
      acc[i][j] = mx4_mfma32<TILE>(FB[j][h], SB[j][h], FA[i][h], SA[i][h], acc[i][j])
  // One step in two halves, A's blocks 0 .. H - 1 then the rest against all
  // of B's.  The first half issues the loads of A's part of step LOAD (and,
  // where TILE is 0, those of the next pair's scales before them), and reads
  // the next step's B blocks and A blocks 0 .. H - 1; the second B's loads and
  // the next step's other A blocks.  WAIT: the loads that may still be in
  // flight when the step begins.
#define FK_MX4_STEP(TILE, FA, FB, NA, NB, SA, SB, NSA, NSB, WAIT, NEXT_PAIR, LOAD, ST_LOAD, ST_READ)          \
  do {                                                                                                        \
    if (under && p == 0) FK_MX4_VMCNT(FK_MX4_UNDER(WAIT));                                                    \
    else FK_MX4_VMCNT(WAIT);                                                                                  \
    FK_MX4_BARRIER();                                                                                         \
    __builtin_amdgcn_sched_barrier(0);                                                                        \
    const uint32_t so_ = (LOAD) * 1024;                                                                       \
    FK_MX4_LDS char *d_ = stage0 + (ST_LOAD) * STAGE;                                                         \
    const u32x4 *s_ = mx4_lds + (ST_READ) * (STAGE / 16);                                                     \
    if (TILE == 0) FK_MX4_SCALES(NSA, NSB, NEXT_PAIR)                                                         \
    _Pragma("unroll") for (uint32_t q = 0; q < Q; q++)                                                        \
        __builtin_amdgcn_raw_ptr_buffer_load_lds(a_src, d_ + q * 1024, 16, a_at[q], so_, 0, 0);               \
    _Pragma("unroll") for (uint32_t j = 0; j < GB; j++)                                                       \
    _Pragma("unroll") for (uint32_t h = 0; h < 2; h++) NB[j][h] = s_[rb + 128 * j + 32 * h];                  \
    _Pragma("unroll") for (uint32_t i = 0; i < H; i++)                                                        \
    _Pragma("unroll") for (uint32_t h = 0; h < 2; h++) NA[i][h] = s_[ra + 128 * i + 32 * h];                  \
    FK_MX4_MFMAS(TILE, FA, FB, SA, SB, 0);                                                                    \
    _Pragma("unroll") for (uint32_t g_ = 0; g_ < 2 * H * GB; g_++) {                                          \
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                                                      \
      __builtin_amdgcn_sched_group_barrier(0x020, TILE == 0 ? 2 : 1, 0);                                      \
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);                                                      \
    }                                                                                                         \
    __builtin_amdgcn_sched_barrier(0);                                                                        \
    _Pragma("unroll") for (uint32_t i = H; i < GB; i++)                                                       \
    _Pragma("unroll") for (uint32_t h = 0; h < 2; h++) FK_MX4_PIN(FA[i][h]);                                  \
    _Pragma("unroll") for (uint32_t q = 0; q < Q; q++)                                                        \
        __builtin_amdgcn_raw_ptr_buffer_load_lds(b_src, d_ + SLAB + q * 1024, 16, b_at[q], so_, 0, 0);        \
    _Pragma("unroll") for (uint32_t i = H; i < GB; i++)                                                       \
    _Pragma("unroll") for (uint32_t h = 0; h < 2; h++) NA[i][h] = s_[ra + 128 * i + 32 * h];                  \
    FK_MX4_MFMAS(TILE, FA, FB, SA, SB, H);                                                                    \
    _Pragma("unroll") for (uint32_t g_ = 0; g_ < H * GB; g_++) {                                              \
      __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);                                                      \
      __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);                                                      \
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);                                                      \
    }                                                                                                         \
    __builtin_amdgcn_sched_barrier(0);                                                                        \
    _Pragma("unroll") for (uint32_t j = 0; j < GB; j++)                                                       \
    _Pragma("unroll") for (uint32_t h = 0; h < 2; h++) FK_MX4_PIN(NB[j][h]);                                  \
    _Pragma("unroll") for (uint32_t i = 0; i < H; i++)                                                        \
    _Pragma("unroll") for (uint32_t h = 0; h < 2; h++) FK_MX4_PIN(NA[i][h]);                                  \
    FK_MX4_PIN_ACC();                                                                                         \
  } while (0)

  // At step s (after its barrier) step s's blocks are in registers but for
  // A's second half, on its way from stage s mod 4, and steps s + 1 and s + 2
  // are in their stages or on their way there.  Loads past the last step
  // repeat it into stages that no step reads, so every wait counts the same
  // loads.
  const uint32_t steps = 2 * pairs, last = steps - 1;
#define FK_MX4_T(X) ((X) < last ? (X) : last)
  // The first three steps of a tile, and its first scales, on their way.
#define FK_MX4_FIRST()                                                                                        \
  do {                                                                                                        \
    FK_MX4_SCALES(sa0, sb0, 0)                                                                                \
    _Pragma("unroll") for (uint32_t t_ = 0; t_ + 1 < FK_MX4_STAGES; t_++) {                                   \
      const uint32_t so_ = FK_MX4_T(t_) * 1024;                                                               \
      FK_MX4_LDS char *d_ = stage0 + t_ * STAGE;                                                              \
      _Pragma("unroll") for (uint32_t q = 0; q < Q; q++) {                                                    \
        __builtin_amdgcn_raw_ptr_buffer_load_lds(a_src, d_ + q * 1024, 16, a_at[q], so_, 0, 0);               \
        __builtin_amdgcn_raw_ptr_buffer_load_lds(b_src, d_ + SLAB + q * 1024, 16, b_at[q], so_, 0, 0);        \
      }                                                                                                       \
    }                                                                                                         \
  } while (0)
  // Tile after tile, the next one's first loads under this one's stores (which
  // go by way of the fourth stage; step 0 loads it).  The counter that a wait
  // looks at has loads and stores in their order, so the waits of a tile's
  // first pair of steps leave out the stores that went out behind its first
  // loads, whose number is known where the tile before was whole: with the
  // operands from memory each time, 8192 x 8192, k 2048 104.7 µs, so 93.6.  (The
  // compiler's own waits for the tile's first scales count none of the stores,
  // which are conditional, and still hold the first products until all but a few
  // are out.)
  constexpr uint32_t STORES = 32 * GB * 32 * GB * mx4_bytes_of(T) / (16 * FK_WAVE);  // of a whole tile, a wavefront's
#define FK_MX4_UNDER(N) ((N) + STORES < 63 ? (N) + STORES : 63)
  bool under = false;
  sources(blockIdx.x);
  FK_MX4_FIRST();
  for (uint32_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
#pragma unroll
    for (uint32_t i = 0; i < GB; i++)
#pragma unroll
      for (uint32_t j = 0; j < GB; j++)
#pragma unroll
        for (int r = 0; r < 16; r++) acc[i][j][r] = 0.0f;
    // step 0 landed
    if (under) FK_MX4_VMCNT(FK_MX4_UNDER(2 * Q * (FK_MX4_STAGES - 2)));
    else FK_MX4_VMCNT(2 * Q * (FK_MX4_STAGES - 2));
    FK_MX4_BARRIER();
#pragma unroll
    for (uint32_t i = 0; i < GB; i++)
#pragma unroll
      for (uint32_t h = 0; h < 2; h++) {
        fb0[i][h] = mx4_lds[rb + 128 * i + 32 * h];
        fa0[i][h] = mx4_lds[ra + 128 * i + 32 * h];
      }
#pragma unroll
    for (uint32_t i = 0; i < GB; i++)
#pragma unroll
      for (uint32_t h = 0; h < 2; h++) {
        FK_MX4_PIN(fb0[i][h]);
        if (i < H) FK_MX4_PIN(fa0[i][h]);
      }
    for (uint32_t p = 0; p < pairs; p++) {
      const uint32_t s = 2 * p, next = p + 1 < pairs ? p + 1 : p;
      FK_MX4_STEP(0, fa0, fb0, fa1, fb1, sa0, sb0, sa1, sb1, 2 * Q, next, FK_MX4_T(s + 3), (s + 3) % 4, (s + 1) % 4);
      FK_MX4_STEP(1, fa1, fb1, fa0, fb0, sa0, sb0, sa1, sb1, 2 * Q + 4 * GB, next, FK_MX4_T(s + 4), s % 4, (s + 2) % 4);
#pragma unroll
      for (uint32_t i = 0; i < GB; i++)
#pragma unroll
        for (uint32_t h = 0; h < 2; h++) sa0[i][h] = sa1[i][h], sb0[i][h] = sb1[i][h];
    }
    // Nothing lands in LDS any more, and no wavefront reads it.
    __builtin_amdgcn_s_waitcnt(0);
    FK_MX4_BARRIER();
    const uint32_t m = 16 * tm + 32 * wm * GB, n = 16 * tn + 32 * wn * GB;
    under = 16 * tm + 64 * GB <= a.m && 16 * tn + 64 * GB <= a.n;
    if (tile + gridDim.x < tiles) {
      sources(tile + gridDim.x);
      FK_MX4_FIRST();
    }
    mx4_store_many<GB, GB, true, T>(a, m, n, acc,
                                    reinterpret_cast<char *>(mx4_lds) + 3 * STAGE + wave * (STAGE / 4));
  }
#undef FK_MX4_PIN
#undef FK_MX4_PIN_ACC
#undef FK_MX4_SCALES
#undef FK_MX4_MFMAS
#undef FK_MX4_STEP
#undef FK_MX4_FIRST
#undef FK_MX4_UNDER
#undef FK_MX4_T
}

}  // namespace fk
