// fk_fp8.h — 8-bit matrices made and read back (include/fkrocm_fp8.h has the
// format and the order they are held in): of plain rows, and as the RMSNorm of
// a residual stream.
//
// One pass each, so the wide side's stream bounds them: 8192 x 2048 bf16 to 8
// bits 11.6 us (4.3 TB/s), 8191 x 5000 back to bf16 20.5 us (6.0).
#pragma once

#include <cfloat>

#include "fk_e4m3.h"
#include "fk_mx4.h"

#include "../../../include/fkrocm_fp8.h"

#define FK_FP8_THREADS 256
#define FK_FP8_NORM_HELD 4  // the most blocks that a lane of the norm holds a piece of

namespace fk {

__host__ __device__ __forceinline__ uint32_t fp8_row_tiles(uint32_t rows) { return (rows >> 4) + ((rows & 15u) != 0); }
// Blocks of 128 along k, and groups of four of them.
__host__ __device__ __forceinline__ uint32_t fp8_blocks(uint32_t k) { return (k >> 7) + ((k & 127u) != 0); }
__host__ __device__ __forceinline__ uint32_t fp8_quads(uint32_t k) { return (fp8_blocks(k) + 3) / 4; }

// The byte of a row's elements 8 piece .. + 7 (8 codes), and of a block's scale.
__device__ __forceinline__ uint64_t fp8_code_at(uint32_t row, uint32_t piece, uint32_t blocks) {
  return ((uint64_t)(row / 16) * blocks * 2 + piece / 8) * 1024 + (piece % 8 / 2 * 16 + row % 16) * 16 + piece % 2 * 8;
}
__device__ __forceinline__ uint64_t fp8_scale_at(uint32_t row, uint32_t block, uint32_t quads) {
  return ((uint64_t)(row / 16) * quads + block / 4) * 64 + row % 16 * 4 + block % 4;
}

// The maximum over the 16 lanes of a block.
__device__ __forceinline__ uint32_t fp8_row_max(uint32_t x) {
  x = max(x, (uint32_t)dpp_i<0xB1>((int)x));
  x = max(x, (uint32_t)dpp_i<0x4E>((int)x));
  x = max(x, (uint32_t)dpp_i<0x141>((int)x));
  return max(x, (uint32_t)dpp_i<0x140>((int)x));
}

// A lane's 8 elements, whose block the 16 lanes of its row share: codes and
// the scale's byte.
__device__ __forceinline__ u32x2 fp8_encode(float (&x)[8], uint32_t &byte) {
  byte = e4m3_exponent(fp8_row_max(e4m3_largest(x)));
  const float scale = e4m3_scale(byte);
  return u32x2{e4m3_codes(x[0], x[1], x[2], x[3], scale), e4m3_codes(x[4], x[5], x[6], x[7], scale)};
}

// Eight elements from `col` on of a row of k, zeros behind it.
template <int T, bool ONCE>
__device__ __forceinline__ void fp8_load8(uint64_t row, uint32_t col, uint32_t k, float (&x)[8]) {
#pragma unroll
  for (int j = 0; j < 8; j++) x[j] = 0.0f;
  if (col + 8 <= k) {
    mx4_load8<T, ONCE>(row, col, x);
  } else if (col < k) {
#pragma unroll
    for (uint32_t j = 0; j < 7; j++)
      if (col + j < k) x[j] = mx4_load<T>(row, col + j);
  }
}
template <int T>
__device__ __forceinline__ void fp8_store8(uint64_t row, uint32_t col, uint32_t k, const float (&x)[8]) {
  if (col + 8 <= k) {
    mx4_store8<T>(row, col, x);
  } else {
#pragma unroll
    for (uint32_t j = 0; j < 7; j++)
      if (col + j < k) mx4_store<T>(row, col + j, x[j]);
  }
}

// The wavefront's 16 rows by a block, and a lane's piece of 8 elements and its
// row of turn i (4 rows a turn).
struct Fp8Place {
  uint32_t tile, block, piece, sub;
  bool there;
};
__device__ __forceinline__ Fp8Place fp8_place(uint32_t rows, uint32_t k) {
  Fp8Place p;
  const uint32_t blocks = fp8_blocks(k);
  const uint64_t w = (uint64_t)blockIdx.x * (FK_FP8_THREADS / FK_WAVE) + threadIdx.x / FK_WAVE;
  p.there = w < (uint64_t)fp8_row_tiles(rows) * blocks;
  p.tile = __builtin_amdgcn_readfirstlane((uint32_t)w / blocks);
  p.block = __builtin_amdgcn_readfirstlane((uint32_t)w % blocks);
  p.piece = threadIdx.x % 16;
  p.sub = threadIdx.x % FK_WAVE / 16;
  return p;
}

template <int T>
__device__ __forceinline__ void fp8_quantize(const fk_fp8_quantize_args &a) {
  const Fp8Place p = fp8_place(a.rows, a.k);
  if (!p.there) return;
  const uint32_t blocks = fp8_blocks(a.k), quads = fp8_quads(a.k);
  const uint32_t col = p.block * 128 + p.piece * 8;
  float x[4][8];
#pragma unroll
  for (uint32_t i = 0; i < 4; i++) {
    const uint32_t row = 16 * p.tile + 4 * i + p.sub;
    const uint64_t at = a.x + (uint64_t)row * a.x_stride * mx4_bytes_of(T);
    fp8_load8<T, false>(at, row < a.rows ? col : a.k, a.k, x[i]);
  }
#pragma unroll
  for (uint32_t i = 0; i < 4; i++) {
    const uint32_t row = 16 * p.tile + 4 * i + p.sub;
    uint32_t byte;
    const u32x2 codes = fp8_encode(x[i], byte);
    *global_at<u32x2>(a.codes + fp8_code_at(row, p.block * 16 + p.piece, blocks)) = codes;
    // (the last block's lanes 1 to 3 write those of the blocks that fill its four up)
    const uint32_t block = p.block + p.piece;
    if (p.piece == 0 || (p.block == blocks - 1 && block < 4 * quads))
      *global_at<uint8_t>(a.scales + fp8_scale_at(row, block, quads)) =
          (uint8_t)(p.piece == 0 && row < a.rows ? byte : 127u);
  }
}

template <int T>
__device__ __forceinline__ void fp8_dequantize(const fk_fp8_dequantize_args &a) {
  const Fp8Place p = fp8_place(a.rows, a.k);
  const uint32_t col = p.block * 128 + p.piece * 8;
  if (!p.there || col >= a.k) return;
  const uint32_t blocks = fp8_blocks(a.k), quads = fp8_quads(a.k);
  u32x2 codes[4];
  uint32_t bytes[4];
#pragma unroll
  for (uint32_t i = 0; i < 4; i++) {
    const uint32_t row = 16 * p.tile + 4 * i + p.sub;
    codes[i] = *global_at<const u32x2>(a.codes + fp8_code_at(row, p.block * 16 + p.piece, blocks));
    bytes[i] = *global_at<const uint8_t>(a.scales + fp8_scale_at(row, p.block, quads));
  }
#pragma unroll
  for (uint32_t i = 0; i < 4; i++) {
    const uint32_t row = 16 * p.tile + 4 * i + p.sub;
    if (row >= a.rows) continue;
    const float scale = e4m3_scale(bytes[i]);
    float y[8], z[2][4];
    e4m3_values(codes[i][0], z[0]);
    e4m3_values(codes[i][1], z[1]);
#pragma unroll
    for (int j = 0; j < 8; j++) {
      y[j] = z[j / 4][j % 4] * scale;
      // (the product is made before it is rounded: fused with the rounding to
      // f16 it adds a zero, and a code of -0 comes out as +0)
      asm volatile("" : "+v"(y[j]));
    }
    fp8_store8<T>(a.y + (uint64_t)row * a.y_stride * mx4_bytes_of(T), col, a.k, y);
    if (a.scales_out && p.piece == 0) global_at<float>(a.scales_out)[(uint64_t)row * blocks + p.block] = scale;
  }
}

// The norm: s = x + residual, y = s / sqrt(mean(s^2) + eps) * gamma, as codes:
// the exact value's, so the squares are added and their root taken in binary64.
// A row is held in registers from the first load to the codes, so that it is
// read once: 16 lanes a block of 128, H blocks a lane, and a wavefront's four 16s
// four blocks of one row or, with ROWS 2, two of two rows.  Bound by what it moves:
// 7 bytes an element of bf16 with a residual and the sum (a copy reaches 5 to
// 6 TB/s).  A lane's 8 codes are half of a piece of 16, 256 bytes from the row's
// next, so that a row's codes leave as many short writes; two rows' pieces lie
// together.  The 16 rows of a tile go to threadgroups on one XCD (a launch's go to
// the 8 in turn), so that each line of codes is whole in one L2 before it leaves.
//   8191 x 5000 bf16: 72 us, 4.0 TB/s (in binary32, where a code in 2 to 3 10^6 is
//   another, 65; by one row a threadgroup 110); 8192 x 4096 49 us, 4.8 TB/s;
//   29631 x 533 f16 46 us; 8 x 2048 f32 3.6 us.
template <uint32_t ROWS>
__device__ __forceinline__ uint32_t fp8_norm_row(uint32_t group) {
  constexpr uint32_t each = 16 / ROWS;
  const uint32_t i = group / 8;
  return (i / each * 8 + group % 8) * 16 + i % each * ROWS;
}

template <int CTRL>
__device__ __forceinline__ double fp8_dpp(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = (uint32_t)dpp_i<CTRL>((int)(uint32_t)b), hi = (uint32_t)dpp_i<CTRL>((int)(uint32_t)(b >> 32));
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// A row's sum over a threadgroup, the same in every lane of the row.
template <uint32_t ROWS>
__device__ __forceinline__ double fp8_norm_sum(double x, double (&slots)[16][4]) {
  x = x + fp8_dpp<0xB1>(x);
  x = x + fp8_dpp<0x4E>(x);
  x = x + fp8_dpp<0x141>(x);
  x = x + fp8_dpp<0x140>(x);
  const uint32_t lane = threadIdx.x % FK_WAVE, waves = blockDim.x / FK_WAVE;
  if (lane % 16 == 0) slots[threadIdx.x / FK_WAVE][lane / 16] = x;
  __syncthreads();
  double sum = 0.0;
  for (uint32_t w = 0; w < waves; w++) {
    if constexpr (ROWS == 2) sum += slots[w][lane / 32 * 2] + slots[w][lane / 32 * 2 + 1];
    else sum += (slots[w][0] + slots[w][1]) + (slots[w][2] + slots[w][3]);
  }
  return sum;
}

// 1 / sqrt(x) to about 2^-50: 0 of infinity.
__device__ __forceinline__ double fp8_rsqrt(double x) {
  double r = __builtin_amdgcn_rsq(x);
#pragma unroll
  for (int i = 0; i < 2; i++) r = r * __builtin_fma(-0.5 * x * r, r, 1.5);
  return x == __builtin_inf() ? 0.0 : r;
}

// x rounded to the nearest binary32, but to the odd one of two that it lies
// between: rounded once more, to fewer bits, it goes where x would.  Past
// binary32's range, infinite or NaN: as the cast has it.
__device__ __forceinline__ float fp8_odd(double x) {
  const float f = (float)x;
  const uint32_t u = __float_as_uint(f);
  const double off = x - (double)f;
  const bool out = (off > 0.0) == (u >> 31 == 0);
  const bool between = off != 0.0 && (u & 0x7F800000u) != 0x7F800000u;
  return between && (u & 1u) == 0 ? __uint_as_float(out ? u + 1 : u - 1) : f;
}

// x rounded to T and widened again.
template <int T>
__device__ __forceinline__ float fp8_rounded(float x) {
  if constexpr (T == FK_T_F32) return x;
  else if constexpr (T == FK_T_F16) return (float)(_Float16)x;
  else return (float)(__bf16)x;
}

template <int T, uint32_t ROWS, uint32_t H>
__device__ __forceinline__ void fp8_add_norm(const fk_fp8_add_norm_args &a, double over_k) {
  __shared__ double slots[16][4];
  constexpr uint32_t B = mx4_bytes_of(T);
  const uint32_t blocks = fp8_blocks(a.k), quads = fp8_quads(a.k), waves = blockDim.x / FK_WAVE;
  const uint32_t lane = threadIdx.x % FK_WAVE, wave = threadIdx.x / FK_WAVE;
  const uint32_t row = fp8_norm_row<ROWS>(blockIdx.x) + (lane / 16 * ROWS / 4);
  if (row >= 16 * fp8_row_tiles(a.rows)) return;  // (whole threadgroups)
  const bool there = row < a.rows;
  // The blocks of a lane, and its piece of each.
  auto block_of = [&](uint32_t i) { return 4 / ROWS * (wave + i * waves) + lane / 16 % (4 / ROWS); };
  const uint32_t within = 8 * (lane % 16);
  float h[H][8], r[H][8];
#pragma unroll
  for (uint32_t i = 0; i < H; i++) {
    const uint32_t col = there ? 128 * block_of(i) + within : a.k;
    fp8_load8<T, true>(a.x + row * a.x_stride * B, col, a.k, h[i]);
    if (a.residual) fp8_load8<T, true>(a.residual + row * a.residual_stride * B, col, a.k, r[i]);
  }
  double squares = 0.0;
#pragma unroll
  for (uint32_t i = 0; i < H; i++) {
    const uint32_t col = there ? 128 * block_of(i) + within : a.k;
    if (a.residual) {
#pragma unroll
      for (int j = 0; j < 8; j++) h[i][j] = fp8_rounded<T>(h[i][j] + r[i][j]);
    }
    if (a.sum) fp8_store8<T>(a.sum + row * a.sum_stride * B, col, a.k, h[i]);
#pragma unroll
    for (int j = 0; j < 8; j++) squares = __builtin_fma((double)h[i][j], (double)h[i][j], squares);
  }
  const double factor = fp8_rsqrt(fp8_norm_sum<ROWS>(squares, slots) * over_k + (double)a.eps);
  // (past binary32's normal range NaN: each y is made anew)
  const float scale = factor >= FLT_MIN && factor <= FLT_MAX ? (float)factor : __builtin_nanf("");
#pragma unroll
  for (uint32_t i = 0; i < H; i++) {
    const uint32_t block = block_of(i), col = 128 * block + within;
    if (block >= blocks) break;  // (the 16 lanes of a block together)
    float g[8];
    if (a.gamma) {
      fp8_load8<FK_T_F32, false>(a.gamma, col, a.k, g);
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++) g[j] = 1.0f;
    }
    // Off by less than 4 of its last places, y goes to another code than the exact
    // value only beside a halfway case, or the largest of a scale: those have 19
    // zeros at their end.  Few wavefronts hold one that near, and make theirs anew;
    // so do those of a y or a product on its way below binary32's normal range, which
    // holds fewer bits.
    // Zeros look like both, but are exact: a wavefront that holds some looks again
    // without them (a block's turn of a bf16 residual sum holds some 4 times in 10: made
    // anew for them too, 8191 x 5000 took 77 us, so 72 to 74).
    float y[8], least = 1.0f;
    uint32_t near = ~0u;
    auto ends = [](float x) { return (__float_as_uint(x) << 13) + (4u << 13); };
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const float t = h[i][j] * scale;
      y[j] = t * g[j];
      near = min(near, ends(y[j]));
      least = __builtin_fminf(least, __builtin_fminf(__builtin_fabsf(t), __builtin_fabsf(y[j])));
    }
    const bool small = there && least < FLT_MIN;
    if (__builtin_amdgcn_ballot_w64((there && near < 8u << 13) || small)) {
      bool anew = true;
      if (__builtin_amdgcn_ballot_w64(small)) {
        anew = scale != scale;
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const float low = __builtin_fminf(__builtin_fabsf(h[i][j] * scale), __builtin_fabsf(y[j]));
          anew = anew || ((ends(y[j]) < 8u << 13 || low < FLT_MIN) && h[i][j] != 0.0f && g[j] != 0.0f);
        }
      }
      if (__builtin_amdgcn_ballot_w64(anew)) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
          float again = h[i][j];
          asm volatile("" : "+v"(again));  // (widened here: the squares' doubles, kept, halve the threadgroups of a CU)
          y[j] = fp8_odd((double)again * factor * (double)g[j]);
        }
      }
    }
    if (!there || col + 8 > a.k) {
      // (what lies behind the rows and the row is 0 whatever the factor)
#pragma unroll
      for (uint32_t j = 0; j < 8; j++) y[j] = there && col + j < a.k ? y[j] : 0.0f;
    }
    uint32_t byte;
    const u32x2 codes = fp8_encode(y, byte);
    *global_at<u32x2>(a.codes + fp8_code_at(row, col / 8, blocks)) = codes;
    // (the last block's lanes 1 to 3 write the scales of those that fill its four up)
    const uint32_t scaled = block + lane % 16;
    if (lane % 16 == 0 || (block == blocks - 1 && scaled < 4 * quads))
      *global_at<uint8_t>(a.scales + fp8_scale_at(row, scaled, quads)) =
          (uint8_t)(lane % 16 == 0 && there ? byte : 127u);
  }
}

}  // namespace fk
