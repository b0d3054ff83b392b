// fk_mx4.h — 4-bit microscaled matrices made and read back (include/
// fkrocm_mx4.h has the format and the order they are held in).
//
// Both are one pass, so the wide side's stream bounds them.  A wavefront
// takes a tile, 16 rows by 128 elements: a lane 8 consecutive elements of a row
// at a time, 16 lanes a row's 128, so loads are whole lines of 4 rows;
// the four lanes of a block share its maximum by quad permutes, and a lane's
// codes are one word, 64 bytes together in the tile's order.  The conversions
// are the hardware's scaled ones (v_cvt_scalef32_pk_fp4_f32 and back).
// Measured on 8192 x 8192, out of memory each time: bf16 made in 33.0 µs (5.2
// TB/s), read back in 32.7; f32 56.9 and 66.4 (73.9 in stores of 16 bytes
// apart).
#pragma once

#include "fk_address.h"
#include "fk_common.h"

#include "../../../include/fkrocm_mx4.h"

#define FK_MX4_THREADS 256

namespace fk {

typedef float mx4_float2 __attribute__((ext_vector_type(2)));
// Pieces of rows, which start anywhere: 16 bytes at any element's address are
// one load or store (8192 rows of 8191 in bf16: 36.5 µs, of 8192 28.3; an
// element at a time took twice the first).
typedef float mx4_float4 __attribute__((ext_vector_type(4), aligned(4)));
typedef _Float16 mx4_half8 __attribute__((ext_vector_type(8), aligned(2)));
typedef __bf16 mx4_bf16x8 __attribute__((ext_vector_type(8), aligned(2)));
typedef uint32_t mx4_u32x4 __attribute__((ext_vector_type(4), aligned(2)));

// Pairs of tiles along k.
__host__ __device__ __forceinline__ uint32_t mx4_pairs(uint32_t k) { return (k >> 8) + ((k & 255u) != 0); }
__host__ __device__ __forceinline__ uint32_t mx4_row_tiles(uint32_t rows) { return (rows >> 4) + ((rows & 15u) != 0); }

__host__ __device__ constexpr uint32_t mx4_bytes_of(int type) { return type == FK_T_F32 ? 4 : 2; }

// Element i of a row of type T.
template <int T>
__device__ __forceinline__ float mx4_load(uint64_t row, uint64_t i) {
  if constexpr (T == FK_T_F32) return global_at<const float>(row)[i];
  else if constexpr (T == FK_T_F16) return (float)global_at<const _Float16>(row)[i];
  else return __uint_as_float((uint32_t)global_at<const uint16_t>(row)[i] << 16);
}
// Eight from element i on.
template <int T, bool ONCE>
__device__ __forceinline__ void mx4_load8(uint64_t row, uint64_t i, float (&x)[8]) {
  if constexpr (T == FK_T_F32) {
    const auto p = global_at<const mx4_float4>(row + 4 * i);
    const mx4_float4 a = load_from<ONCE, mx4_float4>(p), b = load_from<ONCE, mx4_float4>(p + 1);
#pragma unroll
    for (int j = 0; j < 4; j++) x[j] = a[j], x[4 + j] = b[j];
  } else if constexpr (T == FK_T_F16) {
    const mx4_half8 h = load_from<ONCE, mx4_half8>(global_at<const mx4_half8>(row + 2 * i));
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = (float)h[j];
  } else {
    const mx4_u32x4 w = load_from<ONCE, mx4_u32x4>(global_at<const mx4_u32x4>(row + 2 * i));
#pragma unroll
    for (int j = 0; j < 4; j++) {
      x[2 * j] = __uint_as_float(w[j] << 16);
      x[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
    }
  }
}
template <int T>
__device__ __forceinline__ void mx4_store(uint64_t row, uint64_t i, float x) {
  if constexpr (T == FK_T_F32) global_at<float>(row)[i] = x;
  else if constexpr (T == FK_T_F16) global_at<_Float16>(row)[i] = (_Float16)x;
  else global_at<__bf16>(row)[i] = (__bf16)x;
}
template <int T>
__device__ __forceinline__ void mx4_store8(uint64_t row, uint64_t i, const float (&x)[8]) {
  if constexpr (T == FK_T_F32) {
    const auto p = global_at<mx4_float4>(row + 4 * i);
    p[0] = mx4_float4{x[0], x[1], x[2], x[3]};
    p[1] = mx4_float4{x[4], x[5], x[6], x[7]};
  } else if constexpr (T == FK_T_F16) {
    mx4_half8 h;
#pragma unroll
    for (int j = 0; j < 8; j++) h[j] = (_Float16)x[j];
    *global_at<mx4_half8>(row + 2 * i) = h;
  } else {
    mx4_bf16x8 h;
#pragma unroll
    for (int j = 0; j < 8; j++) h[j] = (__bf16)x[j];
    *global_at<mx4_bf16x8>(row + 2 * i) = h;
  }
}

// The wavefront's tile: its row tile and place along k (the second of the last
// pair may lie past k), and where a lane's 8 elements of turn i lie.
struct Mx4Place {
  uint32_t tile, step, piece, sub;
  bool there;
};
__device__ __forceinline__ Mx4Place mx4_place(uint32_t rows, uint32_t k) {
  Mx4Place p;
  const uint32_t steps = 2 * mx4_pairs(k);
  const uint64_t w = (uint64_t)blockIdx.x * (FK_MX4_THREADS / FK_WAVE) + threadIdx.x / FK_WAVE;
  p.there = w < (uint64_t)mx4_row_tiles(rows) * steps;
  p.tile = __builtin_amdgcn_readfirstlane((uint32_t)w / steps);
  p.step = __builtin_amdgcn_readfirstlane((uint32_t)w % steps);
  p.piece = threadIdx.x % 16;
  p.sub = threadIdx.x % FK_WAVE / 16;
  return p;
}
// The byte of a lane's word of codes, and of its block's scale.
__device__ __forceinline__ uint64_t mx4_code_at(const Mx4Place &p, uint32_t k, uint32_t i) {
  return ((uint64_t)p.tile * 2 * mx4_pairs(k) + p.step) * 1024 + (p.piece / 4 * 16 + 4 * i + p.sub) * 16 +
         p.piece % 4 * 4;
}
__device__ __forceinline__ uint64_t mx4_scale_at(const Mx4Place &p, uint32_t k, uint32_t i) {
  return ((uint64_t)p.tile * mx4_pairs(k) + p.step / 2) * 128 + (p.piece / 4 * 16 + 4 * i + p.sub) * 2 + p.step % 2;
}

template <int T, bool ONCE>
__device__ __forceinline__ void mx4_quantize(const fk_mx4_quantize_args &a) {
  const Mx4Place p = mx4_place(a.rows, a.k);
  if (!p.there) return;
  const uint32_t col = p.step * 128 + p.piece * 8;
  float x[4][8];
#pragma unroll
  for (uint32_t i = 0; i < 4; i++) {
    const uint32_t row = 16 * p.tile + 4 * i + p.sub;
    const uint64_t at = a.x + (uint64_t)row * a.x_stride * mx4_bytes_of(T);
#pragma unroll
    for (int j = 0; j < 8; j++) x[i][j] = 0.0f;
    if (row < a.rows && col + 8 <= a.k) {
      mx4_load8<T, ONCE>(at, col, x[i]);
    } else if (row < a.rows && col < a.k) {
#pragma unroll
      for (uint32_t j = 0; j < 7; j++)
        if (col + j < a.k) x[i][j] = mx4_load<T>(at, col + j);
    }
  }
#pragma unroll
  for (uint32_t i = 0; i < 4; i++) {
    // the largest magnitude as its bits (NaN above infinity above the rest)
    uint32_t big = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) big = max(big, __float_as_uint(x[i][j]) & 0x7FFFFFFFu);
    big = max(big, (uint32_t)dpp_i<0xB1>((int)big));
    big = max(big, (uint32_t)dpp_i<0x4E>((int)big));
    const uint32_t e = big >> 23;
    const uint32_t b = big == 0 ? 127u : (e == 255 ? 255u : (e > 2 ? e - 2 : 0u));
    // small scales with the elements at 2^64 times themselves: the conversion
    // takes a normal scale
    const bool low = b < 64;
    const float up = low ? 18446744073709551616.0f : 1.0f;
    const float scale = __uint_as_float((low ? b + 64 : b) << 23);
    uint32_t code = 0;
#define FK_MX4_CODE(J) \
  code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x[i][2 * J] * up, x[i][2 * J + 1] * up, scale, J)
    FK_MX4_CODE(0);
    FK_MX4_CODE(1);
    FK_MX4_CODE(2);
    FK_MX4_CODE(3);
#undef FK_MX4_CODE
    *global_at<uint32_t>(a.codes + mx4_code_at(p, a.k, i)) = b == 255 ? 0u : code;
    if (p.piece % 4 == 0) *global_at<uint8_t>(a.scales + mx4_scale_at(p, a.k, i)) = (uint8_t)b;
  }
}

template <int T>
__device__ __forceinline__ void mx4_dequantize(const fk_mx4_dequantize_args &a) {
  const Mx4Place p = mx4_place(a.rows, a.k);
  const uint32_t col = p.step * 128 + p.piece * 8;
  if (!p.there || col >= a.k) return;
  uint32_t code[4], scales[4];
#pragma unroll
  for (uint32_t i = 0; i < 4; i++) {
    scales[i] = *global_at<const uint8_t>(a.scales + mx4_scale_at(p, a.k, i));
    code[i] = *global_at<const uint32_t>(a.codes + mx4_code_at(p, a.k, i));
  }
#pragma unroll
  for (uint32_t i = 0; i < 4; i++) {
    const uint32_t row = 16 * p.tile + 4 * i + p.sub, b = scales[i];
    if (row >= a.rows) continue;
    // 2^(b - 127), of which b = 0 is no normal number
    const float scale = b == 255 ? __builtin_nanf("") : __uint_as_float(b ? b << 23 : 0x00400000u);
    float y[8];
#define FK_MX4_VALUE(J)                                                                     \
  {                                                                                         \
    const mx4_float2 v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code[i], 1.0f, J);        \
    y[2 * J] = v[0] * scale;                                                                \
    y[2 * J + 1] = v[1] * scale;                                                            \
  }
    FK_MX4_VALUE(0);
    FK_MX4_VALUE(1);
    FK_MX4_VALUE(2);
    FK_MX4_VALUE(3);
#undef FK_MX4_VALUE
    // (the product is made before it is rounded: fused with the rounding to
    // f16 it adds a zero, and a code of -0 comes out as +0)
#pragma unroll
    for (int j = 0; j < 8; j++) asm volatile("" : "+v"(y[j]));
    const uint64_t at = a.y + (uint64_t)row * a.y_stride * mx4_bytes_of(T);
    if (T == FK_T_F32 && p.step * 128 + p.piece / 4 * 32 + 32 <= a.k) {
      // a whole block: its four lanes' 128 bytes as two stores of 64 together
      const uint32_t q = p.piece % 4;
      mx4_float4 w[2];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        // (quad_perm [0, 0, 1, 1] and [2, 2, 3, 3])
        const float lo[2] = {dpp_f<0x50>(y[j]), dpp_f<0xFA>(y[j])};
        const float hi[2] = {dpp_f<0x50>(y[4 + j]), dpp_f<0xFA>(y[4 + j])};
        w[0][j] = q % 2 ? hi[0] : lo[0];
        w[1][j] = q % 2 ? hi[1] : lo[1];
      }
      const auto to = global_at<mx4_float4>(at + 4ull * (p.step * 128 + p.piece / 4 * 32));
      to[q] = w[0];
      to[4 + q] = w[1];
    } else if (col + 8 <= a.k) {
      mx4_store8<T>(at, col, y);
    } else {
#pragma unroll
      for (uint32_t j = 0; j < 7; j++)
        if (col + j < a.k) mx4_store<T>(at, col + j, y[j]);
    }
    if (a.scales_out && p.piece % 4 == 0)
      global_at<float>(a.scales_out)[(uint64_t)row * ((a.k >> 5) + ((a.k & 31u) != 0)) + col / 32] = scale;
  }
}

}  // namespace fk
