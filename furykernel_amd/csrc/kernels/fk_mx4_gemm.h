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

// Four consecutive columns n .. n + 3 of row m of C; WIDE: n and the stride
// are multiples of 4 and c is aligned.
template <int T>
__device__ __forceinline__ void mx4_store_c(const fk_mx4_gemm_args &a, bool wide, uint32_t m, uint32_t n, fk_float4v v) {
  if (m >= a.m || n >= a.n) return;
  const uint64_t at = a.c + ((uint64_t)m * a.c_stride + n) * mx4_bytes_of(T);
  if (wide) {
    if constexpr (T == FK_T_F32) {
      *global_at<fk_float4v>(at) = v;
    } else if constexpr (T == FK_T_F16) {
      typedef _Float16 half4 __attribute__((ext_vector_type(4)));
      *global_at<half4>(at) = half4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
    } else {
      typedef __bf16 bf4 __attribute__((ext_vector_type(4)));
      *global_at<bf4>(at) = bf4{(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
    }
  } else {
#pragma unroll
    for (uint32_t r = 0; r < 4; r++)
      if (n + r < a.n) mx4_store<T>(at, r, v[r]);
  }
}
__device__ __forceinline__ bool mx4_wide_c(const fk_mx4_gemm_args &a) {
  return a.n % 4 == 0 && a.c_stride % 4 == 0 && a.c % 16 == 0;
}

// Few rows: a threadgroup takes MB × NB blocks of 16 × 16, its W wavefronts
// every W-th pair of tiles along k, the operands straight from memory; the
// wavefronts' sums are added in their order in LDS.
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
  if (wave < pairs) {
    Pair now = load(wave);
    for (uint32_t p = wave; p < pairs; p += W) {
      const Pair next = load(min(p + W, pairs - 1));
#pragma unroll
      for (uint32_t i = 0; i < MB; i++)
#pragma unroll
        for (uint32_t j = 0; j < NB; j++) acc[i][j] = mx4_mfma<0>(now.b[j][0], now.bs[j], now.a[i][0], now.as[i], acc[i][j]);
#pragma unroll
      for (uint32_t i = 0; i < MB; i++)
#pragma unroll
        for (uint32_t j = 0; j < NB; j++) acc[i][j] = mx4_mfma<1>(now.b[j][1], now.bs[j], now.a[i][1], now.as[i], acc[i][j]);
      now = next;
    }
  }
#pragma unroll
  for (uint32_t i = 0; i < MB; i++)
#pragma unroll
    for (uint32_t j = 0; j < NB; j++) sums[wave][i * NB + j][lane] = acc[i][j];
  __syncthreads();
  const bool wide = mx4_wide_c(a);
  for (uint32_t b = wave; b < MB * NB; b += W) {
    fk_float4v v = sums[0][b][lane];
#pragma unroll
    for (uint32_t w = 1; w < W; w++) v += sums[w][b][lane];
    mx4_store_c<T>(a, wide, 16 * (tm + b / NB) + lane % 16, 16 * (tn + b % NB) + 4 * (lane / 16), v);
  }
}

}  // namespace fk
