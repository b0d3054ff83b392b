// fk_paged_store.h — a step's q, k and v rows: RoPE, q to 16-bit rows, k and v
// into the paged pools at their tokens' slots (include/fkrocm_serve.h:
// fk_paged_store).
//
// Elementwise, so the rows' read and the caches' write bound it.  A thread
// takes 8 elements of a head's first half and the 8 they are paired with:
// 16-byte loads and stores, and each pair's cosine and sine once for both.
#pragma once

#include "fk_common.h"

#include "../../../include/fkrocm_serve.h"

#define FK_STORE_THREADS 256

namespace fk {

typedef _Float16 store_half8 __attribute__((ext_vector_type(8)));
typedef __bf16 store_bf16x8 __attribute__((ext_vector_type(8)));

// Eight elements of a row, widened.
template <int T>
__device__ __forceinline__ void load8(const void *rows, uint64_t at, float (&x)[8]) {
  if constexpr (T == FK_T_F32) {
    const float4 a = reinterpret_cast<const float4 *>(static_cast<const float *>(rows) + at)[0];
    const float4 b = reinterpret_cast<const float4 *>(static_cast<const float *>(rows) + at)[1];
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else if constexpr (T == FK_T_F16) {
    const store_half8 h = *reinterpret_cast<const store_half8 *>(static_cast<const uint16_t *>(rows) + at);
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = (float)h[i];
  } else {
    const uint4 w = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(rows) + at);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      x[2 * i] = __uint_as_float(u[i] << 16);
      x[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
    }
  }
}

// Eight elements rounded once, to nearest even, and stored.
template <bool BF16>
__device__ __forceinline__ void store8(uint16_t *to, const float (&x)[8]) {
  if constexpr (BF16) {
    store_bf16x8 h;
#pragma unroll
    for (int i = 0; i < 8; i++) h[i] = (__bf16)x[i];
    *reinterpret_cast<store_bf16x8 *>(to) = h;
  } else {
    store_half8 h;
#pragma unroll
    for (int i = 0; i < 8; i++) h[i] = (_Float16)x[i];
    *reinterpret_cast<store_half8 *>(to) = h;
  }
}

// T: the rows' type.  Unit u of a token: head u / (head_dim / 16) of q, then
// k's, then v's, and its elements 8 (u mod (head_dim / 16)) .. + 7 with those
// half a head further.
template <int T, bool BF16>
__device__ __forceinline__ void paged_store(const fk_paged_store_args &a) {
  const uint32_t per = a.head_dim / 16;
  const uint32_t q_heads = a.q ? a.heads : 0u;
  const uint32_t units = (q_heads + 2 * a.kv_heads) * per;
  const uint32_t i = blockIdx.x * FK_STORE_THREADS + threadIdx.x;
  const uint32_t token = i / units;
  if (token >= a.tokens) return;
  const uint32_t u = i - token * units;
  const uint32_t slot = reinterpret_cast<const uint32_t *>(a.slots)[token];
  if (slot >= a.blocks * a.block_size) return;
  const uint32_t h = u / per, e = 8 * (u - h * per), half = a.head_dim / 2;
  const bool is_q = h < q_heads, is_v = h >= q_heads + a.kv_heads;
  const uint32_t head = is_q ? h : h - q_heads - (is_v ? a.kv_heads : 0u);
  const void *rows = reinterpret_cast<const void *>(is_q ? a.q : (is_v ? a.v : a.k));
  const uint64_t at = token * (is_q ? a.q_stride : (is_v ? a.v_stride : a.k_stride)) + head * a.head_dim + e;
  float x[8], y[8];
  load8<T>(rows, at, x);
  load8<T>(rows, at + half, y);
  if (!is_v && e < a.rotated) {
    const uint32_t pos = min(reinterpret_cast<const uint32_t *>(a.positions)[token], a.rope_rows - 1);
    const float *cs = reinterpret_cast<const float *>(a.rope) + 2 * ((uint64_t)pos * a.rotated + e);
#pragma unroll
    for (int j = 0; j < 8; j++)
      if (e + j < a.rotated) {
        const float c = cs[2 * j], s = cs[2 * j + 1];
        const float first = x[j] * c - y[j] * s;
        y[j] = y[j] * c + x[j] * s;
        x[j] = first;
      }
  }
  uint16_t *to;
  if (is_q) {
    to = reinterpret_cast<uint16_t *>(a.qr) + ((uint64_t)token * a.heads + head) * a.head_dim + e;
  } else {
    const uint32_t block = slot / a.block_size, within = slot - block * a.block_size;
    to = reinterpret_cast<uint16_t *>(is_v ? a.vpool : a.kpool) +
         (((uint64_t)block * a.kv_heads + head) * a.block_size + within) * a.head_dim + e;
  }
  store8<BF16>(to, x);
  store8<BF16>(to + half, y);
}

}  // namespace fk
