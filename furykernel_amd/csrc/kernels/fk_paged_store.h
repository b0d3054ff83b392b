// fk_paged_store.h — a step's q, k and v rows: RoPE, q to 16-bit rows, k and v
// into the paged pools at their tokens' slots (include/fkrocm_serve.h:
// fk_paged_store).
//
// Elementwise, so the rows' read and the caches' write bound it.  A thread
// takes 8 elements of a head's first half and the 8 they are paired with:
// 16-byte loads and stores, and each pair's cosine and sine once for both.
// Rows of 16 bits and the caches' elements pass the caches by: 8191 tokens of 32
// and 8 heads of 128 in bf16, out of memory each time, took 41.7 µs, so 35.9
// (203 MB, 5.7 TB/s; the store alone, without what an attention that reads the
// rows next would save); f32 rows, two loads a line, lose by it (4096 tokens of
// heads of 64 16.4 µs, 17.5).  8 tokens take 2.8: the launch and three loads,
// one behind another.
#pragma once

#include "fk_address.h"
#include "fk_common.h"

#include "../../../include/fkrocm_serve.h"

#define FK_STORE_THREADS 256

namespace fk {

typedef float store_float4 __attribute__((ext_vector_type(4)));
typedef float store_float2 __attribute__((ext_vector_type(2)));
typedef _Float16 store_half8 __attribute__((ext_vector_type(8)));
typedef __bf16 store_bf16x8 __attribute__((ext_vector_type(8)));

// Eight elements `at` elements from an address, widened.
template <int T>
__device__ __forceinline__ void load8(uint64_t rows, uint64_t at, float (&x)[8]) {
  if constexpr (T == FK_T_F32) {
    const auto p = global_at<const store_float4>(rows + 4 * at);
    const store_float4 a = p[0], b = p[1];
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = a[i], x[4 + i] = b[i];
  } else if constexpr (T == FK_T_F16) {
    const store_half8 h = load_from<true, store_half8>(global_at<const store_half8>(rows + 2 * at));
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = (float)h[i];
  } else {
    const u32x4 w = load_from<true, u32x4>(global_at<const u32x4>(rows + 2 * at));
#pragma unroll
    for (int i = 0; i < 4; i++) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
}

// Eight elements rounded once, to nearest even, and stored.
template <bool BF16>
__device__ __forceinline__ void store8(uint64_t to, const float (&x)[8]) {
  if constexpr (BF16) {
    store_bf16x8 h;
#pragma unroll
    for (int i = 0; i < 8; i++) h[i] = (__bf16)x[i];
    __builtin_nontemporal_store(h, global_at<store_bf16x8>(to));
  } else {
    store_half8 h;
#pragma unroll
    for (int i = 0; i < 8; i++) h[i] = (_Float16)x[i];
    __builtin_nontemporal_store(h, global_at<store_half8>(to));
  }
}

// Elements e .. e + 7 of a head's first half and those they are paired with,
// turned by row `pos` of the table where they are among the `rotated` pairs.
__device__ __forceinline__ void store_turn(uint64_t rope, uint32_t pos, uint32_t rotated, uint32_t e, float (&x)[8],
                                           float (&y)[8]) {
  const uint64_t cs = rope + 8 * ((uint64_t)pos * rotated + e);
  float c[8], s[8];
  if (rotated % 8 == 0) {
    // whole eights, so four 16-byte loads
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const store_float4 w = global_at<const store_float4>(cs)[j];
      c[2 * j] = w.x, s[2 * j] = w.y, c[2 * j + 1] = w.z, s[2 * j + 1] = w.w;
    }
  } else {
    // the last pair in the place of those past it, which stay as they are
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const store_float2 w = global_at<const store_float2>(cs)[min((uint32_t)j, rotated - 1 - e)];
      c[j] = w.x, s[j] = w.y;
    }
  }
#pragma unroll
  for (int j = 0; j < 8; j++) {
    const float first = x[j] * c[j] - y[j] * s[j], second = y[j] * c[j] + x[j] * s[j];
    x[j] = e + j < rotated ? first : x[j];
    y[j] = e + j < rotated ? second : y[j];
  }
}

// T: the rows' type.  Unit u of a token: head u / (head_dim / 16) of q, then
// k's, then v's, and its elements 8 (u mod (head_dim / 16)) .. + 7 with those
// half a head further.
template <int T, bool BF16>
__device__ __forceinline__ void paged_store(const fk_paged_store_args &a) {
  // (as values: a choice between the struct's fields would put it in scratch)
  const uint64_t q = a.q, k = a.k, v = a.v, q_stride = a.q_stride, k_stride = a.k_stride, v_stride = a.v_stride;
  const uint64_t kpool = a.kpool, vpool = a.vpool;
  const uint32_t heads = a.heads, kv_heads = a.kv_heads, d = a.head_dim, rotated = a.rotated;
  const uint32_t per = d / 16;
  const uint32_t q_heads = q ? heads : 0u;
  const uint32_t units = (q_heads + 2 * kv_heads) * per;
  const uint32_t i = blockIdx.x * FK_STORE_THREADS + threadIdx.x;
  const uint32_t token = i / units;
  if (token >= a.tokens) return;
  const uint32_t u = i - token * units;
  const uint32_t h = u / per, e = 8 * (u - h * per), half = d / 2;
  const bool is_q = h < q_heads, is_v = h >= q_heads + kv_heads;
  const uint32_t head = is_q ? h : h - q_heads - (is_v ? kv_heads : 0u);
  const uint64_t rows = is_q ? q : (is_v ? v : k);
  const uint64_t at = token * (is_q ? q_stride : (is_v ? v_stride : k_stride)) + head * d + e;
  // the rows, the slot and the position in flight together
  float x[8], y[8];
  load8<T>(rows, at, x);
  load8<T>(rows, at + half, y);
  const uint32_t slot = global_at<const uint32_t>(a.slots)[token];
  if (!is_v && e < rotated) {
    store_turn(a.rope, min(global_at<const uint32_t>(a.positions)[token], a.rope_rows - 1), rotated, e, x, y);
  }
  if (slot >= a.blocks * a.block_size) return;
  uint64_t to;
  if (is_q) {
    to = a.qr + 2 * (((uint64_t)token * heads + head) * d + e);
  } else {
    const uint32_t block = slot / a.block_size, within = slot - block * a.block_size;
    to = (is_v ? vpool : kpool) + 2 * ((((uint64_t)block * kv_heads + head) * a.block_size + within) * d + e);
  }
  store8<BF16>(to, x);
  store8<BF16>(to + 2 * half, y);
}

}  // namespace fk
