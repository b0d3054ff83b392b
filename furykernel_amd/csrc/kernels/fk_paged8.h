// fk_paged8.h — 8-bit paged caches written and read back (include/
// fkrocm_paged8.h: fk_paged_store8, fk_paged_load8).
//
// The store.  A block's scale needs the largest magnitude of its new rows
// before the first code, so W wavefronts take a run (the step's tokens of one
// block) for one head's keys or values: they make the rows, hold them in
// registers where the run is at most a piece a thread, meet at the largest,
// and write the codes.  Rows held before a scale that grew are brought to it
// by the same wavefronts; the scales are powers of two, so only codes that fall
// below the new scale's smallest step change their value.  The queries are
// elementwise and go to threadgroups of their own in the same launch.
//
// Bound by what it moves (a head's row of bf16: 3 bytes an element of k and v, 4
// of q) where there are many tokens, by its chain of loads (slots; rows and
// turns; then the codes) where there are few.  6443 tokens of 32 + 16 heads of 128
// in blocks of 16: 30.3 us, 4.8 TB/s (its queries alone 22.7, its runs alone
// 16.9; with two pieces a thread, and so half the wavefronts, and each token's slot
// and position read where they are used, 43.6).  8 tokens: 3.8 us.
// The load is bound by its writes: 32767 tokens of 8 heads of 128 to bf16 31.6 us,
// 6.4 TB/s.
#pragma once

#include "fk_divisor.h"
#include "fk_e4m3.h"
#include "fk_paged_store.h"

#include "../../../include/fkrocm_paged8.h"

namespace fk {

// What the store's kernel takes beside the call's arguments.
struct Store8Plan {
  Divisor block;        // by block_size
  uint32_t kv_groups;   // the first threadgroups: runs; the rest: queries
  uint32_t chunk;       // tokens whose runs (begun among them) a run's wavefronts take
};

// A token's position, if there are any.
__device__ __forceinline__ uint32_t store8_position(const fk_paged_store8_args &a, uint32_t token) {
  return a.rotated ? global_at<const uint32_t>(a.positions)[token] : 0u;
}

// T: the rows' type.  One piece of a row: elements e .. e + 7 of a head and
// those half a head further, turned if they are a query's or a key's.
template <int T>
__device__ __forceinline__ void store8_piece(const fk_paged_store8_args &a, uint64_t rows, uint64_t stride,
                                             uint32_t token, uint32_t position, uint32_t head, uint32_t e,
                                             bool turned, float (&x)[8], float (&y)[8]) {
  const uint64_t at = token * stride + head * a.head_dim + e;
  load8<T>(rows, at, x);
  load8<T>(rows, at + a.head_dim / 2, y);
  if (turned && e < a.rotated) store_turn(a.rope, min(position, a.rope_rows - 1), a.rotated, e, x, y);
}

template <int T, bool BF16>
__device__ __forceinline__ void store8_queries(const fk_paged_store8_args &a, uint32_t group) {
  const uint32_t per = a.head_dim / 16, units = a.heads * per;
  const uint32_t i = group * blockDim.x + threadIdx.x;
  const uint32_t token = i / units;
  if (token >= a.tokens) return;
  const uint32_t u = i - token * units, h = u / per, e = 8 * (u - h * per);
  const uint32_t slot = global_at<const uint32_t>(a.slots)[token];
  float x[8], y[8];
  store8_piece<T>(a, a.q, a.q_stride, token, store8_position(a, token), h, e, true, x, y);
  if (slot >= a.blocks * a.block_size) return;
  const uint64_t to = a.qr + 2 * (((uint64_t)token * a.heads + h) * a.head_dim + e);
  store8<BF16>(to, x);
  store8<BF16>(to + a.head_dim, y);
}

// The maximum over a wavefront, in every lane.
__device__ __forceinline__ uint32_t wave_most(uint32_t v) {
  v = max(v, (uint32_t)dpp_i<0xB1>((int)v));
  v = max(v, (uint32_t)dpp_i<0x4E>((int)v));
  v = max(v, (uint32_t)dpp_i<0x141>((int)v));
  v = max(v, (uint32_t)dpp_i<0x140>((int)v));
  const uint32_t a = max((uint32_t)__builtin_amdgcn_readlane((int)v, 0), (uint32_t)__builtin_amdgcn_readlane((int)v, 16));
  const uint32_t b = max((uint32_t)__builtin_amdgcn_readlane((int)v, 32), (uint32_t)__builtin_amdgcn_readlane((int)v, 48));
  return max(a, b);
}

// W wavefronts a run: 1 (four runs' a threadgroup), 2, 4 or 8.
template <int T, uint32_t W>
__device__ __forceinline__ void store8_runs(const fk_paged_store8_args &a, const Store8Plan &pl) {
  __shared__ uint32_t most[W];
  constexpr uint32_t THREADS = 64 * W;
  const uint32_t lane = threadIdx.x % FK_WAVE;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / FK_WAVE);
  const uint32_t thread = W == 1 ? lane : threadIdx.x;
  // The unit: a chunk of tokens, and a head's keys or values.
  const uint32_t units = 2 * a.kv_heads;
  const uint32_t unit = W == 1 ? blockIdx.x * 4 + wave : blockIdx.x;
  const uint32_t first = unit / units * pl.chunk;
  if (first >= a.tokens) return;  // (whole runs of wavefronts)
  const uint32_t pair = unit % units;
  const bool is_v = pair >= a.kv_heads;
  const uint32_t head = is_v ? pair - a.kv_heads : pair;
  const auto slots = global_at<const uint32_t>(a.slots);
  const uint32_t places = a.blocks * a.block_size, tokens = a.tokens, d = a.head_dim, per = d / 16;
  const uint64_t rows = is_v ? a.v : a.k, stride = is_v ? a.v_stride : a.k_stride;
  const uint64_t pool = is_v ? a.vpool : a.kpool;
  // A token's block; NONE if it is stored nowhere.
  constexpr uint32_t NONE = 0xFFFFFFFFu;
  auto block_of = [&](uint32_t slot) { return slot < places ? quotient(slot, pl.block) : NONE; };

  // 64 tokens from `base` on, a lane each: what the runs within them need of
  // them is read once, and together.
  uint32_t base = first, my_slot, my_block, my_position;
  auto look = [&]() {
    const uint32_t t = min(base + lane, tokens - 1);
    my_slot = slots[t];
    my_position = is_v ? 0u : store8_position(a, t);
    my_block = block_of(my_slot);
  };
  const uint32_t before = slots[max(min(first + lane, tokens - 1), 1u) - 1];
  look();
  // The chunk's tokens that begin runs.
  const uint32_t my_token = first + lane;
  uint64_t begins = __builtin_amdgcn_ballot_w64(lane < pl.chunk && my_token < tokens && my_block != NONE &&
                                                (my_token == 0 || my_block != block_of(before)));
  const uint32_t my_row = thread / per, my_e = 8 * (thread - my_row * per);
  for (; begins; begins &= begins - 1) {
    const uint32_t t0 = first + __builtin_ctzll(begins);
    const uint32_t block = __builtin_amdgcn_readlane((int)my_block, (int)(t0 - base));
    // Its tokens from `from` on among the 64 that the lanes hold there.
    auto tokens_at = [&](uint32_t from) {
      const uint64_t run = __builtin_amdgcn_ballot_w64(base + lane < tokens && my_block == block) >> (from - base);
      return ~run ? (uint32_t)__builtin_ctzll(~run) : 64u;
    };
    uint32_t n = tokens_at(t0);
    if (t0 != base && t0 + n == base + 64) {  // a run that may go on: the lanes from its start
      base = t0;
      look();
      n = tokens_at(t0);
    }
    const uint32_t offset = t0 - base;
    const uint32_t place0 = (uint32_t)__builtin_amdgcn_readlane((int)my_slot, (int)offset) - block * a.block_size;
    if (n == 64) {
      uint64_t run;
      for (;; n += 64) {
        const uint32_t t = t0 + n + lane;
        run = __builtin_amdgcn_ballot_w64(t < tokens && block_of(slots[min(t, tokens - 1)]) == block);
        if (~run) break;
      }
      n += __builtin_ctzll(~run);
    }
    const uint64_t at = (uint64_t)block * a.kv_heads + head;
    const auto scale_at = global_at<uint32_t>(a.scales + 8 * at + 4 * is_v);
    const uint32_t old = place0 ? *scale_at : 0u;
    const uint32_t pieces = n * per;
    float x[8], y[8];
    auto make = [&](uint32_t row, uint32_t e, uint32_t position) {
      store8_piece<T>(a, rows, stride, t0 + row, position, head, e, !is_v, x, y);
      return max(e4m3_largest(x), e4m3_largest(y));
    };
    const bool held = pieces <= THREADS && n <= 64;
    uint32_t big = 0, my_place = 0;  // (the place of the thread's row if the run is held)
    if (held) {
      const int from = 4 * (int)(offset + min(my_row, n - 1));
      my_place = (uint32_t)__builtin_amdgcn_ds_bpermute(from, (int)my_slot) - block * a.block_size;
      const uint32_t position = (uint32_t)__builtin_amdgcn_ds_bpermute(from, (int)my_position);
      if (thread < pieces) big = make(my_row, my_e, position);
    } else {
      for (uint32_t i = thread; i < pieces; i += THREADS) {
        const uint32_t row = i / per;
        big = max(big, make(row, 8 * (i - row * per), is_v ? 0u : store8_position(a, t0 + row)));
      }
    }
    big = wave_most(big);
    asm volatile("" ::"v"(old));  // read before the scale is written
    if constexpr (W > 1) {
      if (lane == 0) most[wave] = big;
      __syncthreads();
      big = most[0];
#pragma unroll
      for (uint32_t w = 1; w < W; w++) big = max(big, most[w]);
    }
    // (positive floats are in the order of their bits; a scale that is not one of
    // a store's makes values that mean nothing)
    const uint32_t bits = max(old, e4m3_exponent(big) << 23);
    const float scale = __uint_as_float(bits);
    if (bits != old) {
      if (thread == 0) *scale_at = bits;
      const float factor = __uint_as_float(old) / scale;
      const uint64_t from = pool + at * a.block_size * d;
      for (uint32_t i = thread; i < place0 * per; i += THREADS) {
        const auto p = global_at<u32x4>(from + 16ull * i);
        u32x4 w = *p;
#pragma unroll
        for (int j = 0; j < 4; j++) {
          float v[4];
          e4m3_values(w[j], v);
          w[j] = e4m3_codes(v[0] * factor, v[1] * factor, v[2] * factor, v[3] * factor, 1.0f);
        }
        *p = w;
      }
    }
    auto put = [&](uint32_t place, uint32_t e) {
      const uint64_t to = pool + (at * a.block_size + place) * d + e;
      *global_at<u32x2>(to) = u32x2{e4m3_codes(x[0], x[1], x[2], x[3], scale), e4m3_codes(x[4], x[5], x[6], x[7], scale)};
      *global_at<u32x2>(to + d / 2) =
          u32x2{e4m3_codes(y[0], y[1], y[2], y[3], scale), e4m3_codes(y[4], y[5], y[6], y[7], scale)};
    };
    if (held) {
      if (thread < pieces) put(my_place, my_e);
    } else {
      for (uint32_t i = thread; i < pieces; i += THREADS) {
        const uint32_t row = i / per, e = 8 * (i - row * per);
        make(row, e, is_v ? 0u : store8_position(a, t0 + row));
        put(slots[t0 + row] - block * a.block_size, e);
      }
    }
    if constexpr (W > 1) __syncthreads();  // the largest are read before the next run's
  }
}

template <int T, bool BF16, uint32_t W>
__device__ __forceinline__ void paged_store8(const fk_paged_store8_args &a, const Store8Plan &pl) {
  if (blockIdx.x < pl.kv_groups) store8_runs<T, W>(a, pl);
  else store8_queries<T, BF16>(a, blockIdx.x - pl.kv_groups);
}

#define FK_LOAD8_THREADS 256

// Eight elements a thread: unit u of a token, of k's heads then v's.
template <int T>
__device__ __forceinline__ void paged_load8(const fk_paged_load8_args &a, const Divisor &block, const Divisor &units) {
  const uint64_t kpool = a.kpool, vpool = a.vpool, k = a.k, v = a.v, k_stride = a.k_stride, v_stride = a.v_stride;
  const uint32_t d = a.head_dim, row = a.kv_heads * d / 8;  // of k, or of v
  const uint32_t i = blockIdx.x * FK_LOAD8_THREADS + threadIdx.x;
  const uint32_t token = quotient(i, units);
  if (token >= a.tokens) return;
  uint32_t u = i - token * 2 * row;
  const uint32_t slot = global_at<const uint32_t>(a.slots)[token];
  if (slot >= a.blocks * a.block_size) return;
  const bool is_v = u >= row;
  u -= is_v ? row : 0u;
  const uint32_t head = 8 * u / d, e = 8 * u - head * d;
  const uint32_t b = quotient(slot, block), within = slot - b * a.block_size;
  const uint64_t at = (uint64_t)b * a.kv_heads + head;
  const u32x2 w = *global_at<const u32x2>((is_v ? vpool : kpool) + (at * a.block_size + within) * d + e);
  const float scale = *global_at<const float>(a.scales + 8 * at + 4 * is_v);
  float x[2][4], y[8];
  e4m3_values(w[0], x[0]);
  e4m3_values(w[1], x[1]);
#pragma unroll
  for (int j = 0; j < 8; j++) {
    y[j] = x[j / 4][j % 4] * scale;
    asm volatile("" : "+v"(y[j]));  // (not fused with its rounding, which would lose a -0's sign)
  }
  const uint64_t to = (is_v ? v : k), where = token * (is_v ? v_stride : k_stride) + 8 * u;
  if constexpr (T == FK_T_F32) {
    const auto p = global_at<store_float4>(to + 4 * where);
    p[0] = store_float4{y[0], y[1], y[2], y[3]};
    p[1] = store_float4{y[4], y[5], y[6], y[7]};
  } else {
    store8<T == FK_T_BF16>(to + 2 * where, y);
  }
}

}  // namespace fk
