// fk_paged_attend8.h — attention of one new token a request over 8-bit paged
// caches (include/fkrocm_paged8.h: fk_paged_attend8).
//
// The sums, the units and how they are shared out are fk_paged_attend.h's; the
// stream of K and V rows bounds it here too, at half the bytes.  A tile stays
// in registers throughout: a wavefront loads a tile's rows in the order the
// matrix operations take them, so nothing goes through LDS or from lane to
// lane, and holds two tiles, one on its way while the other is worked on.
//
//   S = K Qᵀ    lane l (c = l mod 16, j = l div 16) holds 16-byte pieces j + 4 p
//               of the rows of keys 16 s + c: two operands of eight elements
//               each, widened to q's type (exactly).  The operand of a piece's
//               half holds d 64 p + 16 j + 8 half .. + 7, and Q's likewise.
//   Oᵀ = Vᵀ Pᵀ  S leaves lane l with keys 16 s + 4 j + i of head c, which is how
//               P goes in; so the lane loads the rows of those keys, DP / 16
//               bytes from d (DP / 16) c on: byte b of eight keys' rows is an
//               operand row of d (DP / 16) c + b.  Bytes of two keys come
//               together by a permute and are widened by pairs, with the scale.
//
// Blocks are of a multiple of 8 positions, so a group of 8 keys (of 16, or the
// whole tile, where the block's size allows) lies in one block, with one scale
// for K and one for V.  Each lane keeps the place and the scales of a block of
// its own, 64 of them along the table's row; a group's come to scalar registers
// from the lane that has them.  K's scale goes onto the scores with the
// softmax's, V's into the widening: powers of two, exact.
//
// The vector operations are what a tile costs beside its bytes, so the running
// maximum is compared lane by lane and joined over the lanes only where one is
// passed, which is rare behind the first tiles, and the sum is joined at the
// end.  The probabilities go in as three bf16 parts, cut off, which hold all
// their 24 bits (by two, which leave 2^-18 of one, 41 requests of up to 700 keys
// took 7.26 µs, by three 7.50; the longest and the largest 48.6 48.8 and 125.0
// 125.6).
//
// Measured, f16 and bf16 out: one request of 131072 keys, 8 heads of 128 (268 MB)
// 43 µs, 6.2 TB/s, and the join 4.7; 64 of up to 16384 (732 MB) 120 to 124 µs, 6 TB/s,
// and 5; 41 of up to 700, 4 heads of 64, 7.5 µs, which the longest's round trips bound.
#pragma once

#include "fk_paged_attend.h"

#include "../../../include/fkrocm_paged8.h"

namespace fk {

// Eight codes of two words, widened to 16 bits.
template <bool BF16>
__device__ __forceinline__ typename PagedOperand<BF16>::vec attend8_widen(uint32_t lo, uint32_t hi) {
  u32x4 w;
  if constexpr (BF16) {
    w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false));
    w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true));
    w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false));
    w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true));
  } else {
    w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false));
    w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true));
    w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false));
    w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true));
  }
  return __builtin_bit_cast(typename PagedOperand<BF16>::vec, w);
}

constexpr uint32_t attend8_keys(uint32_t dp) { return dp == 64 ? 64 : 32; }  // a tile's

// DP: the head's width in the tiles (64, 128 or 256; head_dim at most that);
// EIGHTS: the keys of a group by eights (1, 2, or a tile's);
// FULL: head_dim is DP; BF16: q's type.
template <uint32_t DP, uint32_t EIGHTS, bool FULL, bool BF16>
__device__ __forceinline__ void paged_attend8(const fk_paged_attend_args &a, uint64_t scales, const PagedPlan &pl) {
  using Op = PagedOperand<BF16>;
  using PV = PagedOperand<true>;
  using vec = typename Op::vec;
  constexpr uint32_t PARTS = PV::parts;
  constexpr uint32_t W = FK_PAGED_WAVES;
  constexpr uint32_t KT = attend8_keys(DP);
  constexpr uint32_t S = KT / 16, P = DP / 64;  // groups of 16 keys, pieces of K that a lane holds of one
  constexpr uint32_t VW = DP / 64;              // words of V that a lane holds of a key
  constexpr uint32_t GROUPS = KT / 8 / EIGHTS;
  __shared__ __attribute__((aligned(16))) float so[W][16 * DP];
  __shared__ float sm[W][16], sl[W][16];
  const uint32_t lane = threadIdx.x & (FK_WAVE - 1);
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / FK_WAVE);
  const uint32_t n = a.requests, D = FULL ? DP : a.head_dim;
  const uint32_t per_request = a.kv_heads * pl.head_tiles;
  auto length_of = [&](uint32_t r) { return paged_length(a, r); };
  const uint32_t width = a.heads * D;
  const auto joins = global_at<u32x4>(a.workspace);
  const auto states = global_at<float>(a.workspace + gridDim.x * sizeof(u32x4));
  auto units_in = [&](uint32_t length) {
    return (paged_keys<KT>(length, a.window, pl.length).tiles + FK_PAGED_WAVES - 1) / FK_PAGED_WAVES * per_request;
  };
  PagedRun mine;
  if (!pl.whole && !paged_share<W>(a, pl, units_in, width, per_request, mine)) return;
  const uint32_t run = mine.run;
  uint32_t begin = mine.begin, end = mine.end, r = mine.request, at = mine.at, here = mine.here, length = mine.length;

  // Scores to log2 units; a negative scale's sign goes into Q, so that the
  // largest product is the largest score.
  const float c2 = __builtin_fabsf(a.scale) * 1.4426950408889634f;
  const uint32_t negate = __float_as_uint(a.scale) >> 31 ? 0x80008000u : 0u;
  const uint32_t c = lane % 16, j = lane / 16;
  // A lane's place in its rows, and its rows in a group of 8 or 16 keys (past
  // the head: a piece of it again, which meets zeros of Q, or goes to no
  // output).
  uint32_t k_in[P];
#pragma unroll
  for (uint32_t p = 0; p < P; p++) k_in[p] = (EIGHTS == 1 ? c % 8 : c) * D + min(64 * p + 16 * j, D - 16);
  const uint32_t v_in = 4 * (EIGHTS == 1 ? j % 2 : j) * D + min(DP / 16 * c, D - DP / 16);
  u32x4 last_join = {0, 0, 0, 0};

  uint32_t pid = blockIdx.x;
  do {
    if (pl.whole) {
      r = pid / per_request;
      length = length_of(r);
      here = units_in(length);
      at = 0;
      begin = pid % per_request * (here / per_request);
      end = begin + here / per_request;
      if (length == 0) {
        const uint32_t g = pid % per_request / pl.head_tiles, t = pid % pl.head_tiles * 16;
        const uint64_t where = r * a.out_stride + (uint64_t)(g * pl.group + t) * D;
        for (uint32_t e = threadIdx.x; e < min(pl.group - t, 16u) * D; e += 64 * W) {
          if (a.out_f32) global_at<float>(a.out)[where + e] = 0.0f;
          else global_at<uint16_t>(a.out)[where + e] = 0;
        }
      }
    }
    for (uint32_t pos = begin; pos < end;) {
      while (pos >= at + here) {
        at += here;
        length = length_of(++r);
        here = units_in(length);
      }
      const PagedKeys ks = paged_keys<KT>(length, a.window, pl.length);
      const uint32_t per_pair = here / per_request;
      const uint32_t pair = (pos - at) / per_pair;
      const uint32_t pair0 = at + pair * per_pair;
      const uint32_t g = pair / pl.head_tiles, h0 = g * pl.group + pair % pl.head_tiles * 16;
      const uint32_t G = min(pl.group - pair % pl.head_tiles * 16, 16u);
      const uint32_t seg1 = min(end, pair0 + per_pair);
      // the segment's tiles, shared out to the wavefronts
      const uint32_t s0 = (pos - pair0) * FK_PAGED_WAVES, s1 = min((seg1 - pair0) * FK_PAGED_WAVES, ks.tiles);
      const uint32_t t0 = __builtin_amdgcn_readfirstlane(ks.tile0 + s0 + wave * (s1 - s0) / W);
      const uint32_t t1 = __builtin_amdgcn_readfirstlane(ks.tile0 + s0 + (wave + 1) * (s1 - s0) / W);

      fk_float4v o[DP / 16];
#pragma unroll
      for (uint32_t d = 0; d < DP / 16; d++) o[d] = fk_float4v{0.0f, 0.0f, 0.0f, 0.0f};
      float m = -__builtin_inff(), l = 0.0f;
      if (t0 < t1) {
        // The table's blocks, a lane each, 64 from the first tile's on: their
        // rows' place in the pools and their scales.
        typedef float float2v __attribute__((ext_vector_type(2)));
        const auto row = global_at<const uint32_t>(a.table) + (uint64_t)r * a.table_len;
        const uint32_t last_entry = __builtin_amdgcn_readfirstlane((ks.last - 1) / a.block_size);
        // The next group: its entry and its place in the block.
        uint32_t entry = __builtin_amdgcn_readfirstlane(min(t0 * KT / a.block_size, last_entry));
        uint32_t within = __builtin_amdgcn_readfirstlane(t0 * KT % a.block_size);
        uint32_t entry0 = entry, off_lo, off_hi;
        float2v scale2;
        auto entries = [&] {
          const uint32_t block = min(row[min(entry0 + lane, last_entry)], a.blocks - 1);
          const uint64_t b = (uint64_t)block * a.kv_heads + g;
          const uint64_t off = b * a.block_size * D;
          off_lo = (uint32_t)off, off_hi = (uint32_t)(off >> 32);
          scale2 = *global_at<const float2v>(scales + 8 * b);
        };
        entries();
        // Q (B of S = K Qᵀ): lane l holds head c (past the group: its last), zeros
        // past the head.
        vec qf[P][2];
        const uint64_t q_row = paged_query(a, r);
#pragma unroll
        for (uint32_t p = 0; p < P; p++)
#pragma unroll
          for (uint32_t h = 0; h < 2; h++) {
            const uint32_t d = 64 * p + 16 * j + 8 * h;
            u32x4 w = {0, 0, 0, 0};
            if (FULL || d < D)
              w = *global_at<const u32x4>(a.q + 2 * (q_row * a.q_stride + (uint64_t)(h0 + min(c, G - 1)) * D + d));
#pragma unroll
            for (int x = 0; x < 4; x++) w[x] ^= negate;
            qf[p][h] = __builtin_bit_cast(vec, w);
          }

        struct Tile {
          u32x4 k[S][P];
          uint32_t v[S][4][VW];
          uint32_t from[GROUPS];  // the lane that has the group's block
        };
        Tile x, y;
        float ks_x[GROUPS], vs_x[GROUPS], ks_y[GROUPS], vs_y[GROUPS];
        // A tile's loads, in the order of the tiles (past the last: the last
        // table entry's again, which goes nowhere).
        auto load = [&](Tile &tile) __attribute__((always_inline)) {
          uint64_t off[GROUPS];
          if (entry + GROUPS - 1 > entry0 + 63) {
            entry0 = entry;
            entries();
            asm volatile("" : "+v"(off_lo), "+v"(off_hi), "+v"(scale2));  // landed before other loads go out
          }
#pragma unroll
          for (uint32_t e = 0; e < GROUPS; e++) {
            tile.from[e] = entry - entry0;
            off[e] = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)off_hi, (int)tile.from[e]) << 32 |
                      (uint32_t)__builtin_amdgcn_readlane((int)off_lo, (int)tile.from[e])) +
                     within * D;
            within += 8 * EIGHTS;
            const bool over = within >= a.block_size;
            within = over ? 0u : within;
            entry = min(entry + over, last_entry);
          }
          // A group's rows: a scalar base that the compiler leaves one.
          auto base = [&](uint64_t pool, uint32_t e, uint32_t rows) {
            uint64_t at = pool + off[e] + rows * D;
            asm volatile("" : "+s"(at));
            return global_at<const char>(at);
          };
          auto rows_at = [&](uint64_t pool, uint32_t s, bool first) {
            if constexpr (EIGHTS == 1) return global_at<const char>(pool) + (first ? off[2 * s] : off[2 * s + 1]);
            else return base(pool, EIGHTS == 2 ? s : 0u, EIGHTS == 2 ? 0u : 16 * s);
          };
          // (made 32-bit offsets again here, which go with a scalar base)
          uint32_t k_at[P], v_at = v_in;
          asm volatile("" : "+v"(v_at));
#pragma unroll
          for (uint32_t p = 0; p < P; p++) {
            k_at[p] = k_in[p];
            asm volatile("" : "+v"(k_at[p]));
          }
#pragma unroll
          for (uint32_t s = 0; s < S; s++) {
            const auto from = rows_at(a.kpool, s, c < 8);
#pragma unroll
            for (uint32_t p = 0; p < P; p++)  // (past the caches where one load takes whole lines)
              tile.k[s][p] = load_from<P == 1, u32x4>((global_ptr<const u32x4>)(from + k_at[p]));
          }
          typedef uint32_t words __attribute__((ext_vector_type(VW)));
#pragma unroll
          for (uint32_t s = 0; s < S; s++) {
            const auto from = rows_at(a.vpool, s, j < 2);
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) {
              const words w = __builtin_nontemporal_load((global_ptr<const words>)(from + v_at + i * D));
#pragma unroll
              for (uint32_t z = 0; z < VW; z++) tile.v[s][i][z] = w[z];
            }
          }
          __builtin_amdgcn_sched_barrier(0);  // (else some of them go out where they are waited for)
        };
        // The groups' scales (of the lanes' blocks as they are when the tile is
        // loaded).
        auto scales_of = [&](const Tile &tile, float (&k)[GROUPS], float (&v)[GROUPS]) __attribute__((always_inline)) {
#pragma unroll
          for (uint32_t e = 0; e < GROUPS; e++) {
            k[e] = readlane_f(scale2[0], (int)tile.from[e]);
            v[e] = readlane_f(scale2[1], (int)tile.from[e]);
          }
        };
        auto of_lane = [&](const float (&x)[GROUPS], uint32_t s) {
          if constexpr (EIGHTS == 1) return j < 2 ? x[2 * s] : x[2 * s + 1];
          else if constexpr (EIGHTS == 2) return x[s];
          else return x[0];
        };
        auto work = [&](Tile &tile, const float (&k_scale)[GROUPS], const float (&v_scale)[GROUPS],
                        uint32_t t) __attribute__((always_inline)) {
          // S: register i of group s is key 16 s + 4 j + i of the tile, head c.
          fk_float4v sc[S];
          float kf[S], vf[S];
#pragma unroll
          for (uint32_t s = 0; s < S; s++) {
            sc[s] = fk_float4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (uint32_t p = 0; p < P; p++)
#pragma unroll
              for (uint32_t h = 0; h < 2; h++)
                sc[s] = Op::mfma(attend8_widen<BF16>(tile.k[s][p][2 * h], tile.k[s][p][2 * h + 1]), qf[p][h], sc[s]);
            kf[s] = of_lane(k_scale, s) * c2;
            vf[s] = of_lane(v_scale, s);
          }
          if (t * KT < ks.first || t * KT + KT > ks.last) {
            // (what lies outside the request's keys may be anything: no score,
            // zeros of V, and for a group that is all outside a scale of 1)
#pragma unroll
            for (uint32_t s = 0; s < S; s++) {
              bool any = false;
#pragma unroll
              for (uint32_t i = 0; i < 4; i++) {
                const uint32_t k = t * KT + 16 * s + 4 * j + i;
                const bool live = k < ks.last && k >= ks.first;
                any = any || live;
                sc[s][i] = live ? sc[s][i] * kf[s] : -__builtin_inff();
#pragma unroll
                for (uint32_t z = 0; z < VW; z++) tile.v[s][i][z] = live ? tile.v[s][i][z] : 0u;
              }
              kf[s] = 1.0f;
              vf[s] = any ? vf[s] : 1.0f;
            }
          }
          float mt = -__builtin_inff();
#pragma unroll
          for (uint32_t s = 0; s < S; s++)
            mt = __builtin_fmaxf(mt, __builtin_fmaxf(__builtin_fmaxf(sc[s][0], sc[s][1]),
                                                     __builtin_fmaxf(sc[s][2], sc[s][3])) * kf[s]);
          if (__builtin_amdgcn_ballot_w64(mt > m)) {
            const float mn = __builtin_fmaxf(m, paged_max(mt));
            const float alpha = __builtin_amdgcn_exp2f(m - paged_ref(mn));
            l *= alpha;
#pragma unroll
            for (uint32_t d = 0; d < DP / 16; d++) o[d] *= alpha;
            m = mn;
          }
          const float mc = paged_ref(m);
          u32x4 parts[KT / 32][PARTS];
#pragma unroll
          for (uint32_t s = 0; s < S; s++)
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
              const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[s][i], kf[s], -mc));
              const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[s][i + 1], kf[s], -mc));
              l += p0 + p1;
              uint32_t words[PARTS];
              PV::cut(p0, p1, words);
#pragma unroll
              for (uint32_t z = 0; z < PARTS; z++) parts[s / 2][z][s % 2 * 2 + i / 2] = words[z];
            }
          // Oᵀ += Vᵀ Pᵀ: four d's words at a time.
#pragma unroll
          for (uint32_t h = 0; h < KT / 32; h++)
#pragma unroll
            for (uint32_t z = 0; z < VW; z++) {
              u32x4 f[4];
#pragma unroll
              for (uint32_t q = 0; q < 4; q++) {  // keys 2 q and 2 q + 1 of the lane's eight
                const uint32_t s = 2 * h + q / 2;
                const uint32_t w0 = tile.v[s][q % 2 * 2][z], w1 = tile.v[s][q % 2 * 2 + 1][z];
                const uint32_t lo = __builtin_amdgcn_perm(w1, w0, 0x05010400);
                const uint32_t hi = __builtin_amdgcn_perm(w1, w0, 0x07030602);
                f[0][q] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, vf[s], false));
                f[1][q] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, vf[s], true));
                f[2][q] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, vf[s], false));
                f[3][q] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, vf[s], true));
              }
#pragma unroll
              for (uint32_t b = 0; b < 4; b++)
#pragma unroll
                for (uint32_t part = 0; part < PARTS; part++)
                  o[4 * z + b] = PV::mfma(__builtin_bit_cast(PV::vec, f[b]),
                                          __builtin_bit_cast(PV::vec, parts[h][part]), o[4 * z + b]);
            }
        };
        load(x);
        load(y);
        scales_of(x, ks_x, vs_x);
        scales_of(y, ks_y, vs_y);
        // (one exit, so that the compiler's waits know what is in flight)
        uint32_t t = t0;
        for (; t + 2 < t1; t += 2) {
          work(x, ks_x, vs_x, t);
          load(x);
          scales_of(x, ks_x, vs_x);
          work(y, ks_y, vs_y, t + 1);
          load(y);
          scales_of(y, ks_y, vs_y);
        }
        work(x, ks_x, vs_x, t);
        if (t + 1 < t1) work(y, ks_y, vs_y, t + 1);
        l = paged_sum(l);
      }

      // The wavefronts' states meet: register i of o[b] is d (DP / 16) (4 j + i)
      // + b of head c.
      if (c < G) {
#pragma unroll
        for (uint32_t i = 0; i < 4; i++)
#pragma unroll
          for (uint32_t b = 0; b < DP / 16; b++) so[wave][c * DP + DP / 16 * (4 * j + i) + b] = o[b][i];
        if (lane < 16) {
          sm[wave][lane] = m;
          sl[wave][lane] = l;
        }
      }
      __syncthreads();
      const bool whole = pos == pair0 && seg1 == pair0 + per_pair;
      const uint32_t side = pair0 < begin ? 0u : 1u;
      auto state_of = [&](uint32_t w) { return (const float *)so[w]; };
      paged_meet<DP, W, BF16>(a, state_of, sm, sl, G, D, whole, r * a.out_stride + (uint64_t)h0 * D,
                              states + paged_state(blockIdx.x, side, pl.rows, D), pl.rows);
      if (!pl.whole && pos == pair0) {
        // the pair starts here: it ends here too, or in the threadgroup of its
        // last unit
        u32x4 join = {0, 0, 0, 0};
        if (!whole) join = paged_join(blockIdx.x, (pair0 + per_pair - 1) / run, r, h0, G);
        if (pl.by_pair && threadIdx.x == 0) joins[r * per_request + pair] = join;
        last_join = join;
      }
      __syncthreads();  // before the next pair's states
      pos = seg1;
    }
    pid += gridDim.x;
  } while (pl.whole && pid < n * per_request);
  if (!pl.whole && !pl.by_pair && threadIdx.x == 0) joins[blockIdx.x] = last_join;
}

}  // namespace fk
