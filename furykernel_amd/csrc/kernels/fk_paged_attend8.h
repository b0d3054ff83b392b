// fk_paged_attend8.h — attention of one new token a request over 8-bit paged
// caches (include/fkrocm_paged8.h: fk_paged_attend8).
//
// The sums, the units and how they are shared out are fk_paged_attend.h's; the
// stream of K and V rows bounds it here too, at half the bytes.  A tile stays
// in registers throughout: a wavefront loads a tile's rows in the order the
// matrix operations take them, so nothing goes through LDS or from lane to
// lane.
//
//   S = K Qᵀ    lane l (c = l mod 16, j = l div 16) holds 16-byte pieces j + 4 p
//               of the rows of keys 16 s + c: two operands of eight elements
//               each, widened to q's type (exactly).  The operand of a piece's
//               half holds d 64 p + 16 j + 8 half .. + 7, and Q's likewise.
//   Oᵀ = Vᵀ Pᵀ  S leaves lane l with keys 16 s + 4 j + i of head c, which is how
//               P goes in; so the lane loads the rows of those keys, DP / 16
//               bytes from d (DP / 16) c on: byte b of eight keys' rows is an
//               operand row of d (DP / 16) c + b.  Bytes of two keys come
//               together by a permute and are widened by pairs.
//
// Blocks are multiples of 8 positions, so 8 keys share a row of the table and
// two scales: the wavefront finds them in scalar registers.  K's scale goes
// onto the scores, V's onto the probabilities: powers of two, exact.  The
// probabilities go in as three bf16 parts, which hold all 24 bits.
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

template <uint32_t DP>
struct Attend8Tile {
  static constexpr uint32_t keys = DP == 64 ? 64 : 32;
};

// DP: the head's width in the tiles (64, 128 or 256; head_dim at most that);
// W: its wavefronts; FULL: head_dim is DP; BF16: q's type.
template <uint32_t DP, uint32_t W, bool FULL, bool BF16>
__device__ __forceinline__ void paged_attend8(const fk_paged_attend_args &a, uint64_t scales, const PagedPlan &pl) {
  using Op = PagedOperand<BF16>;
  using PV = PagedOperand<true>;
  using vec = typename Op::vec;
  constexpr uint32_t KT = Attend8Tile<DP>::keys;
  constexpr uint32_t S = KT / 16, EIGHTS = KT / 8, P = DP / 64;  // groups of 16 and 8 keys, pieces of K a lane holds
  constexpr uint32_t VW = DP / 64;                               // words of V a key a lane holds
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

  const float c2 = a.scale * 1.4426950408889634f;  // scores to log2 units
  const uint32_t c = lane % 16, j = lane / 16;
  // A lane's place in its rows, and its rows among 8 keys (past the head: a
  // piece of it again, which meets zeros of Q, or goes to no output).
  uint32_t k_in[P];
#pragma unroll
  for (uint32_t p = 0; p < P; p++) k_in[p] = c % 8 * D + min(64 * p + 16 * j, D - 16);
  const uint32_t v_in = 4 * (j % 2) * D + min(DP / 16 * c, D - DP / 16);
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
          qf[p][h] = __builtin_bit_cast(vec, w);
        }

      // The table's entries, 64 of them a lane each, from the first tile's on.
      const auto row = global_at<const uint32_t>(a.table) + (uint64_t)r * a.table_len;
      const uint32_t last_entry = __builtin_amdgcn_readfirstlane((ks.last - 1) / a.block_size);
      uint32_t entry0 = 0, entries = 0;
      // The next tile's first 8 keys: their entry and place in its block.
      uint32_t entry = 0, within = 0;
      uint64_t off[EIGHTS];                // 8 keys' rows in the pools
      float k_scale[EIGHTS], v_scale[EIGHTS];
      auto first_rows = [&] {
        entry = __builtin_amdgcn_readfirstlane(min(t0 * KT / a.block_size, last_entry));
        within = __builtin_amdgcn_readfirstlane(t0 * KT % a.block_size);
        entry0 = entry;
        entries = row[min(entry0 + lane, last_entry)];
      };
      auto rows_of_next = [&] {
#pragma unroll
        for (uint32_t e = 0; e < EIGHTS; e++) {
          if (entry > entry0 + 63) {
            entry0 = entry;
            entries = row[min(entry0 + lane, last_entry)];
          }
          const uint32_t block =
              min((uint32_t)__builtin_amdgcn_readlane((int)entries, (int)(entry - entry0)), a.blocks - 1);
          const uint64_t b = (uint64_t)block * a.kv_heads + g;
          off[e] = (b * a.block_size + within) * D;
          typedef float float2v __attribute__((ext_vector_type(2)));
          const float2v s = *(const float2v __attribute__((address_space(4))) *)(scales + 8 * b);
          k_scale[e] = s[0];
          v_scale[e] = s[1];
          // (past the last entry: the last one's again, which the masks leave out)
          within += 8;
          const bool over = within >= a.block_size;
          within = over ? 0u : within;
          entry = min(entry + over, last_entry);
        }
      };
      u32x4 kr[S][P];
      uint32_t vr[S][4][VW];
      auto load_k = [&] {
#pragma unroll
        for (uint32_t s = 0; s < S; s++) {
          const uint64_t from = a.kpool + (c < 8 ? off[2 * s] : off[2 * s + 1]);
#pragma unroll
          for (uint32_t p = 0; p < P; p++)
            kr[s][p] = __builtin_nontemporal_load(global_at<const u32x4>(from + k_in[p]));
        }
      };
      auto load_v = [&] {
        typedef uint32_t words __attribute__((ext_vector_type(VW)));
#pragma unroll
        for (uint32_t s = 0; s < S; s++) {
          const uint64_t from = a.vpool + (j < 2 ? off[2 * s] : off[2 * s + 1]) + v_in;
#pragma unroll
          for (uint32_t i = 0; i < 4; i++) {
            const words w = __builtin_nontemporal_load(global_at<const words>(from + i * D));
#pragma unroll
            for (uint32_t x = 0; x < VW; x++) vr[s][i][x] = w[x];
          }
        }
      };

      fk_float4v o[DP / 16];
#pragma unroll
      for (uint32_t d = 0; d < DP / 16; d++) o[d] = fk_float4v{0.0f, 0.0f, 0.0f, 0.0f};
      float m = -__builtin_inff(), l = 0.0f;
      if (t0 < t1) {
        first_rows();
        rows_of_next();
        load_k();
        load_v();
      }
      for (uint32_t t = t0; t < t1; t++) {
        const bool more = t + 1 < t1;
        const bool edge = t * KT < ks.first || t * KT + KT > ks.last;
        // S: register i of group s is key 16 s + 4 j + i of the tile, head c.
        fk_float4v sc[S];
#pragma unroll
        for (uint32_t s = 0; s < S; s++) {
          sc[s] = fk_float4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (uint32_t p = 0; p < P; p++)
#pragma unroll
            for (uint32_t h = 0; h < 2; h++)
              sc[s] = Op::mfma(attend8_widen<BF16>(kr[s][p][2 * h], kr[s][p][2 * h + 1]), qf[p][h], sc[s]);
        }
        float vs[S];
#pragma unroll
        for (uint32_t s = 0; s < S; s++) {
          sc[s] *= (j < 2 ? k_scale[2 * s] : k_scale[2 * s + 1]) * c2;
          vs[s] = j < 2 ? v_scale[2 * s] : v_scale[2 * s + 1];
        }
        if (more) {
          rows_of_next();
          load_k();
        }
        if (edge) {
          // (values outside the request's keys may be anything: zeros, and no scale)
#pragma unroll
          for (uint32_t s = 0; s < S; s++) {
            bool any = false;
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) {
              const uint32_t k = t * KT + 16 * s + 4 * j + i;
              const bool live = k < ks.last && k >= ks.first;
              any = any || live;
              sc[s][i] = live ? sc[s][i] : -__builtin_inff();
#pragma unroll
              for (uint32_t x = 0; x < VW; x++) vr[s][i][x] = live ? vr[s][i][x] : 0u;
            }
            vs[s] = any ? vs[s] : 0.0f;
          }
        }
        float mt = -__builtin_inff();
#pragma unroll
        for (uint32_t s = 0; s < S; s++)
#pragma unroll
          for (int i = 0; i < 4; i++) mt = __builtin_fmaxf(mt, sc[s][i]);
        const float mn = __builtin_fmaxf(m, paged_max(mt));
        const float mc = paged_ref(mn);
        if (__builtin_amdgcn_ballot_w64(mn != m)) {  // (rare behind the first tiles)
          const float alpha = __builtin_amdgcn_exp2f(m - mc);
          l *= alpha;
#pragma unroll
          for (uint32_t d = 0; d < DP / 16; d++) o[d] *= alpha;
          m = mn;
        }
        u32x4 parts[KT / 32][PV::parts];
        float sum = 0.0f;
#pragma unroll
        for (uint32_t s = 0; s < S; s++)
#pragma unroll
          for (int i = 0; i < 4; i += 2) {
            const float p0 = __builtin_amdgcn_exp2f(sc[s][i] - mc), p1 = __builtin_amdgcn_exp2f(sc[s][i + 1] - mc);
            sum += p0 + p1;
            uint32_t words[PV::parts];
            PV::cut(p0 * vs[s], p1 * vs[s], words);
#pragma unroll
            for (uint32_t x = 0; x < PV::parts; x++) parts[s / 2][x][s % 2 * 2 + i / 2] = words[x];
          }
        l += paged_sum(sum);
        // Oᵀ += Vᵀ Pᵀ: four d's words at a time.
#pragma unroll
        for (uint32_t h = 0; h < KT / 32; h++)
#pragma unroll
          for (uint32_t x = 0; x < VW; x++) {
            u32x4 f[4];
#pragma unroll
            for (uint32_t y = 0; y < 4; y++) {  // keys 2 y and 2 y + 1 of the lane's eight
              const uint32_t w0 = vr[2 * h + y / 2][y % 2 * 2][x], w1 = vr[2 * h + y / 2][y % 2 * 2 + 1][x];
              const uint32_t lo = __builtin_amdgcn_perm(w1, w0, 0x05010400), hi = __builtin_amdgcn_perm(w1, w0, 0x07030602);
              f[0][y] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false));
              f[1][y] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true));
              f[2][y] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false));
              f[3][y] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true));
            }
#pragma unroll
            for (uint32_t b = 0; b < 4; b++)
#pragma unroll
              for (uint32_t part = 0; part < PV::parts; part++)
                o[4 * x + b] = PV::mfma(__builtin_bit_cast(PV::vec, f[b]),
                                        __builtin_bit_cast(PV::vec, parts[h][part]), o[4 * x + b]);
          }
        if (more) load_v();
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
