// fk_paged_attend.h — attention of one new token a request over paged caches
// (include/fkrocm_serve.h: fk_paged_attend).
//
// out = softmax(scale q Kᵀ) V, one pass over the keys with a running maximum m,
// sum l and weighted values o: a tile's scores s give m' = max(m, max s),
// o' = o e^(m - m') + e^(s - m') V, l' likewise, and two such states of one
// row join the same way.  The K and V rows' stream bounds it: 4 bytes an
// element pair against 4 flops a query head.
//
// How the work is split.  A pair is a request, a kv head and up to 16 of its
// query heads (the columns of the matrix operations); its keys are cut into
// units of 4 tiles.  The units of all pairs, in order, are shared out evenly
// over the launch's threadgroups (two a CU), each a run of units: a long
// request goes to as many threadgroups as its share of the batch's keys, a
// run of short ones to one, whatever the mix, and no length is needed on the
// host.  Every threadgroup finds its run by a prefix sum of the lengths of its
// own.  A run's pair that ends in another threadgroup leaves its state in the
// workspace, at most two a threadgroup, and paged_attend_join adds them in
// order, so the same lengths give the same bits.  Where a table holds few units
// a request, pairs go whole to the threadgroups instead: no prefix sum, no
// states, no join (the launch's rule has both sides measured).
//
// In a threadgroup each of the 4 wavefronts (8 where few pairs go whole) takes
// its share of a pair's tiles with a state of its own; nothing is shared until
// they meet at the pair's end.  A tile's K and V rows (KT keys) go straight
// into the wavefront's LDS; the next tile's K is loaded as soon as the scores
// are made and its V after the values, so loads are in flight all the time
// without a second buffer.
// That needs reads of one beside loads into the other, which the compiler
// would not let pass each other: they are written out (a tile took 2.4 µs where
// latency alone counts, now 2.0).
// Measured: one request of 131072 keys, 32 heads over 8 of 128, 82 µs (537 MB,
// 6.5 TB/s) and 4.6 for the join; 64 requests of up to 16384, 228 and 5.9
// (1.46 GB, 6.4 TB/s).  A tile's block lookups all go out before the first is
// waited for, and a run's first table entries beside Q (a short table beside
// the lengths): 41 requests of 512 keys of 64 13.4 µs, so 11.8.
// Pages may end anywhere in a tile: each lane finds its key's block, from 64
// table entries that the wavefront holds a lane each.
//
// Matrix operations (v_mfma_f32_16x16x32): S = K Qᵀ, then Oᵀ = Vᵀ Pᵀ with the
// probabilities in the registers that made them, V transposed by the LDS's
// transposing reads.  The probabilities go in as 16-bit parts, p cut off and
// what that leaves: three in bf16, which hold all 24 bits of a binary32 (two
// hold 16, and took as long: 64 requests of up to 16384 keys 232 µs), two in
// f16, which hold 21, as many as a binary32 exponential keeps of scores of
// about 10 (three: 41 requests of up to 700 keys 9.55 µs, so 9.25).  In f16 a
// reference 15 below the running maximum keeps the smallest step at 2^-39 of the
// largest probability.
//
// A part of 0 times a value of infinity is no number, where the probability
// itself would give infinity.  A wavefront whose tiles gave such a sum makes
// them again with the parts that are 0 at the type's smallest step, those of
// keys of a score of -infinity excepted: infinite values then give infinity,
// whatever their keys' weights, and rows whose sums are finite never come here.
#pragma once

#include "fk_address.h"
#include "fk_common.h"
#include "fk_mfma.h"

#include "../../../include/fkrocm_serve.h"

#define FK_PAGED_WAVES 4
#define FK_PAGED_LDS __attribute__((address_space(3)))
// s_waitcnt vmcnt(n), the other counters untouched (vmcnt's low four bits at
// 3:0, its high two at 15:14).
#define FK_PAGED_VMCNT(N) (((N) & 15) | (((N) >> 4) << 14) | (0x7 << 4) | (0xf << 8))

typedef __bf16 fk_paged_bf16x8 __attribute__((ext_vector_type(8)));

namespace fk {

// What the kernels take beside the call's arguments.
struct PagedPlan {
  uint32_t group;      // query heads a kv head
  uint32_t head_tiles; // groups of up to 16 of them
  uint32_t rows;       // query heads a pair's state holds: min(group, 16)
  uint32_t length;     // positions a table row covers
  uint32_t by_pair;    // the joins' entries are the pairs'
  uint32_t whole;      // each pair to one threadgroup: no states, no joins
};

// A pair that ends in another threadgroup than it starts in, in the workspace
// (an entry for each pair, or for the last pair that each threadgroup starts,
// whichever are fewer): its first and last threadgroup, its request, its first
// query head and how many it has.  A first word of 0: there is no such pair.
__device__ __forceinline__ u32x4 paged_join(uint32_t first, uint32_t last, uint32_t request, uint32_t head,
                                            uint32_t rows) {
  return u32x4{first << 16 | last, request, head << 4 | (rows - 1), 0};
}

// A pair's state in the workspace: `rows` rows of head_dim values, then the
// maximum and the sum of each.
__device__ __forceinline__ uint64_t paged_state(uint32_t group, uint32_t side, uint32_t rows, uint32_t d) {
  return ((uint64_t)group * 2 + side) * rows * (d + 2);
}

// The keys of a request that its token sees, in tiles of KT aligned to KT.
struct PagedKeys {
  uint32_t first, last;   // positions first .. last - 1
  uint32_t tile0, tiles;
};

template <uint32_t KT>
__device__ __forceinline__ PagedKeys paged_keys(uint32_t length, uint32_t window, uint32_t most) {
  PagedKeys k;
  k.last = min(length, most);
  k.first = window && k.last > window ? k.last - window : 0u;
  k.tile0 = k.first / KT;
  k.tiles = (k.last + KT - 1) / KT - k.tile0;
  return k;
}

// A request's positions, 0 if it has no query, and its query's row.
__device__ __forceinline__ uint32_t paged_length(const fk_paged_attend_args &a, uint32_t r) {
  const uint32_t length = global_at<const uint32_t>(a.lengths)[r];
  if (!a.starts) return length;
  const auto s = global_at<const uint32_t>(a.starts) + r;
  return s[1] > s[0] && s[1] <= a.q_rows ? length : 0u;
}
__device__ __forceinline__ uint64_t paged_query(const fk_paged_attend_args &a, uint32_t r) {
  return a.starts ? global_at<const uint32_t>(a.starts)[r + 1] - 1u : r;
}

// Over lanes l, l ^ 16, l ^ 32 and l ^ 48.
__device__ __forceinline__ float paged_max(float x) {
  auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __builtin_fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
  s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __builtin_fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float paged_sum(float x) {
  auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(s[0]) + __uint_as_float(s[1]);
  s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

// Reads of LDS that loads into it may still be landing on elsewhere: the
// compiler, which cannot tell the wavefront's K rows from its V rows, would
// wait for every load in flight before a read of its own.  Their data are
// there when the block ends.
#define FK_PAGED_READ8(NAME, OP, T)                                                                       \
  template <uint32_t STEP>                                                                                \
  __device__ __forceinline__ void NAME(const uint32_t (&at)[4], T (&x)[8]) {                              \
    asm volatile(OP " %0, %8\n\t" OP " %1, %9\n\t" OP " %2, %10\n\t" OP " %3, %11\n\t"                 \
                 OP " %4, %8 offset:%12\n\t" OP " %5, %9 offset:%12\n\t"                                 \
                 OP " %6, %10 offset:%12\n\t" OP " %7, %11 offset:%12\n\ts_waitcnt lgkmcnt(0)"           \
                 : "=&v"(x[0]), "=&v"(x[1]), "=&v"(x[2]), "=&v"(x[3]), "=&v"(x[4]), "=&v"(x[5]),          \
                   "=&v"(x[6]), "=&v"(x[7])                                                               \
                 : "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "n"(STEP)                              \
                 : "memory");                                                                             \
  }
FK_PAGED_READ8(paged_read8, "ds_read_b128", u32x4)
FK_PAGED_READ8(paged_read8_tr, "ds_read_b64_tr_b16", u32x2)

// A reference to take exponentials from: 0 in place of that of a row that has
// seen no score.
__device__ __forceinline__ float paged_ref(float m) { return m == -__builtin_inff() ? 0.0f : m; }

// A state's value times its factor, onto another: one that infinite values made
// stays so where the factor is too small for a binary32.
__device__ __forceinline__ float paged_plus(float sum, float o, float f) {
  return sum + (__builtin_isinf(o) ? o : o * f);
}

// Eight 16-bit operands of a matrix operation.
template <bool BF16>
struct PagedOperand;
template <>
struct PagedOperand<false> {
  typedef _Float16 elem;
  typedef fk_half8 vec;
  static constexpr float shift = 15.0f;  // the reference below the running maximum: probabilities to 2^15
  static constexpr uint32_t tiny = 1;    // 2^-24
  static __device__ __forceinline__ fk_float4v mfma(vec a, vec b, fk_float4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  // The parts of two probabilities, a word each: cut off, and what that leaves
  // to the nearest.
  static constexpr uint32_t parts = 2;
  static __device__ __forceinline__ void cut(float p0, float p1, uint32_t (&to)[parts]) {
    typedef _Float16 half2 __attribute__((ext_vector_type(2)));
    const auto h = __builtin_amdgcn_cvt_pkrtz(p0, p1);
    to[0] = __builtin_bit_cast(uint32_t, h);
    to[1] = __builtin_bit_cast(uint32_t, half2{(_Float16)(p0 - (float)h[0]), (_Float16)(p1 - (float)h[1])});
  }
};
template <>
struct PagedOperand<true> {
  typedef __bf16 elem;
  typedef fk_paged_bf16x8 vec;
  static constexpr float shift = 0.0f;       // (values may be as large as a binary32's)
  static constexpr uint32_t tiny = 27 << 7;  // 2^-100
  static __device__ __forceinline__ fk_float4v mfma(vec a, vec b, fk_float4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  // (each part eight bits: the third is all that the first two leave)
  static constexpr uint32_t parts = 3;
  static __device__ __forceinline__ void cut(float p0, float p1, uint32_t (&to)[parts]) {
#pragma unroll
    for (uint32_t x = 0; x < parts; x++) {
      const uint32_t u0 = __float_as_uint(p0), u1 = __float_as_uint(p1);
      to[x] = __builtin_amdgcn_perm(u1, u0, 0x07060302);  // the upper halves
      p0 -= __uint_as_float(u0 & 0xFFFF0000u);
      p1 -= __uint_as_float(u1 & 0xFFFF0000u);
    }
  }
};

template <bool BF16>
__device__ __forceinline__ uint16_t paged_round(float x) {
  return __builtin_bit_cast(uint16_t, (typename PagedOperand<BF16>::elem)x);
}

// DP: the head's width in the tiles (64, 128 or 256; head_dim at most that);
// W: its wavefronts, 4, or 8 of whole pairs; FULL: head_dim is DP.
template <uint32_t DP, uint32_t W, bool FULL, bool BF16>
__device__ __forceinline__ void paged_attend(const fk_paged_attend_args &a, const PagedPlan &pl) {
  using Op = PagedOperand<BF16>;
  using vec = typename Op::vec;
  constexpr uint32_t KT = DP == 64 ? 64 : 32;    // keys a tile: 8 KB of K at 64 and 128, 16 KB at 256
  constexpr uint32_t UNITS = DP / 8;             // 16-byte pieces of a row
  constexpr uint32_t KPL = 64 / UNITS;           // rows a load of the wavefront covers
  constexpr uint32_t LOADS = KT / KPL;           // loads a tile's K or V takes
  constexpr uint32_t THREADS = 64 * W;
  __shared__ __attribute__((aligned(16))) uint16_t kv[W][2][KT * DP];
  __shared__ float sm[W][16], sl[W][16];
  __shared__ uint32_t wave_units[W];
  __shared__ u32x4 found;
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
  auto units_of = [&](uint32_t r) { return units_in(length_of(r)); };
  // (rows of pieces past head_dim are zeros in K, which no load writes)
  if (!FULL)
    for (uint32_t i = threadIdx.x; i < W * KT * UNITS; i += THREADS)
      reinterpret_cast<uint4 *>(kv[i / (KT * UNITS)][0])[i % (KT * UNITS)] = make_uint4(0, 0, 0, 0);
  // The run: units begin .. end - 1 of `total`, of which request r's `here`
  // start at `at`.
  uint32_t run = 1, total = 0, begin = 0, end = 0, r = 0, at = 0, here = 0, length = 0;
  if (pl.whole) {
    __syncthreads();
  } else {
    // The units of each thread's requests, and before them.
    const uint32_t chunk = (n + THREADS - 1) / THREADS;
    const uint32_t r0 = min(threadIdx.x * chunk, n), r1 = min(r0 + chunk, n);
    uint32_t mine = 0;
    for (uint32_t r = r0; r < r1; r++) mine += units_of(r);
    uint32_t upto = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const uint32_t o = __shfl_up(upto, d, 64);
      if (lane >= (uint32_t)d) upto += o;
    }
    if (lane == 63) wave_units[wave] = upto;
    __syncthreads();
    uint32_t before = upto - mine;
#pragma unroll
    for (uint32_t w = 0; w < W; w++) {
      before += w < wave ? wave_units[w] : 0u;
      total += wave_units[w];
    }
    // This threadgroup's run of units, its request found by the thread that
    // holds it.
    run = max((total + gridDim.x - 1) / gridDim.x, 1u);
    begin = min(blockIdx.x * run, total);
    end = min(begin + run, total);
    if (before <= begin && begin < before + mine) {
      uint32_t r = r0, at = before, here = units_of(r);
      while (at + here <= begin) {
        at += here;
        here = units_of(++r);
      }
      found = u32x4{r, at, here, length_of(r)};
    }
    __syncthreads();

    // Requests that see nothing: rows of zeros.
    for (uint32_t r = blockIdx.x; r < n; r += gridDim.x)
      if (length_of(r) == 0) {
        for (uint32_t e = threadIdx.x; e < width; e += THREADS) {
          if (a.out_f32) global_at<float>(a.out)[r * a.out_stride + e] = 0.0f;
          else global_at<uint16_t>(a.out)[r * a.out_stride + e] = 0;
        }
        if (pl.by_pair)
          for (uint32_t p = threadIdx.x; p < per_request; p += THREADS)
            joins[r * per_request + p] = u32x4{0, 0, 0, 0};
      }
    if (begin == end) {
      if (!pl.by_pair && threadIdx.x == 0) joins[blockIdx.x] = u32x4{0, 0, 0, 0};
      return;
    }
    r = __builtin_amdgcn_readfirstlane(found[0]);
    at = __builtin_amdgcn_readfirstlane(found[1]);
    here = __builtin_amdgcn_readfirstlane(found[2]);
    length = __builtin_amdgcn_readfirstlane(found[3]);
  }

  uint16_t *const kbuf = kv[wave][0], *const vbuf = kv[wave][1];
  const auto kpool = global_at<const char>(a.kpool);
  const auto vpool = global_at<const char>(a.vpool);
  const float c = a.scale * 1.4426950408889634f;  // scores to log2 units
  const uint32_t piece = lane % UNITS, krow = lane / UNITS;
  // What a lane reads of its wavefront's rows: places and turns that a step of
  // 16 rows leaves as they are.
  const uint32_t tk = 4 * (lane / 16) + lane % 16 / 4, td = 4 * (lane & 3);
  const uint32_t k_turn = DP == 64 ? (lane >> 1) & 7u : lane & 15u, v_turn = DP == 64 ? (tk >> 1) & 3u : tk & 7u;
  const uint32_t k_lds = (uint32_t)(uintptr_t)(FK_PAGED_LDS uint16_t *)kbuf;
  const uint32_t v_lds = (uint32_t)(uintptr_t)(FK_PAGED_LDS uint16_t *)vbuf;
  u32x4 last_join = {0, 0, 0, 0};

  uint32_t pid = blockIdx.x, entries = 0;
  do {
    if (pl.whole) {
      r = pid / per_request;
      // a whole table of no more than a wavefront's lanes, beside the length
      if (a.table_len <= FK_WAVE)
        entries = global_at<const uint32_t>(a.table)[(uint64_t)r * a.table_len + min(lane, a.table_len - 1)];
      length = length_of(r);
      here = units_in(length);
      at = 0;
      begin = pid % per_request * (here / per_request);
      end = begin + here / per_request;
      if (length == 0) {
        const uint32_t g = pid % per_request / pl.head_tiles, t = pid % pl.head_tiles * 16;
        const uint64_t where = r * a.out_stride + (uint64_t)(g * pl.group + t) * D;
        for (uint32_t e = threadIdx.x; e < min(pl.group - t, 16u) * D; e += THREADS) {
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
      const uint32_t t0 = ks.tile0 + s0 + wave * (s1 - s0) / W;
      const uint32_t t1 = ks.tile0 + s0 + (wave + 1) * (s1 - s0) / W;

      // Q (B of S = K Qᵀ): lane l holds head l mod 16 (past the group: its
      // last), d 32 h + 8 (l div 16) .. + 7, zeros past the head.
      vec qf[DP / 32];
      const uint64_t q_row = paged_query(a, r);
#pragma unroll
      for (uint32_t h = 0; h < DP / 32; h++) {
        const uint32_t d = 32 * h + 8 * (lane / 16);
        u32x4 w = {0, 0, 0, 0};
        if (FULL || d < D)
          w = *global_at<const u32x4>(a.q + 2 * (q_row * a.q_stride + (uint64_t)(h0 + min(lane % 16, G - 1)) * D + d));
        qf[h] = __builtin_bit_cast(vec, w);
      }

      const auto row = global_at<const uint32_t>(a.table) + (uint64_t)r * a.table_len;
      const uint32_t last_entry = (ks.last - 1) / a.block_size;
      // The table entries entry0 + lane, from the first tile's on unless they are
      // there already, landed with Q: no tile without a load of them waits for
      // one.
      uint32_t entry0 = 0;
      auto first_entries = [&] {
        if (!pl.whole || a.table_len > FK_WAVE) {
          entry0 = min(max(t0 * KT, ks.first) / a.block_size, last_entry);
          entries = row[min(entry0 + lane, last_entry)];
        }
      };
      first_entries();
      __builtin_amdgcn_s_waitcnt(FK_PAGED_VMCNT(0));
      asm volatile("" : "+v"(entries));
#pragma unroll
      for (uint32_t h = 0; h < DP / 32; h++) asm volatile("" : "+v"(qf[h]));
      entries = min(entries, a.blocks - 1);
      uint64_t off[LOADS];                // the tile's rows in the pools, in bytes
      // K's piece u at place u ^ (key's) of its row, V's 32-byte pairs of pieces
      // likewise, so that the reads below meet different banks.
      auto rows_of = [&](uint32_t tile) {
        if ((min(tile * KT + KT, ks.last) - 1) / a.block_size > entry0 + 63) {
          entry0 = max(tile * KT, ks.first) / a.block_size;
          entries = min(row[min(entry0 + lane, last_entry)], a.blocks - 1);
          __builtin_amdgcn_s_waitcnt(FK_PAGED_VMCNT(0));
          asm volatile("" : "+v"(entries));
        }
        uint32_t block[LOADS], within[LOADS];
#pragma unroll
        for (uint32_t q = 0; q < LOADS; q++) {
          // keys outside the request's own are its own all the same (masked)
          const uint32_t key = min(max(tile * KT + q * KPL + krow, ks.first), ks.last - 1);
          const uint32_t entry = key / a.block_size;
          within[q] = key - entry * a.block_size;
          block[q] = __builtin_amdgcn_ds_bpermute((entry - entry0) * 4, entries);
        }
        __builtin_amdgcn_sched_barrier(0);  // all asked for before the first is waited for
#pragma unroll
        for (uint32_t q = 0; q < LOADS; q++)
          off[q] = (((uint64_t)block[q] * a.kv_heads + g) * a.block_size + within[q]) * (2 * D);
      };
      auto load = [&](global_ptr<const char> pool, uint16_t *buf, bool keys) {
#pragma unroll
        for (uint32_t q = 0; q < LOADS; q++) {
          const uint32_t key = q * KPL + krow;
          const uint32_t turn = keys ? (DP == 64 ? (key >> 1) & 7u : key & 15u)
                                     : (DP == 64 ? ((key >> 1) & 3u) << 1 : (key & 7u) << 1);
          const uint32_t u = piece ^ turn;
          if (FULL || u * 8 < D)
            __builtin_amdgcn_global_load_lds((global_ptr<const void>)(pool + off[q] + u * 16),
                                             (FK_PAGED_LDS void *)(buf + q * 512), 16, 0, 2);
        }
      };

      fk_float4v o[DP / 16];
      float m, l;
      // The wavefront's tiles; whether a sum of a row that has weights is not a
      // number (a second making of its own: a branch in each tile and 30 registers
      // more took 41 requests of up to 700 keys 9.6 µs, so 9.25; 8.95 without).
      auto make = [&](auto once_more) __attribute__((always_inline)) {
        constexpr bool again = decltype(once_more)::value;
#pragma unroll
        for (uint32_t d = 0; d < DP / 16; d++) o[d] = fk_float4v{0.0f, 0.0f, 0.0f, 0.0f};
        m = -__builtin_inff(), l = 0.0f;
        if (t0 < t1) {
          rows_of(t0);
          load(kpool, kbuf, true);
          load(vpool, vbuf, false);
        }
        for (uint32_t t = t0; t < t1; t++) {
          const bool more = t + 1 < t1;
          __builtin_amdgcn_s_waitcnt(FK_PAGED_VMCNT(LOADS));  // K landed, V's loads in flight
          asm volatile("" ::: "memory");
          // S: groups of 16 keys; register i of group s is key 16 s + 4 (l div 16)
          // + i of the tile, head l mod 16.
          fk_float4v sc[KT / 16];
#pragma unroll
          for (uint32_t s = 0; s < KT / 16; s++) sc[s] = fk_float4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (uint32_t c = 0; c < KT * DP / 4096; c++) {
            // of 4 addresses and STEP rows further: at 64, pieces h of groups s and
            // s + 1 (and s + 2); else four pieces of a group (and the next)
            constexpr uint32_t HS = DP == 64 ? 2 : 4, ROWS = DP == 64 ? 32 : 16;
            uint32_t at[4];
            u32x4 w[8];
#pragma unroll
            for (uint32_t i = 0; i < 4; i++)
              at[i] = k_lds + (lane % 16 + i / HS * 16) * (2 * DP) +
                      ((4 * (c * HS + i % HS) + lane / 16) ^ k_turn) * 16;
            paged_read8<ROWS * 2 * DP>(at, w);
#pragma unroll
            for (uint32_t i = 0; i < 8; i++) {
              const uint32_t s = i % 4 / HS + i / 4 * (ROWS / 16), h = c * HS + i % HS;
              sc[s] = Op::mfma(__builtin_bit_cast(vec, w[i]), qf[h], sc[s]);
            }
          }
          // The reads are done before the next tile's loads land on them.
#pragma unroll
          for (uint32_t s = 0; s < KT / 16; s++) asm volatile("" : "+v"(sc[s])::"memory");
          if (more) {
            rows_of(t + 1);
            load(kpool, kbuf, true);
          }
          float mt = -__builtin_inff();
#pragma unroll
          for (uint32_t s = 0; s < KT / 16; s++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
              const uint32_t k = t * KT + 16 * s + 4 * (lane / 16) + i;
              sc[s][i] = k < ks.last && k >= ks.first ? sc[s][i] * c : -__builtin_inff();
              mt = __builtin_fmaxf(mt, sc[s][i]);
            }
          const float mn = __builtin_fmaxf(m, paged_max(mt) - Op::shift);
          const float mc = paged_ref(mn);
          float alpha = __builtin_amdgcn_exp2f(m - mc);
          if (again) alpha = __builtin_fmaxf(alpha, 0x1p-126f);
          m = mn;
          u32x4 parts[KT / 32][Op::parts];
          float sum = 0.0f;
#pragma unroll
          for (uint32_t s = 0; s < KT / 16; s++)
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
              const float p0 = __builtin_amdgcn_exp2f(sc[s][i] - mc), p1 = __builtin_amdgcn_exp2f(sc[s][i + 1] - mc);
              sum += p0 + p1;
              uint32_t words[Op::parts];
              Op::cut(p0, p1, words);
#pragma unroll
              for (uint32_t x = 0; x < Op::parts; x++) parts[s / 2][x][s % 2 * 2 + i / 2] = words[x];
            }
          if (again) {
#pragma unroll
            for (uint32_t h = 0; h < KT / 32; h++)
#pragma unroll
              for (uint32_t i = 0; i < 8; i++)
#pragma unroll
                for (uint32_t x = 0; x < Op::parts; x++) {
                  const uint32_t at = 16 * (i % 2);
                  if (sc[2 * h + i / 4][i % 4] > -__builtin_inff() && (parts[h][x][i / 2] >> at & 0xFFFFu) == 0)
                    parts[h][x][i / 2] |= Op::tiny << at;
                }
          }
          l = l * alpha + paged_sum(sum);
#pragma unroll
          for (uint32_t d = 0; d < DP / 16; d++) o[d] *= alpha;
          if (more) __builtin_amdgcn_s_waitcnt(FK_PAGED_VMCNT(LOADS));  // V landed, the next K in flight
          else __builtin_amdgcn_s_waitcnt(FK_PAGED_VMCNT(0));
          asm volatile("" ::: "memory");
          if (t * KT < ks.first || t * KT + KT > ks.last) {
            // Rows outside the request's keys hold other values: zeros, so that
            // an infinity there is nothing to a probability of 0.
#pragma unroll
            for (uint32_t q = 0; q < LOADS; q++) {
              const uint32_t k = t * KT + q * KPL + krow;
              if (k < ks.first || k >= ks.last)
                reinterpret_cast<uint4 *>(vbuf)[q * 64 + lane] = make_uint4(0, 0, 0, 0);
            }
            asm volatile("" ::: "memory");
          }
          // Oᵀ += Vᵀ Pᵀ.  Transposed reads: within 16 lanes, lane 4 k + q reads key
          // K0 + k, d D0 + 4 q .. + 3 and receives keys K0 .. K0 + 3 of d D0 + (its
          // index): keys 32 h + 4 (l div 16) .. + 3 and 16 further, parts[h]'s order.
#pragma unroll
          for (uint32_t c = 0; c < KT * DP / 2048; c++) {
            // of 4 addresses and 16 rows further: at 64, two 16s of d by two 32s of
            // keys; else four 16s of d
            constexpr uint32_t DS = DP == 64 ? 2 : 4;
            uint32_t at[4];
            u32x2 w[8];
#pragma unroll
            for (uint32_t i = 0; i < 4; i++)
              at[i] = v_lds + (tk + i / DS * 32) * (2 * DP) + ((16 * (c * DS + i % DS) + td) ^ (v_turn << 4)) * 2;
            paged_read8_tr<16 * 2 * DP>(at, w);
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) {
              const uint32_t d = c * DS + i % DS, h = i / DS;
              const vec vf = __builtin_bit_cast(vec, u32x4{w[i][0], w[i][1], w[4 + i][0], w[4 + i][1]});
#pragma unroll
              for (uint32_t x = 0; x < Op::parts; x++)
                o[d] = Op::mfma(vf, __builtin_bit_cast(vec, parts[h][x]), o[d]);
            }
          }
#pragma unroll
          for (uint32_t d = 0; d < DP / 16; d++) asm volatile("" : "+v"(o[d])::"memory");
          if (more) load(vpool, vbuf, false);
        }
        if (again) return false;
        // (not a number where one of the head's own d is not)
        fk_float4v any = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (uint32_t d = 0; d < DP / 16; d++)
          if (FULL || 16 * d + 4 * (lane / 16) < D) any += o[d];
        const float sum = (any[0] + any[1]) + (any[2] + any[3]);
        return __builtin_amdgcn_ballot_w64(sum != sum && l == l) != 0;
      };
      if (make(fk_bool_tag<false>{})) {
        first_entries();
        __builtin_amdgcn_s_waitcnt(FK_PAGED_VMCNT(0));
        asm volatile("" : "+v"(entries));
        entries = min(entries, a.blocks - 1);
        make(fk_bool_tag<true>{});
      }

      // The wavefronts' states meet, each in the place of its V rows: head l
      // mod 16, d 16 dt + 4 (l div 16) + i.
      float *const so = reinterpret_cast<float *>(vbuf);
      if (lane % 16 < G) {
#pragma unroll
        for (uint32_t d = 0; d < DP / 16; d++)
          *reinterpret_cast<fk_float4v *>(&so[lane % 16 * DP + 16 * d + 4 * (lane / 16)]) = o[d];
        if (lane < 16) {
          sm[wave][lane] = m;
          sl[wave][lane] = l;
        }
      }
      __syncthreads();
      const bool whole = pos == pair0 && seg1 == pair0 + per_pair;
      const uint32_t side = pair0 < begin ? 0u : 1u;
      const auto to = states + paged_state(blockIdx.x, side, pl.rows, D);
      for (uint32_t e = threadIdx.x; e < G * D; e += THREADS) {
        const uint32_t q = e / D, d = e - q * D;
        float mm = sm[0][q];
#pragma unroll
        for (uint32_t w = 1; w < W; w++) mm = __builtin_fmaxf(mm, sm[w][q]);
        const float mc = paged_ref(mm);
        float ll = 0.0f, oo = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < W; w++) {
          const float f = __builtin_amdgcn_exp2f(sm[w][q] - mc);
          ll += sl[w][q] * f;
          oo = paged_plus(oo, reinterpret_cast<const float *>(kv[w][1])[q * DP + d], f);
        }
        if (whole) {
          const uint64_t where = r * a.out_stride + (uint64_t)(h0 + q) * D + d;
          if (a.out_f32) global_at<float>(a.out)[where] = oo / ll;
          else global_at<uint16_t>(a.out)[where] = paged_round<BF16>(oo / ll);
        } else {
          to[q * D + d] = oo;
          if (d == 0) {
            to[pl.rows * D + 2 * q] = mm;
            to[pl.rows * D + 2 * q + 1] = ll;
          }
        }
      }
      if (!pl.whole && pos == pair0) {
        // the pair starts here: it ends here too, or in the threadgroup of its
        // last unit
        u32x4 join = {0, 0, 0, 0};
        if (!whole)
          join = paged_join(blockIdx.x, (pair0 + per_pair - 1) / run, r, h0, G);
        if (pl.by_pair && threadIdx.x == 0) joins[r * per_request + pair] = join;
        last_join = join;
      }
      __syncthreads();  // before the next pair's rows land on the states
      pos = seg1;
    }
    pid += gridDim.x;
  } while (pl.whole && pid < n * per_request);
  if (!pl.whole && !pl.by_pair && threadIdx.x == 0) joins[blockIdx.x] = last_join;
}

// The states of a pair that several threadgroups made, joined in their order:
// threadgroup (entry of the joins, query head), its W wavefronts every W-th
// state each, 8 states at a time.  W is what the pairs have in states on
// average, 2 to 8: the launch is short, and its waves are what it takes (512
// pairs of about 2 states and 4 heads: 5.9 µs by 8 wavefronts, 5.2 by 2).
template <uint32_t W, bool BF16>
__device__ __forceinline__ void paged_attend_join(const fk_paged_attend_args &a, const PagedPlan &pl,
                                                  uint32_t groups) {
  __shared__ float so[W][256], sm[W], sl[W];
  const uint32_t q = blockIdx.x % pl.rows;
  const u32x4 j = global_at<const u32x4>(a.workspace)[blockIdx.x / pl.rows];
  const uint32_t first = j[0] >> 16, last = j[0] & 0xFFFFu;
  if (last == 0 || q > (j[2] & 15u)) return;
  const auto states = global_at<const float>(a.workspace + groups * sizeof(u32x4));
  const uint32_t D = a.head_dim;
  const uint32_t lane = threadIdx.x & (FK_WAVE - 1), wave = threadIdx.x / FK_WAVE;
  float mm = -__builtin_inff(), ll = 0.0f, oo[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  constexpr uint32_t U = 8;  // states at once
  for (uint32_t w0 = first + wave; w0 <= last; w0 += U * W) {
    float m[U], l[U], o[U][4];
#pragma unroll
    for (uint32_t s = 0; s < U; s++) {
      const uint32_t w = min(w0 + s * W, last);
      const auto from = states + paged_state(w, w == first ? 1u : 0u, pl.rows, D);
      const bool there = w0 + s * W <= last;
      m[s] = there ? from[pl.rows * D + 2 * q] : -__builtin_inff();
      l[s] = there ? from[pl.rows * D + 2 * q + 1] : 0.0f;
#pragma unroll
      for (uint32_t i = 0; i < 4; i++) {
        const uint32_t d = lane + 64 * i;
        o[s][i] = there && d < D ? from[q * D + d] : 0.0f;
      }
    }
    float mn = mm;
#pragma unroll
    for (uint32_t s = 0; s < U; s++) mn = __builtin_fmaxf(mn, m[s]);
    const float mc = paged_ref(mn);
    const float f0 = __builtin_amdgcn_exp2f(mm - mc);
    ll *= f0;
#pragma unroll
    for (uint32_t i = 0; i < 4; i++) oo[i] = paged_plus(0.0f, oo[i], f0);
#pragma unroll
    for (uint32_t s = 0; s < U; s++) {
      const float f = __builtin_amdgcn_exp2f(m[s] - mc);
      ll += l[s] * f;
#pragma unroll
      for (uint32_t i = 0; i < 4; i++) oo[i] = paged_plus(oo[i], o[s][i], f);
    }
    mm = mn;
  }
#pragma unroll
  for (uint32_t i = 0; i < 4; i++) so[wave][lane + 64 * i] = oo[i];
  if (lane == 0) {
    sm[wave] = mm;
    sl[wave] = ll;
  }
  __syncthreads();
  mm = sm[0];
#pragma unroll
  for (uint32_t w = 1; w < W; w++) mm = __builtin_fmaxf(mm, sm[w]);
  const float mc = paged_ref(mm);
  float l = 0.0f, f[W];
#pragma unroll
  for (uint32_t w = 0; w < W; w++) {
    f[w] = __builtin_amdgcn_exp2f(sm[w] - mc);
    l += sl[w] * f[w];
  }
  for (uint32_t d = threadIdx.x; d < D; d += 64 * W) {
    float o = 0.0f;
#pragma unroll
    for (uint32_t w = 0; w < W; w++) o = paged_plus(o, so[w][d], f[w]);
    const uint64_t where = j[1] * a.out_stride + (uint64_t)((j[2] >> 4) + q) * D + d;
    if (a.out_f32) global_at<float>(a.out)[where] = o / l;
    else global_at<uint16_t>(a.out)[where] = paged_round<BF16>(o / l);
  }
}

}  // namespace fk
