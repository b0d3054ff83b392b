// fk_page_plan.h — block tables and slot maps of a step, from the requests'
// lengths (include/fkrocm_serve.h: fk_page_plan).
//
// Two prefix sums over the requests (tokens, new blocks), then one search a
// token for its request.  A few KB of lengths go in and 12 bytes a token come
// out, so latency bounds it: one launch, in which every threadgroup makes the
// prefix sums for itself (no threadgroup waits for another, nothing is kept
// in memory between) and then takes its own tokens.
//
// Up to 2048 requests stay in LDS, one to four a thread: their lengths are read
// once, and a token finds its request by a search there.  Of more, each of
// the 1024 threads holds the sums of n / 1024 consecutive ones; a token finds
// its thread's chunk by bisection and its request by walking the chunk.  A
// block is the free list's next, so its number follows from the sums alone: no
// token waits for a table entry that this launch writes.  A request's new page
// is written by the token that opens it.
//
// What a thread does before the tokens is one long chain, so its parts are
// short: quotients by the launch's block size as products, no branches, all
// that memory gives asked for before the first wait (8 requests of 256
// threads 3.6 µs with divisions, branches and loads where they are used, 2.9
// so; 1500 with 59 thousand tokens 7.2 and 6.5).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fk_address.h"
#include "fk_divisor.h"

#include "../../../include/fkrocm_serve.h"

#define FK_PLAN_THREADS 1024

namespace fk {

// A request of the plan: how it stands before the blocks are shared out.
struct PlanRequest {
  uint32_t cached, fresh;
  uint32_t held, need;  // blocks it holds, and those it needs if it fits
  bool fits;            // its table row and the step's tokens hold it
};

__device__ __forceinline__ uint32_t plan_pages(uint32_t positions, const Divisor &block) {
  const uint32_t some = min(positions, 1u);
  return quotient(positions - some, block) + some;
}

// Sums of tokens stop at 2^32 - 1, which no step has: what is past it is past
// every step's end.
__device__ __forceinline__ uint32_t plan_add(uint32_t x, uint32_t y) { return __builtin_elementwise_add_sat(x, y); }

// A request whose tokens start at `start`.
__device__ __forceinline__ PlanRequest plan_request(const fk_page_plan_args &a, const Divisor &block, uint32_t cached,
                                                    uint32_t fresh, uint32_t start) {
  PlanRequest q;
  q.cached = cached;
  q.fresh = fresh;
  const uint64_t total = (uint64_t)q.cached + q.fresh;
  q.fits = total <= (uint64_t)a.table_len * block.by && plan_add(start, fresh) <= a.tokens;
  const uint32_t held = plan_pages(q.cached, block), all = plan_pages((uint32_t)total, block);
  q.held = q.fits ? held : 0u;
  q.need = q.fits ? all - held : 0u;
  return q;
}

__device__ __forceinline__ PlanRequest plan_request(const fk_page_plan_args &a, const Divisor &block, uint32_t r,
                                                    uint32_t start) {
  return plan_request(a, block, global_at<const uint32_t>(a.cached)[r], global_at<const uint32_t>(a.fresh)[r], start);
}

// A lane's value from DPP control CTRL's lane, 0 where there is none or the
// row is none of ROWS.
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t plan_dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}

// The sum of the lanes up to this one.
__device__ __forceinline__ uint32_t wave_upto(uint32_t v) {
  v = plan_add(v, plan_dpp<0x111, 0xF>(v));  // row_shr 1, 2, 4, 8
  v = plan_add(v, plan_dpp<0x112, 0xF>(v));
  v = plan_add(v, plan_dpp<0x114, 0xF>(v));
  v = plan_add(v, plan_dpp<0x118, 0xF>(v));
  v = plan_add(v, plan_dpp<0x142, 0xA>(v));  // row_bcast 15: rows 0 and 2 onto 1 and 3
  return plan_add(v, plan_dpp<0x143, 0xC>(v));  // row_bcast 31: the lower half onto the upper
}

// The sum of the threads before this one, and the threadgroup's; `slots`
// holds a value a wavefront and is used once.
template <uint32_t THREADS>
__device__ __forceinline__ uint32_t group_before(uint32_t v, uint32_t *slots, uint32_t *total) {
  const uint32_t upto = wave_upto(v), wave = threadIdx.x / 64, lane = threadIdx.x & 63;
  // (before this lane: the lane below's sum, which a difference would lose
  // where the sum has stopped)
  const uint32_t below = __shfl_up(upto, 1, 64);
  if (lane == 63) slots[wave] = upto;
  __syncthreads();
  uint32_t before = 0, all = 0;
#pragma unroll
  for (uint32_t w = 0; w < THREADS / 64; w++) {
    before = plan_add(before, w < wave ? slots[w] : 0u);
    all = plan_add(all, slots[w]);
  }
  *total = all;
  return plan_add(before, lane ? below : 0u);
}

// x, or the largest count for what is past it.
__device__ __forceinline__ uint32_t plan_u32(uint64_t x) { return x < 0xFFFFFFFFull ? (uint32_t)x : 0xFFFFFFFFu; }

// Token t of a request whose position is pos: its slot.  `held` blocks are in
// the table, new ones in the free list from `first` on.
__device__ __forceinline__ uint32_t plan_slot(const fk_page_plan_args &a, const Divisor &size, uint32_t r,
                                              uint32_t pos, uint32_t held, uint32_t first) {
  const auto table = global_at<uint32_t>(a.table) + (uint64_t)r * a.table_len;
  const uint32_t page = quotient(pos, size), within = pos - page * size.by;
  uint32_t block;
  if (page < held) {
    block = table[page];
  } else {
    block = global_at<const uint32_t>(a.free_blocks)[first + (page - held)];
    if (within == 0) table[page] = block;
  }
  return plan_u32((uint64_t)block * size.by + within);
}

__device__ __forceinline__ void plan_token(const fk_page_plan_args &a, uint32_t t, uint32_t slot, uint32_t pos,
                                           uint32_t owner) {
  global_at<uint32_t>(a.slots)[t] = slot;
  global_at<uint32_t>(a.positions)[t] = pos;
  global_at<uint32_t>(a.owner)[t] = owner;
}

__device__ __forceinline__ void plan_counts(const fk_page_plan_args &a, uint32_t total, uint32_t head, uint32_t taken,
                                            uint32_t refused) {
  global_at<uint32_t>(a.starts)[a.requests] = total;
  const auto c = global_at<uint32_t>(a.counts);
  c[0] = total;
  c[1] = taken;
  c[2] = refused;
  c[3] = head + taken;
}

// At most PER THREADS requests, PER a thread.
template <uint32_t THREADS, uint32_t PER>
__device__ __forceinline__ void page_plan_held(const fk_page_plan_args &a, const Divisor &block, uint32_t groups) {
  constexpr uint32_t HELD = PER * THREADS;
  __shared__ uint32_t token_slots[THREADS / 64], block_slots[THREADS / 64], refused, taken;
  // a request's first token, its cached positions, its first new block's place
  // in the free list (below free_len; FK_NO_SLOT: it does not fit)
  __shared__ uint32_t starts[HELD], held_at[HELD], firsts[HELD];
  const uint32_t tid = threadIdx.x, n = a.requests;
  uint32_t head = *global_at<const uint32_t>(a.head), free_len = a.free_len;
  uint32_t c[PER], f[PER];
#pragma unroll
  for (uint32_t i = 0; i < PER; i++) {
    // (past the last: the last again, put to 0 below, so that the loads need no
    // branches)
    const uint32_t r = min(PER * tid + i, n - 1);
    c[i] = global_at<const uint32_t>(a.cached)[r];
    f[i] = global_at<const uint32_t>(a.fresh)[r];
  }
  // (everything on its way before the first wait)
  asm volatile("" : "+s"(head), "+s"(free_len));
#pragma unroll
  for (uint32_t i = 0; i < PER; i++) {
    c[i] = PER * tid + i < n ? c[i] : 0u;
    f[i] = PER * tid + i < n ? f[i] : 0u;
  }
  const uint32_t avail = free_len > head ? free_len - head : 0u;
  if (tid == 0) refused = taken = 0;
  uint32_t mine = f[0], total;
#pragma unroll
  for (uint32_t i = 1; i < PER; i++) mine = plan_add(mine, f[i]);
  uint32_t first[PER];
  first[0] = group_before<THREADS>(mine, token_slots, &total);
#pragma unroll
  for (uint32_t i = 1; i < PER; i++) first[i] = plan_add(first[i - 1], f[i - 1]);
  // (requests that fit need a block a token at most, so the step's fewer than
  // 2^32)
  PlanRequest q[PER];
  uint32_t need = 0, needed;
#pragma unroll
  for (uint32_t i = 0; i < PER; i++) {
    q[i] = plan_request(a, block, c[i], f[i], first[i]);
    need += q[i].need;
  }
  uint32_t after = group_before<THREADS>(need, block_slots, &needed);
  uint32_t out = 0, most = 0;
  // a wavefront's requests' own outputs: by the threadgroup of its number
  const bool writes = min(__builtin_amdgcn_readfirstlane(tid / 64), groups - 1) == blockIdx.x;
#pragma unroll
  for (uint32_t i = 0; i < PER; i++) {
    const uint32_t r = PER * tid + i;
    const uint32_t before = after;
    after += q[i].need;
    const bool fits = q[i].fits && (q[i].need == 0 || after <= avail);
    const uint32_t start = r < n ? first[i] : 0xFFFFFFFFu;
    starts[r] = start;
    held_at[r] = c[i];
    firsts[r] = fits ? (q[i].need ? head + before : 0u) : FK_NO_SLOT;
    if (r < n) {
      if (fits && q[i].need) most = after;
      out += !fits;
      if (writes) {
        global_at<uint32_t>(a.lengths)[r] = fits ? c[i] + f[i] : c[i];
        global_at<uint32_t>(a.starts)[r] = start;
      }
    }
  }
  if (blockIdx.x == 0) {
    if (out) atomicAdd(&refused, out);
    if (most) atomicMax(&taken, most);
  }
  __syncthreads();
  if (blockIdx.x == 0 && tid == 0) plan_counts(a, total, head, taken, refused);
  for (uint64_t t64 = (uint64_t)blockIdx.x * THREADS + tid; t64 < a.tokens;
       t64 += (uint64_t)groups * THREADS) {
    const uint32_t t = (uint32_t)t64;
    uint32_t slot = FK_NO_SLOT, pos = 0, owner = FK_NO_SLOT;
    if (t < total) {
      // the last request that starts at or before t: one without tokens starts
      // where the next does
      // (by quarters, three reads beside each other in place of two behind: 1 to
      // 2 % of the launch)
      constexpr bool ODD = HELD & 0xAAAAAAAAu;  // an odd power of 2: a half first
      owner = ODD && starts[HELD / 2] <= t ? HELD / 2 : 0u;
#pragma unroll
      for (uint32_t step = HELD / (ODD ? 8 : 4); step > 0; step /= 4) {
        const uint32_t s1 = starts[owner + step], s2 = starts[owner + 2 * step], s3 = starts[owner + 3 * step];
        owner += step * ((s1 <= t) + (s2 <= t) + (s3 <= t));
      }
      const uint32_t cached = held_at[owner], free_at = firsts[owner];
      pos = cached + (t - starts[owner]);
      if (free_at != FK_NO_SLOT) slot = plan_slot(a, block, owner, pos, plan_pages(cached, block), free_at);
    }
    plan_token(a, t, slot, pos, owner);
  }
}

__device__ __forceinline__ void page_plan(const fk_page_plan_args &a, const Divisor &block) {
  __shared__ uint32_t token_slots[FK_PLAN_THREADS / 64], block_slots[FK_PLAN_THREADS / 64];
  __shared__ uint32_t first_token[FK_PLAN_THREADS];  // the tokens before a chunk's first request
  __shared__ uint32_t first_block[FK_PLAN_THREADS];  // the new blocks before it
  __shared__ uint32_t refused, taken;
  const uint32_t tid = threadIdx.x;
  const uint32_t n = a.requests;
  const uint32_t chunk = (uint32_t)(((uint64_t)n + FK_PLAN_THREADS - 1) / FK_PLAN_THREADS);
  const uint32_t r0 = (uint32_t)min((uint64_t)tid * chunk, (uint64_t)n);
  const uint32_t r1 = (uint32_t)min((uint64_t)r0 + chunk, (uint64_t)n);
  const auto fresh = global_at<const uint32_t>(a.fresh);
  const uint32_t head = *global_at<const uint32_t>(a.head);
  const uint32_t avail = a.free_len > head ? a.free_len - head : 0u;
  if (tid == 0) refused = taken = 0;

  uint32_t mine = 0, total;
  for (uint32_t r = r0; r < r1; r++) mine = plan_add(mine, fresh[r]);
  const uint32_t tokens0 = group_before<FK_PLAN_THREADS>(mine, token_slots, &total);
  uint32_t need = 0, needed;
  {
    uint32_t at = tokens0;
    for (uint32_t r = r0; r < r1; r++) {
      const PlanRequest q = plan_request(a, block, r, at);
      need += q.need;
      at = plan_add(at, q.fresh);
    }
  }
  const uint32_t blocks0 = group_before<FK_PLAN_THREADS>(need, block_slots, &needed);
  first_token[tid] = tokens0;
  first_block[tid] = blocks0;
  __syncthreads();

  // The requests' own outputs: a chunk's by one threadgroup, the counts by
  // the first, which walks them all.
  const bool writes = tid % gridDim.x == blockIdx.x, counts = blockIdx.x == 0;
  if (writes || counts) {
    uint32_t at = tokens0, after = blocks0;
    uint32_t out = 0, most = 0;
    for (uint32_t r = r0; r < r1; r++) {
      const PlanRequest q = plan_request(a, block, r, at);
      after += q.need;
      const bool fits = q.fits && (q.need == 0 || after <= avail);
      if (fits && q.need) most = after;
      out += !fits;
      if (writes) {
        global_at<uint32_t>(a.lengths)[r] = fits ? q.cached + q.fresh : q.cached;
        global_at<uint32_t>(a.starts)[r] = at;
      }
      at = plan_add(at, q.fresh);
    }
    if (counts) {
      if (out) atomicAdd(&refused, out);
      if (most) atomicMax(&taken, most);
    }
  }
  if (counts) {
    __syncthreads();
    if (tid == 0) plan_counts(a, total, head, taken, refused);
  }

  for (uint64_t t64 = (uint64_t)blockIdx.x * FK_PLAN_THREADS + tid; t64 < a.tokens;
       t64 += (uint64_t)gridDim.x * FK_PLAN_THREADS) {
    const uint32_t t = (uint32_t)t64;
    uint32_t slot = FK_NO_SLOT, pos = 0, owner = FK_NO_SLOT;
    if (t < total) {
      // the last chunk whose first token is not past t: the tokens of empty
      // chunks start where the next one's do
      uint32_t lo = 0;
#pragma unroll
      for (uint32_t step = FK_PLAN_THREADS / 2; step > 0; step /= 2)
        if (first_token[lo + step] <= t) lo += step;
      uint32_t r = lo * chunk;
      uint32_t at = first_token[lo], blocks = first_block[lo];
      PlanRequest q = plan_request(a, block, r, at);
      while (plan_add(at, q.fresh) <= t) {
        at = plan_add(at, q.fresh);
        blocks += q.need;
        q = plan_request(a, block, ++r, at);
      }
      owner = r;
      pos = q.cached + (t - at);
      if (q.fits && (q.need == 0 || blocks + q.need <= avail))
        slot = plan_slot(a, block, r, pos, q.held, head + blocks);
    }
    plan_token(a, t, slot, pos, owner);
  }
}

}  // namespace fk
