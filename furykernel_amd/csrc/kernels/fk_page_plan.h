// fk_page_plan.h — block tables and slot maps of a step, from the requests'
// lengths (include/fkrocm_serve.h: fk_page_plan).
//
// Two prefix sums over the requests (tokens, new blocks), then one search a
// token for its request.  A few KB of lengths go in and 12 bytes a token come
// out, so latency bounds it: one launch, in which every threadgroup makes the
// prefix sums for itself (no threadgroup waits for another, nothing is kept
// in memory between) and then takes its own tokens.
//
// The 1024 threads hold the sums of n / 1024 consecutive requests each; a
// token finds its thread's chunk by bisection in LDS and its request by
// walking the chunk.  A block is the free list's next, so its number follows
// from the sums alone: no token waits for a table entry that this launch
// writes.  A request's new page is written by the token that opens it.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fk_address.h"

#include "../../../include/fkrocm_serve.h"

#define FK_PLAN_THREADS 1024
#define FK_PLAN_WAVES (FK_PLAN_THREADS / 64)

namespace fk {

// A request of the plan: how it stands before the blocks are shared out.
struct PlanRequest {
  uint32_t cached, fresh;
  uint32_t held, need;  // blocks it holds, and those it needs if it fits
  bool fits;            // its table row and the step's tokens hold it
};

__device__ __forceinline__ uint32_t plan_pages(uint64_t positions, uint32_t block) {
  return (uint32_t)((positions + block - 1) / block);
}

// Request r whose tokens start at `start` (64 bits: no sum of lengths wraps).
__device__ __forceinline__ PlanRequest plan_request(const fk_page_plan_args &a, uint32_t r, uint64_t start) {
  PlanRequest q;
  q.cached = global_at<const uint32_t>(a.cached)[r];
  q.fresh = global_at<const uint32_t>(a.fresh)[r];
  const uint64_t total = (uint64_t)q.cached + q.fresh;
  q.fits = total <= (uint64_t)a.table_len * a.block_size && start + q.fresh <= a.tokens;
  q.held = q.fits ? plan_pages(q.cached, a.block_size) : 0u;
  q.need = q.fits ? plan_pages(total, a.block_size) - q.held : 0u;
  return q;
}

// The sum of the lanes before this one, and the wavefront's.
template <typename T>
__device__ __forceinline__ T wave_before(T v, T *total) {
  const int lane = threadIdx.x & 63;
  T s = v;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const T o = __shfl_up(s, d, 64);
    if (lane >= d) s += o;
  }
  *total = __shfl(s, 63, 64);
  return s - v;
}

// The sum of the threads before this one, and the threadgroup's; `slots`
// holds a value a wavefront and is free again when every thread is past its
// next barrier.
template <typename T>
__device__ __forceinline__ T group_before(T v, T *slots, T *total) {
  T mine;
  const T within = wave_before(v, &mine);
  const uint32_t wave = threadIdx.x / 64;
  if ((threadIdx.x & 63) == 0) slots[wave] = mine;
  __syncthreads();
  T before = 0, all = 0;
#pragma unroll
  for (uint32_t w = 0; w < FK_PLAN_WAVES; w++) {
    const T s = slots[w];
    before += w < wave ? s : (T)0;
    all += s;
  }
  *total = all;
  return before + within;
}

__device__ __forceinline__ uint32_t plan_u32(uint64_t x) { return x < 0xFFFFFFFFull ? (uint32_t)x : 0xFFFFFFFFu; }

__device__ __forceinline__ void page_plan(const fk_page_plan_args &a) {
  __shared__ uint64_t token_slots[FK_PLAN_WAVES], block_slots[FK_PLAN_WAVES];
  __shared__ uint64_t first_token[FK_PLAN_THREADS];  // the tokens before a chunk's first request
  __shared__ uint64_t first_block[FK_PLAN_THREADS];  // the new blocks before it
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

  uint64_t mine = 0, total;
  for (uint32_t r = r0; r < r1; r++) mine += fresh[r];
  const uint64_t tokens0 = group_before(mine, token_slots, &total);
  uint64_t need = 0, needed;
  {
    uint64_t at = tokens0;
    for (uint32_t r = r0; r < r1; r++) {
      const PlanRequest q = plan_request(a, r, at);
      need += q.need;
      at += q.fresh;
    }
  }
  const uint64_t blocks0 = group_before(need, block_slots, &needed);
  first_token[tid] = tokens0;
  first_block[tid] = blocks0;
  __syncthreads();

  // The requests' own outputs: a chunk's by one threadgroup, the counts by
  // the first, which walks them all.
  const bool writes = tid % gridDim.x == blockIdx.x, counts = blockIdx.x == 0;
  if (writes || counts) {
    uint64_t at = tokens0, after = blocks0;
    uint32_t out = 0, most = 0;
    for (uint32_t r = r0; r < r1; r++) {
      const PlanRequest q = plan_request(a, r, at);
      after += q.need;
      const bool fits = q.fits && (q.need == 0 || after <= avail);
      if (fits && q.need) most = (uint32_t)after;
      out += !fits;
      if (writes) {
        global_at<uint32_t>(a.lengths)[r] = fits ? q.cached + q.fresh : q.cached;
        global_at<uint32_t>(a.starts)[r] = plan_u32(at);
      }
      at += q.fresh;
    }
    if (counts) {
      if (out) atomicAdd(&refused, out);
      if (most) atomicMax(&taken, most);
    }
  }
  if (counts) {
    __syncthreads();
    if (tid == 0) {
      global_at<uint32_t>(a.starts)[n] = plan_u32(total);
      const auto c = global_at<uint32_t>(a.counts);
      c[0] = plan_u32(total);
      c[1] = taken;
      c[2] = refused;
      c[3] = head + taken;
    }
  }

  const auto table = global_at<const uint32_t>(a.table);
  const auto free_blocks = global_at<const uint32_t>(a.free_blocks);
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
      uint64_t at = first_token[lo], blocks = first_block[lo];
      PlanRequest q = plan_request(a, r, at);
      while (at + q.fresh <= t) {
        at += q.fresh;
        blocks += q.need;
        q = plan_request(a, ++r, at);
      }
      owner = r;
      pos = q.cached + (uint32_t)(t - at);
      if (q.fits && (q.need == 0 || blocks + q.need <= avail)) {
        const uint32_t page = pos / a.block_size, within = pos - page * a.block_size;
        uint32_t block;
        if (page < q.held) {
          block = table[(uint64_t)r * a.table_len + page];
        } else {
          block = free_blocks[head + (uint32_t)blocks + (page - q.held)];
          if (within == 0) global_at<uint32_t>(a.table)[(uint64_t)r * a.table_len + page] = block;
        }
        slot = plan_u32((uint64_t)block * a.block_size + within);
      }
    }
    global_at<uint32_t>(a.slots)[t] = slot;
    global_at<uint32_t>(a.positions)[t] = pos;
    global_at<uint32_t>(a.owner)[t] = owner;
  }
}

}  // namespace fk
