// fk_serve.hip — the operators of a served batch as one C call each
// (include/fkrocm_serve.h), their kernels compiled into the C ABI's library.
//
// Each entry checks its arguments against what its kernels take, on the host
// and before anything is queued, then launches on the caller's stream.

#include "../../include/fkrocm_serve.h"

#include <hip/hip_runtime.h>

#include <cstdio>
#include <cstring>

#include "fk_admit.h"
#include "kernels/fk_page_plan.h"
#include "kernels/fk_paged_attend.h"
#include "kernels/fk_paged_store.h"

using fk::admit;
using fk::check_spans;
using fk::launched;
using fk::Refusal;
using fk::Span;
using fk::stream_of;

namespace {

template <uint32_t THREADS, uint32_t PER>
__global__ void __launch_bounds__(THREADS) op_page_plan_held(fk_page_plan_args a, fk::Divisor block, uint32_t groups) {
  fk::page_plan_held<THREADS, PER>(a, block, groups);
}
__global__ void __launch_bounds__(FK_PLAN_THREADS) op_page_plan(fk_page_plan_args a, fk::Divisor block, uint32_t) {
  fk::page_plan(a, block);
}

template <int T, bool BF16>
__global__ void __launch_bounds__(FK_STORE_THREADS) op_paged_store(fk_paged_store_args a) {
  fk::paged_store<T, BF16>(a);
}

template <uint32_t DP, uint32_t W, bool FULL, bool BF16>
__global__ void __launch_bounds__(64 * W, DP == 256 || W == 8 ? 1 : 2)
    op_paged_attend(fk_paged_attend_args a, fk::PagedPlan pl) {
  fk::paged_attend<DP, W, FULL, BF16>(a, pl);
}

template <uint32_t W, bool BF16>
__global__ void __launch_bounds__(64 * W)
    op_paged_attend_join(fk_paged_attend_args a, fk::PagedPlan pl, uint32_t groups) {
  fk::paged_attend_join<W, BF16>(a, pl, groups);
}

// The attention's launch for these sizes: head_dim's tile width, its wavefronts
// and threadgroups, the joins' entries and what the kernels take; 0
// threadgroups and the reason if the kernels do not take them.
struct AttendLaunch {
  uint32_t width = 0, waves = 4, groups = 0, joins = 0;
  fk::PagedPlan plan{};
  const char *why = "";
};

AttendLaunch attend_launch(const fk_paged_attend_args &a) {
  AttendLaunch l;
  const uint64_t length = (uint64_t)a.table_len * a.block_size;
  if (a.requests == 0 || a.kv_heads == 0 || a.heads == 0 || a.heads % a.kv_heads) {
    l.why = "requests and heads that kv_heads divides";
  } else if (a.head_dim == 0 || a.head_dim % 8 || a.head_dim > 256) {
    l.why = "head_dim a multiple of 8, at most 256";
  } else if (a.block_size == 0 || a.blocks == 0 || a.table_len == 0) {
    l.why = "blocks, their size and a table";
  } else if (length >= 1ull << 31 || (uint64_t)a.blocks * a.block_size >= 1ull << 32) {
    l.why = "a table of fewer than 2^31 positions, a pool of fewer than 2^32";
  } else if ((uint64_t)a.heads * a.head_dim >= 1ull << 31 || a.requests >= 1u << 24) {
    l.why = "rows of fewer than 2^31 elements, fewer than 2^24 requests";
  } else {
    l.width = a.head_dim <= 64 ? 64 : (a.head_dim <= 128 ? 128 : 256);
    l.plan.group = a.heads / a.kv_heads;
    l.plan.head_tiles = (l.plan.group + 15) / 16;
    l.plan.rows = l.plan.group < 16 ? l.plan.group : 16;
    l.plan.length = (uint32_t)length;
    const uint64_t unit = (l.width == 64 ? 64 : 32) * FK_PAGED_WAVES;
    const uint64_t seen = a.window && a.window < length ? a.window + unit : length;
    // the kernels count units in 32 bits
    const __uint128_t units = (__uint128_t)a.requests * a.kv_heads * l.plan.head_tiles * ((seen + unit - 1) / unit);
    if (units >= 1ull << 31) {
      l.why = "fewer than 2^31 units of keys";
      return l;
    }
    // as many as the chip's 256 compute units hold at once
    const uint64_t most = l.width == 256 ? 256 : 512;
    l.groups = (uint32_t)(units < most ? (uint64_t)units : most);
    const uint64_t pairs = (uint64_t)a.requests * a.kv_heads * l.plan.head_tiles;
    l.plan.by_pair = pairs <= l.groups;
    l.joins = l.plan.by_pair ? (uint32_t)pairs : l.groups;
    // Few units a pair at most: a threadgroup takes pairs whole, which saves the
    // prefix sum and the join and costs each further unit's time, and a long
    // pair's to the launch; where the pairs do not fill the CUs by 8 wavefronts,
    // which share all but three units better than 4.  Requests of up to u units
    // (256 keys of 64, 128 of 128), evenly spread (the one has u), µs split,
    // whole by 4, whole by 8:
    //    pairs, width    u = 2           3               4               5               6
    //      8 of 64   10.0  7.2  6.9  10.3  8.8  8.9  10.6 10.4  9.2  10.6 12.1 11.3  10.6 13.7 11.6
    //     80 of 64   10.7  7.6  7.3  11.0  9.1  9.3  11.5 10.7  9.8  11.9 12.2 11.8  13.6 14.0 12.4
    //    164 of 64   11.6  7.9  7.8  13.3  9.5 10.0  13.8 11.1 10.5  14.4 12.8 12.9  16.7 14.5 13.0
    //    328 of 64   13.9  9.2 12.8  18.1 11.2 15.3  17.6 13.6 16.3  20.4 16.2 18.8  22.0 18.1 19.6
    //      8 of 128  11.0  7.8  7.2  11.1  9.2  9.1  11.4 10.6  9.5  11.3 12.1 11.1  11.4 13.5 11.7
    //     80 of 128  11.5  8.1  7.5  11.9  9.5  9.3  12.5 11.0  9.9  12.9 12.2 11.5  14.3 13.8 12.3
    //    164 of 128  12.5  8.4  7.9  14.1  9.9  9.9  14.6 11.4 10.5  15.0 13.0 12.3  17.9 14.2 13.2
    //    328 of 128  14.7  9.7 13.3  19.7 11.7 15.5  18.8 14.0 16.7  22.1 16.2 18.9  23.8 18.2 19.9
    // (f16; bf16 within 4 % of it).  Of 256 (128 keys), 2, 32 and 82 pairs of all
    // u units, split and whole by 4: 14.5 11.9, 15.0 12.5 and 16.4 13.4 at 2, 14.4
    // 14.5, 15.8 15.1 and 17.9 15.9 at 3.  (Many pairs gain at more units too, but one of the table's length
    // among short ones would cost more: that is what the host knows.)
    const uint64_t each = (seen + unit - 1) / unit;
    l.waves = l.width != 256 && pairs <= 256 && each >= 2 && each != 3 ? 8 : 4;
    l.plan.whole = each <= (l.width == 256 ? 2 : pairs < 64 ? 4 : 6);
    if (!l.plan.whole) l.waves = 4;
    if (l.plan.whole) l.groups = (uint32_t)(pairs < most ? pairs : most);
  }
  return l;
}

size_t attend_bytes(const fk_paged_attend_args &a, const AttendLaunch &l) {
  return l.groups * (sizeof(fk::u32x4) + 2 * (size_t)l.plan.rows * (a.head_dim + 2) * sizeof(float));
}

template <uint32_t DP, uint32_t W, bool BF16>
void queue_attend(const fk_paged_attend_args &a, const AttendLaunch &l, hipStream_t s) {
  if (a.head_dim == DP)
    hipLaunchKernelGGL((op_paged_attend<DP, W, true, BF16>), dim3(l.groups), dim3(64 * W), 0, s, a, l.plan);
  else
    hipLaunchKernelGGL((op_paged_attend<DP, W, false, BF16>), dim3(l.groups), dim3(64 * W), 0, s, a, l.plan);
}

template <bool BF16>
void queue_attend(const fk_paged_attend_args &a, const AttendLaunch &l, hipStream_t s) {
  if (l.width == 256) queue_attend<256, 4, BF16>(a, l, s);
  else if (l.width == 128) l.waves == 8 ? queue_attend<128, 8, BF16>(a, l, s) : queue_attend<128, 4, BF16>(a, l, s);
  else l.waves == 8 ? queue_attend<64, 8, BF16>(a, l, s) : queue_attend<64, 4, BF16>(a, l, s);
}

template <uint32_t W>
void queue_join(const fk_paged_attend_args &a, const AttendLaunch &l, hipStream_t s) {
  const dim3 grid(l.joins * l.plan.rows), block(64 * W);
  if (a.cache_bf16) hipLaunchKernelGGL((op_paged_attend_join<W, true>), grid, block, 0, s, a, l.plan, l.groups);
  else hipLaunchKernelGGL((op_paged_attend_join<W, false>), grid, block, 0, s, a, l.plan, l.groups);
}

}  // namespace

namespace fk {

static int check(const fk_page_plan_args &a, Refusal &no) {
  if (a.requests == 0 || a.requests >= 1u << 24 || a.table_len == 0 || a.block_size == 0)
    return no(FK_ERR_ARG, "%u requests (1 to 2^24 - 1), tables of %u blocks of %u", a.requests, a.table_len,
              a.block_size);
  if ((uint64_t)a.table_len * a.block_size >= 1ull << 32 || a.tokens == 0xFFFFFFFFu)
    return no(FK_ERR_RANGE, "tables of %u blocks of %u, %u tokens: past 32 bits", a.table_len, a.block_size, a.tokens);
  const uint64_t n = a.requests, t = a.tokens;
  const Span reads[] = {{"cached", a.cached, 4 * n, 4},
                        {"fresh", a.fresh, 4 * n, 4},
                        {"free_blocks", a.free_blocks, 4ull * a.free_len, 4},
                        {"head", a.head, 4, 4}};
  const Span writes[] = {{"table", a.table, 4 * n * a.table_len, 4}, {"lengths", a.lengths, 4 * n, 4},
                         {"starts", a.starts, 4 * (n + 1), 4},       {"slots", a.slots, 4 * t, 4},
                         {"positions", a.positions, 4 * t, 4},       {"owner", a.owner, 4 * t, 4},
                         {"counts", a.counts, 16, 4}};
  return check_spans(no, reads, 4, writes, 7);
}

// Units of 16 elements that a token's rows have: one thread's work.
static uint64_t store_units(const fk_paged_store_args &a) {
  return ((a.q ? (uint64_t)a.heads : 0) + 2ull * a.kv_heads) * (a.head_dim / 16);
}

static int check(const fk_paged_store_args &a, Refusal &no) {
  if (a.kv_heads == 0 || a.head_dim == 0 || a.head_dim % 16 || a.head_dim > 256 || (a.q && a.heads == 0))
    return no(FK_ERR_ARG, "%u heads over %u of width %u (a multiple of 16, at most 256)", a.heads, a.kv_heads,
              a.head_dim);
  if (a.block_size == 0 || a.blocks == 0 || (uint64_t)a.blocks * a.block_size >= 1ull << 32)
    return no(FK_ERR_RANGE, "%u blocks of %u", a.blocks, a.block_size);
  if (a.rows_type > FK_T_BF16) return no(FK_ERR_ARG, "rows of type %u", a.rows_type);
  if (2ull * a.rotated > a.head_dim || (a.rotated && a.rope_rows == 0))
    return no(FK_ERR_ARG, "RoPE of %u pairs of a head of %u from a table of %u rows", a.rotated, a.head_dim,
              a.rope_rows);
  const uint64_t T = a.tokens, wide = a.rows_type == FK_T_F32 ? 4 : 2, row16 = 16 / wide;
  const uint64_t qw = a.q ? (uint64_t)a.heads * a.head_dim : 0, kw = (uint64_t)a.kv_heads * a.head_dim;
  const uint64_t most = 1ull << 40;
  if ((a.q && (a.q_stride % row16 || a.q_stride < qw || a.q_stride >= most)) || a.k_stride % row16 ||
      a.k_stride < kw || a.k_stride >= most || a.v_stride % row16 || a.v_stride < kw || a.v_stride >= most)
    return no(FK_ERR_ARG, "row strides %llu, %llu, %llu: at least a row, multiples of 16 bytes",
              (unsigned long long)a.q_stride, (unsigned long long)a.k_stride, (unsigned long long)a.v_stride);
  if ((__uint128_t)store_units(a) * T >= (1ull << 32) - FK_STORE_THREADS)
    return no(FK_ERR_RANGE, "%u tokens of %llu units of 16 elements: past 32 bits", a.tokens,
              (unsigned long long)store_units(a));
  // (the kernel counts a row's elements in 32 bits)
  if (qw >= 1ull << 31 || kw >= 1ull << 31)
    return no(FK_ERR_RANGE, "%u heads over %u of width %u: rows of 2^31 elements and more", a.heads, a.kv_heads,
              a.head_dim);
  auto rows = [&](uint64_t stride, uint64_t width) { return fk::rows_span(T, stride, width, wide); };
  const __uint128_t pool = (__uint128_t)a.blocks * a.block_size * kw * 2;
  if (pool >= 1ull << 48) return no(FK_ERR_RANGE, "a pool of 2^48 bytes and more");
  const Span reads[] = {{"q", a.q, a.q ? rows(a.q_stride, qw) : 0},
                        {"k", a.k, rows(a.k_stride, kw)},
                        {"v", a.v, rows(a.v_stride, kw)},
                        {"slots", a.slots, 4 * T, 4},
                        {"positions", a.positions, a.rotated ? 4 * T : 0, 4},
                        {"rope", a.rope, a.rotated ? 8ull * a.rope_rows * a.rotated : 0}};
  const Span writes[] = {{"qr", a.qr, T * qw * 2},
                         {"kpool", a.kpool, (uint64_t)pool},
                         {"vpool", a.vpool, (uint64_t)pool}};
  return check_spans(no, reads, 6, writes, 3);
}

static int check(const fk_paged_attend_args &a, const AttendLaunch &l, Refusal &no) {
  if (l.groups == 0)
    return no(FK_ERR_ARG, "%u requests, %u heads over %u of width %u, %u blocks of %u, tables of %u: it takes %s",
              a.requests, a.heads, a.kv_heads, a.head_dim, a.blocks, a.block_size, a.table_len, l.why);
  const uint64_t n = a.requests, w = (uint64_t)a.heads * a.head_dim, most = 1ull << 38;
  if (a.q_stride < w || a.q_stride % 8 || a.q_stride >= most || a.out_stride < w || a.out_stride >= most)
    return no(FK_ERR_ARG, "row strides %llu and %llu: at least %llu, q's a multiple of 8",
              (unsigned long long)a.q_stride, (unsigned long long)a.out_stride, (unsigned long long)w);
  const size_t bytes = attend_bytes(a, l);
  if (a.workspace_bytes < bytes)
    return no(FK_ERR_RANGE, "a workspace of %llu bytes, %zu needed", (unsigned long long)a.workspace_bytes, bytes);
  const __uint128_t pool = (__uint128_t)a.blocks * a.block_size * a.kv_heads * a.head_dim * 2;
  if (pool >= 1ull << 48) return no(FK_ERR_RANGE, "a pool of 2^48 bytes and more");
  if (a.starts && a.q_rows == 0) return no(FK_ERR_ARG, "starts of no rows of q");
  const uint64_t q_rows = a.starts ? a.q_rows : n;
  const Span reads[] = {{"q", a.q, fk::rows_span(q_rows, a.q_stride, w, 2)},
                        {"kpool", a.kpool, (uint64_t)pool},
                        {"vpool", a.vpool, (uint64_t)pool},
                        {"table", a.table, 4 * n * a.table_len, 4},
                        {"lengths", a.lengths, 4 * n, 4},
                        {"starts", a.starts, a.starts ? 4 * (n + 1) : 0, 4}};
  const Span writes[] = {{"out", a.out, fk::rows_span(n, a.out_stride, w, a.out_f32 ? 4 : 2)},
                         {"workspace", a.workspace, bytes}};
  return check_spans(no, reads, 6, writes, 2);
}

}  // namespace fk

using fk::check;
using fk::store_units;

extern "C" int fk_serve_check(const char *entry, const void *args, size_t args_bytes, char *err, size_t err_cap) {
  Refusal no;
  int st = FK_OK;
  auto is = [&](const char *name, size_t bytes) {
    if (!entry || std::strcmp(entry, name)) return false;
    if (!args || args_bytes != bytes) {
      st = no(FK_ERR_ARG, "%s: %zu bytes of arguments, it takes %zu", name, args_bytes, bytes);
      return false;
    }
    return true;
  };
  if (is("fk_page_plan", sizeof(fk_page_plan_args))) {
    st = check(*static_cast<const fk_page_plan_args *>(args), no);
  } else if (is("fk_paged_store", sizeof(fk_paged_store_args))) {
    st = check(*static_cast<const fk_paged_store_args *>(args), no);
  } else if (is("fk_paged_attend", sizeof(fk_paged_attend_args))) {
    const fk_paged_attend_args &a = *static_cast<const fk_paged_attend_args *>(args);
    st = check(a, attend_launch(a), no);
  } else if (is("fk_mx4_quantize", sizeof(fk_mx4_quantize_args))) {
    st = check(*static_cast<const fk_mx4_quantize_args *>(args), no);
  } else if (is("fk_mx4_dequantize", sizeof(fk_mx4_dequantize_args))) {
    st = check(*static_cast<const fk_mx4_dequantize_args *>(args), no);
  } else if (is("fk_mx4_gemm", sizeof(fk_mx4_gemm_args))) {
    st = check(*static_cast<const fk_mx4_gemm_args *>(args), no);
  } else if (is("fk_fp8_quantize", sizeof(fk_fp8_quantize_args))) {
    st = check(*static_cast<const fk_fp8_quantize_args *>(args), no);
  } else if (is("fk_fp8_dequantize", sizeof(fk_fp8_dequantize_args))) {
    st = check(*static_cast<const fk_fp8_dequantize_args *>(args), no);
  } else if (is("fk_fp8_add_norm", sizeof(fk_fp8_add_norm_args))) {
    st = check(*static_cast<const fk_fp8_add_norm_args *>(args), no);
  } else if (is("fk_fp8_gemm", sizeof(fk_fp8_gemm_args))) {
    st = check(*static_cast<const fk_fp8_gemm_args *>(args), no);
  } else if (is("fk_paged_store8", sizeof(fk_paged_store8_args))) {
    st = check(*static_cast<const fk_paged_store8_args *>(args), no);
  } else if (is("fk_paged_load8", sizeof(fk_paged_load8_args))) {
    st = check(*static_cast<const fk_paged_load8_args *>(args), no);
  } else if (is("fk_paged_attend8", sizeof(fk_paged_attend8_args))) {
    st = check(*static_cast<const fk_paged_attend8_args *>(args), no);
  } else if (st == FK_OK) {
    st = no(FK_ERR_NOT_FOUND, "no operator %s", entry ? entry : "(null)");
  }
  if (err && err_cap) snprintf(err, err_cap, "%s", no.text);
  return st;
}

extern "C" int fk_page_plan(fk_ctx *ctx, const fk_page_plan_args *a, fk_stream *stream) {
  if (int st = admit(ctx, "fk_page_plan", a, stream)) return st;
  auto queue = [&](auto kernel, uint32_t threads) {
    const uint64_t groups = ((uint64_t)a->tokens + threads - 1) / threads;
    const uint32_t g = (uint32_t)(groups < 1 ? 1 : (groups > 256 ? 256 : groups));
    hipLaunchKernelGGL(kernel, dim3(g), dim3(threads), 0, stream_of(ctx, stream), *a, fk::divisor(a->block_size), g);
  };
  // The fewest wavefronts that hold the requests, one or two a thread: a barrier
  // and a sum of few beats another request a thread, but not another two.  µs,
  // one behind another, by threads x requests a thread:
  //   requests, tokens    256x1  256x2  512x2  256x4  512x4  1024x2
  //       8,     8         2.93   3.17   3.36   3.46   3.75   3.99
  //     200,   200         3.21   3.53   3.72   3.86   4.17   4.18
  //     500,   500                3.53   3.89   4.09   4.53   4.33
  //     500, 51480                5.13   5.51   5.55   6.00   6.05
  //    1000,  1000                       3.89   4.06   4.59   4.74
  //    1500, 58169                                     6.46   7.01
  //    2000,  2000                                     5.17   5.30
  const uint32_t n = a->requests;
  if (n <= 256) queue(op_page_plan_held<256, 1>, 256);
  else if (n <= 512) queue(op_page_plan_held<256, 2>, 256);
  else if (n <= 1024) queue(op_page_plan_held<512, 2>, 512);
  else if (n <= 2048) queue(op_page_plan_held<512, 4>, 512);
  else queue(op_page_plan, FK_PLAN_THREADS);
  return launched(ctx, "fk_page_plan");
}

extern "C" int fk_paged_store(fk_ctx *ctx, const fk_paged_store_args *a, fk_stream *stream) {
  if (int st = admit(ctx, "fk_paged_store", a, stream)) return st;
  if (a->tokens == 0) return FK_OK;
  const uint64_t units = store_units(*a) * a->tokens;
  const dim3 grid((uint32_t)((units + FK_STORE_THREADS - 1) / FK_STORE_THREADS)), block(FK_STORE_THREADS);
  const hipStream_t s = stream_of(ctx, stream);
#define FK_STORE_CASE(T_)                                                                                 \
  case T_:                                                                                                \
    if (a->cache_bf16) hipLaunchKernelGGL((op_paged_store<T_, true>), grid, block, 0, s, *a);             \
    else hipLaunchKernelGGL((op_paged_store<T_, false>), grid, block, 0, s, *a);                          \
    break
  switch (a->rows_type) {
    FK_STORE_CASE(FK_T_F32);
    FK_STORE_CASE(FK_T_F16);
    FK_STORE_CASE(FK_T_BF16);
  }
#undef FK_STORE_CASE
  return launched(ctx, "fk_paged_store");
}

extern "C" size_t fk_paged_attend_workspace(const fk_paged_attend_args *a) {
  return a ? attend_bytes(*a, attend_launch(*a)) : 0;
}

extern "C" const char *fk_paged_attend_form(const fk_paged_attend_args *a) {
  const AttendLaunch l = a ? attend_launch(*a) : AttendLaunch{};
  return l.groups == 0 ? "" : (!l.plan.whole ? "split" : (l.waves == 8 ? "whole 8" : "whole 4"));
}

extern "C" int fk_paged_attend(fk_ctx *ctx, const fk_paged_attend_args *a, fk_stream *stream) {
  const AttendLaunch l = a ? attend_launch(*a) : AttendLaunch{};
  if (int st = admit(ctx, "fk_paged_attend", a, stream, l)) return st;
  const hipStream_t s = stream_of(ctx, stream);
  if (a->cache_bf16) queue_attend<true>(*a, l, s);
  else queue_attend<false>(*a, l, s);
  if (int st = launched(ctx, "fk_paged_attend")) return st;
  if (l.plan.whole) return FK_OK;
  const uint32_t states = l.groups / l.joins;  // of a pair, about
  if (states >= 8) queue_join<8>(*a, l, s);
  else if (states >= 4) queue_join<4>(*a, l, s);
  else queue_join<2>(*a, l, s);
  return launched(ctx, "fk_paged_attend (join)");
}
