// fk_paged8.hip — the operators over 8-bit paged caches as one C call each
// (include/fkrocm_paged8.h), their kernels compiled into the C ABI's library.

#include "../../include/fkrocm_paged8.h"

#include <hip/hip_runtime.h>

#include "fk_admit.h"
#include "kernels/fk_paged8.h"
#include "kernels/fk_paged_attend8.h"

using fk::admit;
using fk::launched;
using fk::of_type;
using fk::Refusal;
using fk::Span;
using fk::stream_of;

namespace {

template <int T, bool BF16, uint32_t W>
__global__ void __launch_bounds__(W == 1 ? 256 : 64 * W) op_pages8_store(fk_paged_store8_args a, fk::Store8Plan pl) {
  fk::paged_store8<T, BF16, W>(a, pl);
}

template <int T>
__global__ void __launch_bounds__(FK_LOAD8_THREADS)
    op_pages8_load(fk_paged_load8_args a, fk::Divisor block, fk::Divisor units) {
  fk::paged_load8<T>(a, block, units);
}

template <uint32_t DP, uint32_t EIGHTS, bool FULL, bool BF16>
__global__ void __launch_bounds__(64 * FK_PAGED_WAVES, DP == 256 ? 1 : 2)
    op_pages8_attend(fk_paged_attend_args a, uint64_t scales, fk::PagedPlan pl) {
  fk::paged_attend8<DP, EIGHTS, FULL, BF16>(a, scales, pl);
}

template <uint32_t W, bool BF16>
__global__ void __launch_bounds__(64 * W)
    op_pages8_join(fk_paged_attend_args a, fk::PagedPlan pl, uint32_t groups) {
  fk::paged_attend_join<W, BF16>(a, pl, groups);
}

// The store's launch: the wavefronts of a run, threadgroups of runs and in all
// (0: past a launch's 2^32 threads), the chunk.
struct StoreLaunch {
  uint32_t waves = 1, threads = 256;
  uint64_t groups = 0;
  fk::Store8Plan plan{};
};

StoreLaunch store_launch(const fk_paged_store8_args &a) {
  StoreLaunch l;
  // as many wavefronts as hold a whole block's rows, a piece of 8 and 8 elements a thread
  const uint64_t pieces = (uint64_t)a.block_size * a.head_dim / 16;
  l.waves = pieces <= 64 ? 1 : (pieces <= 128 ? 2 : (pieces <= 256 ? 4 : 8));
  l.threads = l.waves == 1 ? 256 : 64 * l.waves;
  const uint64_t T = a.tokens, units = 2ull * a.kv_heads, most = 8192 / l.waves;
  // a token a chunk while that is what fills the chip
  const uint64_t chunk = T * units / most;
  l.plan.chunk = (uint32_t)(chunk < 1 ? 1 : (chunk > 64 ? 64 : chunk));
  l.plan.block = fk::divisor(a.block_size);
  const uint64_t runs = (T + l.plan.chunk - 1) / l.plan.chunk * units;
  const uint64_t kv_groups = l.waves == 1 ? (runs + 3) / 4 : runs;
  const uint64_t queries = a.q ? T * a.heads * (a.head_dim / 16) : 0;
  l.groups = kv_groups + (queries + l.threads - 1) / l.threads;
  if ((__uint128_t)T * a.heads * (a.head_dim / 16) >= 1ull << 31 || l.groups * l.threads >= 1ull << 32) l.groups = 0;
  l.plan.kv_groups = (uint32_t)kv_groups;
  return l;
}

// The attention's launch, as fk_serve.hip's: head_dim's tile width, its
// threadgroups, the joins' entries and what the kernels take; 0
// threadgroups and the reason if the kernels do not take them.
struct AttendLaunch {
  uint32_t width = 0, groups = 0, joins = 0;
  fk::PagedPlan plan{};
  const char *why = "";
};

AttendLaunch attend_launch(const fk_paged_attend8_args &a) {
  AttendLaunch l;
  const uint64_t length = (uint64_t)a.table_len * a.block_size;
  if (a.requests == 0 || a.kv_heads == 0 || a.heads == 0 || a.heads % a.kv_heads) {
    l.why = "requests and heads that kv_heads divides";
  } else if (a.head_dim == 0 || a.head_dim % 16 || a.head_dim > 256) {
    l.why = "head_dim a multiple of 16, at most 256";
  } else if (a.block_size == 0 || a.block_size % 8 || a.blocks == 0 || a.table_len == 0) {
    l.why = "blocks of a multiple of 8 positions, and a table";
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
    // Threadgroups: one a CU of heads past 128 (more registers) and of few pairs
    // (whose states are then fewer to join), two, or three of heads of 64, whose
    // tiles cost more operations a byte.  µs by 1, 2 and 3 a CU: one request of
    // 131072 keys, 8 pairs of 128, 46.5 48.1 53.7; 512 pairs of 128 and up to
    // 16384 129.1 130.9 130.1, of 64 84.8 78.2 75.2; 128 of 256 74.7 81.1 80.9; 160
    // of 128 and up to 3000 23.8 21.2 23.2.
    const uint64_t pairs = (uint64_t)a.requests * a.kv_heads * l.plan.head_tiles;
    const uint64_t most = l.width == 64 ? 768 : (l.width == 256 || pairs <= 16 ? 256 : 512);
    l.groups = (uint32_t)(units < most ? (uint64_t)units : most);
    l.plan.by_pair = pairs <= l.groups;
    l.joins = l.plan.by_pair ? (uint32_t)pairs : l.groups;
    // Few units a pair at most: a threadgroup takes pairs whole, which saves the
    // prefix sum and the join and costs each further unit's time, and a long
    // pair's to the launch.  µs (by two parts of a probability; three take 0.1 to 0.3
    // more) whole and split of requests of up to u units (256
    // keys of 64, 128 of 128 and 256), evenly spread | of one unit but for one:
    //   pairs, width   u = 4                  6                      8                      12
    //     8 of 64    7.6  9.5              9.5  9.5             11.4  9.7             15.2  9.9
    //    80 of 64    8.7 12.4| 8.1 10.3   10.5 12.6|10.0 10.2   12.3 13.3|12.0 10.4   16.1 13.6|15.5 10.5
    //   328 of 64   13.3 16.8| 9.0 11.9   15.2 19.5|11.0 12.0   18.1 19.8|12.3 12.0   27.7 24.9|15.9 12.2
    //     8 of 128   7.1  9.8              8.5  9.8              9.8 10.2             12.5 10.1
    //    80 of 128   7.6 12.2| 7.2 10.0    8.9 12.6| 8.8 10.0   10.3 13.0| 9.9 10.0   13.1 13.3|12.7 10.2
    //   328 of 128  12.6 16.7| 8.3 11.9   14.0 21.8|10.2 11.7   16.7 19.7|10.8 11.9   24.0 26.0|12.9 12.1
    //     8 of 256  12.0 12.8             14.6 12.8             17.3 13.1             21.8 13.2
    //    80 of 256  12.8 18.0|12.1 12.7   15.6 19.0|14.8 12.9   18.1 20.3|17.2 12.8   23.2 20.8|22.2 13.2
    //   328 of 256  24.6 32.4|17.4 19.4   27.5 37.8|21.4 19.5   31.7 43.8|22.4 19.5   45.0 48.2|27.2 19.8
    const uint64_t each = (seen + unit - 1) / unit;
    l.plan.whole = each <= (l.width == 64 ? (pairs < 64 ? 6 : 8)
                            : l.width == 128 ? (pairs < 128 ? 8 : 12) : (pairs < 64 ? 4 : 6));
    if (l.plan.whole) l.groups = (uint32_t)(pairs < most ? pairs : most);
  }
  return l;
}

size_t attend_bytes(const fk_paged_attend8_args &a, const AttendLaunch &l) {
  return l.groups * (sizeof(fk::u32x4) + 2 * (size_t)l.plan.rows * (a.head_dim + 2) * sizeof(float));
}

// The call's arguments as the kernels that both attentions share take them.
fk_paged_attend_args shared_args(const fk_paged_attend8_args &a) {
  fk_paged_attend_args s{};
  s.q = a.q, s.kpool = a.kpool, s.vpool = a.vpool, s.table = a.table, s.lengths = a.lengths, s.starts = a.starts;
  s.out = a.out, s.workspace = a.workspace, s.workspace_bytes = a.workspace_bytes;
  s.q_stride = a.q_stride, s.out_stride = a.out_stride;
  s.requests = a.requests, s.heads = a.heads, s.kv_heads = a.kv_heads, s.head_dim = a.head_dim;
  s.block_size = a.block_size, s.blocks = a.blocks, s.table_len = a.table_len, s.window = a.window;
  s.q_rows = a.q_rows, s.cache_bf16 = a.q_bf16, s.out_f32 = a.out_f32, s.scale = a.scale;
  return s;
}

// The keys of a group: a tile's where blocks are of whole tiles, 16, or 8 (and
// heads that do not fill their tiles).
template <uint32_t DP, bool BF16>
void queue_attend(const fk_paged_attend_args &a, uint64_t scales, const AttendLaunch &l, hipStream_t s) {
  constexpr uint32_t tile = fk::attend8_keys(DP);
  auto queue = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(l.groups), dim3(64 * FK_PAGED_WAVES), 0, s, a, scales, l.plan);
  };
  if (a.head_dim != DP || a.block_size % 16) queue(op_pages8_attend<DP, 1, false, BF16>);
  else if (a.block_size % tile) queue(op_pages8_attend<DP, 2, true, BF16>);
  else queue(op_pages8_attend<DP, tile / 8, true, BF16>);
}

template <bool BF16>
void queue_attend(const fk_paged_attend_args &a, uint64_t scales, const AttendLaunch &l, hipStream_t s) {
  if (l.width == 256) queue_attend<256, BF16>(a, scales, l, s);
  else if (l.width == 128) queue_attend<128, BF16>(a, scales, l, s);
  else queue_attend<64, BF16>(a, scales, l, s);
}

template <uint32_t W>
void queue_join(const fk_paged_attend_args &a, const AttendLaunch &l, hipStream_t s) {
  const dim3 grid(l.joins * l.plan.rows), block(64 * W);
  if (a.cache_bf16) hipLaunchKernelGGL((op_pages8_join<W, true>), grid, block, 0, s, a, l.plan, l.groups);
  else hipLaunchKernelGGL((op_pages8_join<W, false>), grid, block, 0, s, a, l.plan, l.groups);
}

// 8-bit pools, and their scales' bytes; 0 bytes and a refusal if there are none
// such.
struct Pools {
  uint64_t bytes = 0, scales = 0;
};
int check_pools(Refusal &no, uint32_t blocks, uint32_t block_size, uint32_t kv_heads, uint32_t head_dim, Pools &p) {
  if (kv_heads == 0 || head_dim == 0 || head_dim % 16 || head_dim > 256)
    return no(FK_ERR_ARG, "%u kv heads of width %u (a multiple of 16, at most 256)", kv_heads, head_dim);
  if (block_size == 0 || block_size % 8 || blocks == 0 || (uint64_t)blocks * block_size >= 1ull << 32)
    return no(FK_ERR_RANGE, "%u blocks of %u (a multiple of 8)", blocks, block_size);
  if ((uint64_t)kv_heads * head_dim >= 1ull << 31)
    return no(FK_ERR_RANGE, "%u kv heads of width %u: rows of 2^31 elements and more", kv_heads, head_dim);
  const __uint128_t pool = (__uint128_t)blocks * block_size * kv_heads * head_dim;
  if (pool >= 1ull << 48) return no(FK_ERR_RANGE, "a pool of 2^48 bytes and more");
  p.bytes = (uint64_t)pool;
  p.scales = 8ull * blocks * kv_heads;  // (no more than the pool's bytes)
  return FK_OK;
}

// Row strides that a call's 16-byte pieces take.
int check_stride(Refusal &no, const char *name, uint64_t stride, uint64_t width, uint32_t type) {
  if (stride < width || stride % (16 / fk::type_bytes(type)) || stride >= 1ull << 40)
    return no(FK_ERR_ARG, "%s's rows of %llu, %llu apart: at least a row, a multiple of 16 bytes", name,
              (unsigned long long)width, (unsigned long long)stride);
  return FK_OK;
}

}  // namespace

namespace fk {

int check(const fk_paged_store8_args &a, Refusal &no) {
  Pools p;
  if (int st = check_pools(no, a.blocks, a.block_size, a.kv_heads, a.head_dim, p)) return st;
  if (a.q && a.heads == 0) return no(FK_ERR_ARG, "queries of no heads");
  if (a.rows_type > FK_T_BF16) return no(FK_ERR_ARG, "rows of type %u", a.rows_type);
  if (2ull * a.rotated > a.head_dim || (a.rotated && a.rope_rows == 0))
    return no(FK_ERR_ARG, "RoPE of %u pairs of a head of %u from a table of %u rows", a.rotated, a.head_dim,
              a.rope_rows);
  const uint64_t T = a.tokens, wide = type_bytes(a.rows_type);
  const uint64_t qw = a.q ? (uint64_t)a.heads * a.head_dim : 0, kw = (uint64_t)a.kv_heads * a.head_dim;
  if (qw >= 1ull << 31) return no(FK_ERR_RANGE, "%u heads of width %u: 2^31 elements and more", a.heads, a.head_dim);
  if (a.q)
    if (int st = check_stride(no, "q", a.q_stride, qw, a.rows_type)) return st;
  if (int st = check_stride(no, "k", a.k_stride, kw, a.rows_type)) return st;
  if (int st = check_stride(no, "v", a.v_stride, kw, a.rows_type)) return st;
  if (T && store_launch(a).groups == 0)
    return no(FK_ERR_RANGE, "%u tokens of %u and %u heads of width %u: past 32 bits", a.tokens, a.q ? a.heads : 0,
              a.kv_heads, a.head_dim);
  const Span reads[] = {{"q", a.q, a.q ? rows_span(T, a.q_stride, qw, wide) : 0},
                        {"k", a.k, rows_span(T, a.k_stride, kw, wide)},
                        {"v", a.v, rows_span(T, a.v_stride, kw, wide)},
                        {"slots", a.slots, 4 * T, 4},
                        {"positions", a.positions, a.rotated ? 4 * T : 0, 4},
                        {"rope", a.rope, a.rotated ? 8ull * a.rope_rows * a.rotated : 0}};
  const Span writes[] = {{"qr", a.qr, T * qw * 2},
                         {"kpool", a.kpool, p.bytes},
                         {"vpool", a.vpool, p.bytes},
                         {"scales", a.scales, p.scales, 8}};
  return check_spans(no, reads, 6, writes, 4);
}

// Threads of a load: 8 elements each.
static uint64_t load_units(const fk_paged_load8_args &a) { return 2ull * a.kv_heads * (a.head_dim / 8); }

int check(const fk_paged_load8_args &a, Refusal &no) {
  Pools p;
  if (int st = check_pools(no, a.blocks, a.block_size, a.kv_heads, a.head_dim, p)) return st;
  if (a.rows_type > FK_T_BF16) return no(FK_ERR_ARG, "rows of type %u", a.rows_type);
  const uint64_t T = a.tokens, wide = type_bytes(a.rows_type), kw = (uint64_t)a.kv_heads * a.head_dim;
  if (int st = check_stride(no, "k", a.k_stride, kw, a.rows_type)) return st;
  if (int st = check_stride(no, "v", a.v_stride, kw, a.rows_type)) return st;
  if ((__uint128_t)load_units(a) * T >= (1ull << 32) - FK_LOAD8_THREADS)
    return no(FK_ERR_RANGE, "%u tokens of %u kv heads of width %u: past 32 bits", a.tokens, a.kv_heads, a.head_dim);
  const Span reads[] = {{"slots", a.slots, 4 * T, 4},
                        {"kpool", a.kpool, p.bytes},
                        {"vpool", a.vpool, p.bytes},
                        {"scales", a.scales, p.scales, 8}};
  const Span writes[] = {{"k", a.k, rows_span(T, a.k_stride, kw, wide)}, {"v", a.v, rows_span(T, a.v_stride, kw, wide)}};
  return check_spans(no, reads, 4, writes, 2);
}

int check(const fk_paged_attend8_args &a, Refusal &no) {
  const AttendLaunch l = attend_launch(a);
  if (l.groups == 0)
    return no(FK_ERR_ARG, "%u requests, %u heads over %u of width %u, %u blocks of %u, tables of %u: it takes %s",
              a.requests, a.heads, a.kv_heads, a.head_dim, a.blocks, a.block_size, a.table_len, l.why);
  Pools p;
  if (int st = check_pools(no, a.blocks, a.block_size, a.kv_heads, a.head_dim, p)) return st;
  const uint64_t n = a.requests, w = (uint64_t)a.heads * a.head_dim, most = 1ull << 38;
  if (a.q_stride < w || a.q_stride % 8 || a.q_stride >= most || a.out_stride < w || a.out_stride >= most)
    return no(FK_ERR_ARG, "row strides %llu and %llu: at least %llu, q's a multiple of 8",
              (unsigned long long)a.q_stride, (unsigned long long)a.out_stride, (unsigned long long)w);
  const size_t bytes = attend_bytes(a, l);
  if (a.workspace_bytes < bytes)
    return no(FK_ERR_RANGE, "a workspace of %llu bytes, %zu needed", (unsigned long long)a.workspace_bytes, bytes);
  if (a.starts && a.q_rows == 0) return no(FK_ERR_ARG, "starts of no rows of q");
  const uint64_t q_rows = a.starts ? a.q_rows : n;
  const Span reads[] = {{"q", a.q, rows_span(q_rows, a.q_stride, w, 2)},
                        {"kpool", a.kpool, p.bytes},
                        {"vpool", a.vpool, p.bytes},
                        {"scales", a.scales, p.scales, 8},
                        {"table", a.table, 4 * n * a.table_len, 4},
                        {"lengths", a.lengths, 4 * n, 4},
                        {"starts", a.starts, a.starts ? 4 * (n + 1) : 0, 4}};
  const Span writes[] = {{"out", a.out, rows_span(n, a.out_stride, w, a.out_f32 ? 4 : 2)},
                         {"workspace", a.workspace, bytes}};
  return check_spans(no, reads, 7, writes, 2);
}

}  // namespace fk

extern "C" int fk_paged_store8(fk_ctx *ctx, const fk_paged_store8_args *a, fk_stream *stream) {
  if (int st = admit(ctx, "fk_paged_store8", a, stream)) return st;
  if (a->tokens == 0) return FK_OK;
  const StoreLaunch l = store_launch(*a);
  const dim3 grid((uint32_t)l.groups), block(l.threads);
  const hipStream_t s = stream_of(ctx, stream);
  of_type(a->rows_type, [&](auto t) {
    constexpr int T = decltype(t)::value;
    auto queue = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, block, 0, s, *a, l.plan); };
    if (l.waves == 1) a->q_bf16 ? queue(op_pages8_store<T, true, 1>) : queue(op_pages8_store<T, false, 1>);
    else if (l.waves == 2) a->q_bf16 ? queue(op_pages8_store<T, true, 2>) : queue(op_pages8_store<T, false, 2>);
    else if (l.waves == 4) a->q_bf16 ? queue(op_pages8_store<T, true, 4>) : queue(op_pages8_store<T, false, 4>);
    else a->q_bf16 ? queue(op_pages8_store<T, true, 8>) : queue(op_pages8_store<T, false, 8>);
  });
  return launched(ctx, "fk_paged_store8");
}

extern "C" int fk_paged_load8(fk_ctx *ctx, const fk_paged_load8_args *a, fk_stream *stream) {
  if (int st = admit(ctx, "fk_paged_load8", a, stream)) return st;
  if (a->tokens == 0) return FK_OK;
  const uint64_t units = fk::load_units(*a), n = units * a->tokens;
  const dim3 grid((uint32_t)((n + FK_LOAD8_THREADS - 1) / FK_LOAD8_THREADS)), block(FK_LOAD8_THREADS);
  of_type(a->rows_type, [&](auto t) {
    hipLaunchKernelGGL((op_pages8_load<decltype(t)::value>), grid, block, 0, stream_of(ctx, stream), *a,
                       fk::divisor(a->block_size), fk::divisor((uint32_t)units));
  });
  return launched(ctx, "fk_paged_load8");
}

extern "C" size_t fk_paged_attend8_workspace(const fk_paged_attend8_args *a) {
  return a ? attend_bytes(*a, attend_launch(*a)) : 0;
}

extern "C" const char *fk_paged_attend8_form(const fk_paged_attend8_args *a) {
  const AttendLaunch l = a ? attend_launch(*a) : AttendLaunch{};
  return l.groups == 0 ? "" : (l.plan.whole ? "whole" : "split");
}

extern "C" int fk_paged_attend8(fk_ctx *ctx, const fk_paged_attend8_args *a, fk_stream *stream) {
  if (int st = admit(ctx, "fk_paged_attend8", a, stream)) return st;
  const AttendLaunch l = attend_launch(*a);
  const fk_paged_attend_args s = shared_args(*a);
  const hipStream_t on = stream_of(ctx, stream);
  a->q_bf16 ? queue_attend<true>(s, a->scales, l, on) : queue_attend<false>(s, a->scales, l, on);
  if (int st = launched(ctx, "fk_paged_attend8")) return st;
  if (l.plan.whole) return FK_OK;
  const uint32_t states = l.groups / l.joins;  // of a pair, about
  if (states >= 8) queue_join<8>(s, l, on);
  else if (states >= 4) queue_join<4>(s, l, on);
  else queue_join<2>(s, l, on);
  return launched(ctx, "fk_paged_attend8 (join)");
}
