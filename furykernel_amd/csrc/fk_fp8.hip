// fk_fp8.hip — the 8-bit matrices' operators as one C call each
// (include/fkrocm_fp8.h), their kernels compiled into the C ABI's library.

#include "../../include/fkrocm_fp8.h"

#include <hip/hip_runtime.h>

#include <cmath>
#include <iterator>
#include <utility>

#include "fk_admit.h"
#include "kernels/fk_fp8.h"
#include "kernels/fk_fp8_gemm.h"

using fk::admit;
using fk::check_rows;
using fk::launched;
using fk::of_type;
using fk::Refusal;
using fk::rows_of;
using fk::Span;
using fk::stream_of;

namespace {

template <int T>
__global__ void __launch_bounds__(FK_FP8_THREADS) op_fp8_quantize(fk_fp8_quantize_args a) {
  fk::fp8_quantize<T>(a);
}

template <int T>
__global__ void __launch_bounds__(FK_FP8_THREADS) op_fp8_dequantize(fk_fp8_dequantize_args a) {
  fk::fp8_dequantize<T>(a);
}

// (two rows of 16 bits: registers for 8 wavefronts a SIMD, three threadgroups of ten)
template <int T, uint32_t ROWS, uint32_t H>
__global__ void __launch_bounds__(1024, ROWS == 2 && T != FK_T_F32 ? 8 : 1)
    op_fp8_add_norm(fk_fp8_add_norm_args a, double over_k) {
  fk::fp8_add_norm<T, ROWS, H>(a, over_k);
}

template <uint32_t MB, uint32_t NB, uint32_t W, int T, bool CUT>
__global__ void __launch_bounds__(64 * W, 2) op_fp8_gemm_few(fk_fp8_gemm_args a) {
  fk::fp8_gemm_few<MB, NB, W, T, CUT>(a);
}

template <uint32_t GM, uint32_t GN, uint32_t STAGES, int T, bool CUT>
__global__ void __launch_bounds__(256, STAGES == 3 ? 3 : 1) op_fp8_gemm_mid(fk_fp8_gemm_args a) {
  fk::fp8_gemm_mid<GM, GN, STAGES, T, CUT>(a);
}

// (whole and cut sums in one kernel, by its arguments)
template <int T>
__global__ void __launch_bounds__(256, 1) op_fp8_gemm_many(fk_fp8_gemm_args a) {
  if constexpr (T != FK_T_F32)
    if (a.c_type & FK_FP8_CUT_SUMS) return fk::fp8_gemm_many<T, true>(a);
  fk::fp8_gemm_many<T, false>(a);
}

uint64_t codes_bytes(uint32_t rows, uint32_t k) { return (uint64_t)fk::fp8_row_tiles(rows) * fk::fp8_blocks(k) * 2048; }
uint64_t scales_bytes(uint32_t rows, uint32_t k) { return (uint64_t)fk::fp8_row_tiles(rows) * fk::fp8_quads(k) * 64; }

// A matrix that one launch of a wavefront for each 16 rows of a block makes, in
// fewer than 2^32 threads of whole threadgroups (1.4 10^11 elements).
bool matrix(uint32_t rows, uint32_t k) {
  return rows > 0 && k > 0 && rows <= 1u << 30 && k <= 1u << 30 &&
         (uint64_t)fk::fp8_row_tiles(rows) * fk::fp8_blocks(k) < (1ull << 26) - 4;
}

// Threadgroups of a wavefront for each 16 rows of a block.
uint32_t block_groups(uint32_t rows, uint32_t k) {
  const uint64_t n = (uint64_t)fk::fp8_row_tiles(rows) * fk::fp8_blocks(k), w = FK_FP8_THREADS / FK_WAVE;
  return (uint32_t)((n + w - 1) / w);
}

// The norm's launch: rows a threadgroup, blocks a lane, and tiles of 16 rows by
// 8, one an XCD.  Where the rows fill the card, rows of up to 64 blocks go by two,
// with two blocks a lane (29631 x 533 f16 44 us, by one 75; 8191 x 5000 bf16 69 and
// 110; 8192 x 2048 f32 47 both); few rows, which wait on their own chain of steps, by
// one, with as few blocks a lane as there are threads for (1 x 5000 4.1 us with one
// block, 4.9 with two, 6.7 with four; by two rows 5.7).
constexpr uint32_t norm_most = 4 * 16 * FK_FP8_NORM_HELD * 128;
struct NormLaunch {
  uint32_t rows, held, threads, groups;
};
NormLaunch norm_launch(const fk_fp8_add_norm_args &a) {
  NormLaunch l;
  const uint32_t blocks = fk::fp8_blocks(a.k);
  l.rows = a.rows >= 1024 && blocks <= 64 ? 2 : 1;
  const uint32_t each = (blocks * l.rows + 3) / 4;  // blocks for the wavefronts' 16 lanes
  l.held = l.rows == 2 ? 2 : (each <= 16 ? 1 : (each <= 32 ? 2 : FK_FP8_NORM_HELD));
  l.threads = 64 * ((each + l.held - 1) / l.held);
  l.groups = (fk::fp8_row_tiles(a.rows) + 7) / 8 * (128 / l.rows);
  return l;
}

// The forms of the product: blocks of 16 of a threadgroup's tile, the
// wavefronts that share a tile's k (few), the stages of its ring (mid).
enum Kind { FEW, MID, MANY };
struct Form {
  const char *name;
  Kind kind;
  uint32_t mb, nb, by, stages;
  // of C of 16 bits with cut sums, of 16 bits, and of f32 (a base below 0: not that C)
  struct Cost {
    double base, step, turn, tile, work;
  } cost[3];
};
// What each costs, in µs, fitted to its times on 221 products (1 to 8192 rows by
// 512 to 16384, k of 512 to 8192, the operands from memory each time), then moved,
// each no further from its times than by 6 % of the fit's own misses, to where the
// least cost names the fastest form most often.  With `turns` the threadgroups of
// the CU that has most,
//   few         base, for each block of k a wavefront takes `step` and `turn` a
//               turn, `tile` a turn, and `work` for a thousand tiles of 2 KB that
//               all threadgroups read
//   mid, many   base, `tile` a turn, and for each block of k the largest of `step`
//               (its latency), `turn` a turn and `work` a threadgroup of each CU
// The form of the least cost takes 1.004, 1.003 and 1.003 times the fastest one's
// time on average over them, at most 1.13, 1.06 and 1.13; over some 90 others (3 to
// 6000 rows by 1000, 4096 and 12000, k of 1024 to 12288) 1.011, 1.006 and 1.005, at
// most 1.16, 1.09 and 1.16.  (Not of k below 512: at one or two blocks of it many
// 16x16 is named for some large C that mid 8x8 makes in 0.6 to 0.8 of the time.)
constexpr Form forms[] = {
    {"few 1x1", FEW, 1, 1, 8, 0,
     {{1.853, 0.397, 0.099, 0.093, 0.139}, {1.785, 0.313, 0.278, 0.154, 0.104}, {1.754, 0.219, 0.317, 0.208, 0.091}}},
    {"few 1x2", FEW, 1, 2, 8, 0,
     {{2.075, 0.191, 0.543, 0.096, 0.120}, {1.852, 0.457, 0.314, 0.32, 0.149}, {1.965, 0.292, 0.520, 0.257, 0.124}}},
    {"few 2x1", FEW, 2, 1, 8, 0,
     {{1.387, 0.513, 0.430, 0.211, 0.061}, {1.219, 0.432, 0.411, 0.504, 0.069}, {1.313, 0.390, 0.449, 0.369, 0.071}}},
    {"few 2x2", FEW, 2, 2, 8, 0,
     {{1.607, 0.315, 0.720, 0.292, 0.082}, {0.814, 0.422, 0.711, 1.382, 0.076}, {1.162, 0.436, 0.790, 1.052, 0.067}}},
    {"few 4x2", FEW, 4, 2, 4, 0,
     {{2.099, 0.056, 0.597, 0.494, 0.059}, {2.466, 0.049, 0.744, 0.472, 0.041}, {1.972, 0.014, 0.894, 0.997, 0}}},
    {"few 8x2", FEW, 8, 2, 8, 0,
     {{0.028, 0.332, 2.227, 1.728, 0.020}, {0.125, 0.393, 2.878, 1.871, 0.026}, {-1, 0, 0, 0, 0}}},
    {"few 4x3", FEW, 4, 3, 8, 0,
     {{0.410, 0.636, 1.366, 1.613, 0.048}, {0.197, 0.067, 1.926, 2.39, 0.035}, {0.154, 0.635, 0.967, 2.560, 0.103}}},
    {"few 4x4", FEW, 4, 4, 8, 0,
     {{0.124, 0.795, 1.188, 2.440, 0.083}, {0.113, 0.499, 1.602, 2.91, 0.084}, {0.184, 0.554, 1.837, 2.738, 0.071}}},
    {"mid 8x8", MID, 8, 8, 0, 3,
     {{0.258, 0.813, 0.553, 1.668, 0.169}, {1.326, 0.948, 0.782, 1.518, 0.858}, {0.324, 0.980, 0.722, 3.243, 0.795}}},
    {"mid 8x8 deep", MID, 8, 8, 0, 8,
     {{0.344, 0.358, 0.531, 3.591, 0.685}, {1.609, 0.059, 0.83, 3.167, 1.067}, {0.116, 0.213, 0.867, 5.308, 1.075}}},
    {"mid 4x8 deep", MID, 4, 8, 0, 10,
     {{1.102, 0.074, 0.415, 2.430, 0.559}, {0.91, 0.219, 0.551, 2.996, 0.698}, {1.293, 0.059, 0.531, 3.237, 0.761}}},
    {"many 16x16", MANY, 16, 16, 0, 0,
     {{0.058, 0.006, 1.172, 8.585, 1.594}, {0.537, 0.799, 2.483, 8.13, 2.829}, {0.129, 1.084, 2.401, 11.874, 3.147}}},
};

uint64_t tiles_of(const Form &f, uint32_t m, uint32_t n) {
  return (uint64_t)((fk::fp8_row_tiles(m) + f.mb - 1) / f.mb) * ((fk::fp8_row_tiles(n) + f.nb - 1) / f.nb);
}

// C's type, and which of a form's costs a product has.
constexpr uint32_t type_of(uint32_t c_type) { return c_type & ~FK_FP8_CUT_SUMS; }
constexpr bool is_cut(uint32_t c_type) { return c_type & FK_FP8_CUT_SUMS; }
constexpr bool is_c(uint32_t c_type) {
  return type_of(c_type) <= FK_T_BF16 && c_type != (FK_T_F32 | FK_FP8_CUT_SUMS);
}
constexpr uint32_t column(uint32_t c_type) { return c_type == FK_T_F32 ? 2 : (is_cut(c_type) ? 0 : 1); }

double cost(const Form &f, uint32_t m, uint32_t n, uint32_t k, uint32_t c_type) {
  const Form::Cost &c = f.cost[column(c_type)];
  const double t = (double)tiles_of(f, m, n), blocks = fk::fp8_blocks(k), turns = std::ceil(t / 256);
  const double ends = c.base + c.tile * turns;
  if (f.kind == FEW)
    return ends + std::ceil(blocks / f.by) * (c.step + c.turn * turns) + c.work * 1e-3 * t * blocks * (f.mb + f.nb);
  return ends + blocks * std::fmax(c.step, std::fmax(c.turn * turns, c.work * t / 256));
}

// mid and many address a tile's slab with 32 bits.
constexpr bool takes(const Form &f, uint32_t k, uint32_t c_type) {
  return f.cost[column(c_type)].base >= 0 && (f.kind == FEW || fk::fp8_blocks(k) < 1u << 16);
}

uint32_t pick(uint32_t m, uint32_t n, uint32_t k, uint32_t c_type) {
  uint32_t best = 0;
  for (uint32_t i = 1; i < std::size(forms); i++)
    if (takes(forms[i], k, c_type) && cost(forms[i], m, n, k, c_type) < cost(forms[best], m, n, k, c_type)) best = i;
  return best;
}

// Why the kernels do not take a product of these sizes; null if they do.
const char *refused(uint32_t m, uint32_t n, uint32_t k, uint32_t c_type) {
  if (!matrix(m, k) || !matrix(n, k)) return "no such matrices";
  if ((uint64_t)fk::fp8_row_tiles(m) * fk::fp8_row_tiles(n) >= 1ull << 31) return "2^31 tiles and more";
  const Form &f = forms[pick(m, n, k, c_type)];
  if (f.kind != MANY && tiles_of(f, m, n) >= 1ull << 23)  // a launch of 2^32 threads
    return "2^23 threadgroups and more";
  return nullptr;
}

template <uint32_t I, int T, bool CUT>
void queue_form(const fk_fp8_gemm_args &a, hipStream_t s) {
  constexpr Form f = forms[I];
  const uint32_t tiles = (uint32_t)tiles_of(f, a.m, a.n);
  if constexpr (f.kind == FEW && takes(f, 1, CUT ? T | FK_FP8_CUT_SUMS : T))
    hipLaunchKernelGGL((op_fp8_gemm_few<f.mb, f.nb, f.by, T, CUT>), dim3(tiles), dim3(64 * f.by), 0, s, a);
  else if constexpr (f.kind == MID)
    hipLaunchKernelGGL((op_fp8_gemm_mid<f.mb / 4, f.nb / 4, f.stages, T, CUT>), dim3(tiles), dim3(256),
                       (fk::fp8_mid_lds<f.mb / 4, f.nb / 4, f.stages>()), s, a);
  else if constexpr (f.kind == MANY)
    hipLaunchKernelGGL((op_fp8_gemm_many<T>), dim3(tiles < 256 ? tiles : 256), dim3(256), fk::fp8_many_lds, s, a);
}

template <int T, bool CUT, size_t... I>
void queue_picked(uint32_t form, const fk_fp8_gemm_args &a, hipStream_t s, std::index_sequence<I...>) {
  ((form == I ? queue_form<I, T, CUT>(a, s) : void()), ...);
}

template <int T, uint32_t ROWS, uint32_t H>
void queue_norm(const fk_fp8_add_norm_args &a, const NormLaunch &l, hipStream_t s) {
  hipLaunchKernelGGL((op_fp8_add_norm<T, ROWS, H>), dim3(l.groups), dim3(l.threads), 0, s, a, 1.0 / a.k);
}
}  // namespace

namespace fk {

int check(const fk_fp8_quantize_args &a, Refusal &no) {
  if (!matrix(a.rows, a.k)) return no(FK_ERR_RANGE, "no matrix of %u rows of %u", a.rows, a.k);
  if (int st = check_rows(no, "x", a.x_stride, a.k, a.x_type)) return st;
  const Span reads[] = {rows_of("x", a.x, a.rows, a.x_stride, a.k, a.x_type)};
  const Span writes[] = {{"codes", a.codes, codes_bytes(a.rows, a.k)}, {"scales", a.scales, scales_bytes(a.rows, a.k)}};
  return check_spans(no, reads, 1, writes, 2);
}

int check(const fk_fp8_dequantize_args &a, Refusal &no) {
  if (!matrix(a.rows, a.k)) return no(FK_ERR_RANGE, "no matrix of %u rows of %u", a.rows, a.k);
  if (int st = check_rows(no, "y", a.y_stride, a.k, a.y_type)) return st;
  const Span reads[] = {{"codes", a.codes, codes_bytes(a.rows, a.k)}, {"scales", a.scales, scales_bytes(a.rows, a.k)}};
  const Span writes[] = {rows_of("y", a.y, a.rows, a.y_stride, a.k, a.y_type),
                         {"scales_out", a.scales_out, a.scales_out ? 4ull * a.rows * fk::fp8_blocks(a.k) : 0, 4}};
  return check_spans(no, reads, 2, writes, 2);
}

int check(const fk_fp8_add_norm_args &a, Refusal &no) {
  if (!matrix(a.rows, a.k) || a.k > norm_most)
    return no(FK_ERR_RANGE, "no matrix of %u rows of %u (at most %u)", a.rows, a.k, norm_most);
  if (fk::fp8_row_tiles(a.rows) >= 1u << 18) return no(FK_ERR_RANGE, "%u rows: 2^22 and more", a.rows);
  const NormLaunch l = norm_launch(a);
  if ((uint64_t)l.groups * l.threads >= 1ull << 32)
    return no(FK_ERR_RANGE, "%u rows of %u: a launch of 2^32 threads", a.rows, a.k);
  if (!(a.eps >= 0.0f) || std::isinf(a.eps)) return no(FK_ERR_ARG, "eps = %g", (double)a.eps);
  if (int st = check_rows(no, "x", a.x_stride, a.k, a.x_type)) return st;
  if (a.residual)
    if (int st = check_rows(no, "residual", a.residual_stride, a.k, a.x_type)) return st;
  if (a.sum)
    if (int st = check_rows(no, "sum", a.sum_stride, a.k, a.x_type)) return st;
  // (over x or the residual, element by element, the sum is no overlap: each is
  // read by the thread that writes it, before; at their address but another stride
  // it is one)
  const bool over_x = a.sum == a.x && (a.rows == 1 || a.sum_stride == a.x_stride);
  const bool over_r = a.sum == a.residual && (a.rows == 1 || a.sum_stride == a.residual_stride);
  const Span x = rows_of("x", a.x, a.rows, a.x_stride, a.k, a.x_type);
  const Span r = rows_of("residual", a.residual, a.residual ? a.rows : 0, a.residual_stride, a.k, a.x_type);
  const Span sum = rows_of("sum", a.sum, a.sum ? a.rows : 0, a.sum_stride, a.k, a.x_type);
  const Span gamma = {"gamma", a.gamma, a.gamma ? 4ull * a.k : 0};
  const Span codes = {"codes", a.codes, codes_bytes(a.rows, a.k)};
  const Span scales = {"scales", a.scales, scales_bytes(a.rows, a.k)};
  {
    const Span reads[] = {x, r, gamma}, writes[] = {codes, scales};
    if (int st = check_spans(no, reads, 3, writes, 2)) return st;
  }
  Span reads[5] = {codes, scales, gamma};
  size_t n = 3;
  if (!over_x) reads[n++] = x;
  if (!over_r) reads[n++] = r;
  const Span one[] = {sum};
  return check_spans(no, reads, n, one, 1);
}

int check(const fk_fp8_gemm_args &a, Refusal &no) {
  const uint32_t type = type_of(a.c_type);
  if (!is_c(a.c_type)) return no(FK_ERR_ARG, "c of type %#x", a.c_type);
  if (const char *why = refused(a.m, a.n, a.k, a.c_type))
    return no(FK_ERR_RANGE, "a product of %u by %u rows of %u: %s", a.m, a.n, a.k, why);
  if (int st = check_rows(no, "c", a.c_stride, a.n, type)) return st;
  const Span reads[] = {{"a_codes", a.a_codes, codes_bytes(a.m, a.k)},
                        {"a_scales", a.a_scales, scales_bytes(a.m, a.k)},
                        {"b_codes", a.b_codes, codes_bytes(a.n, a.k)},
                        {"b_scales", a.b_scales, scales_bytes(a.n, a.k)}};
  const Span writes[] = {rows_of("c", a.c, a.m, a.c_stride, a.n, type)};
  return check_spans(no, reads, 4, writes, 1);
}

}  // namespace fk

extern "C" size_t fk_fp8_codes_bytes(uint32_t rows, uint32_t k) { return matrix(rows, k) ? codes_bytes(rows, k) : 0; }
extern "C" size_t fk_fp8_scales_bytes(uint32_t rows, uint32_t k) { return matrix(rows, k) ? scales_bytes(rows, k) : 0; }

extern "C" int fk_fp8_quantize(fk_ctx *ctx, const fk_fp8_quantize_args *a, fk_stream *stream) {
  if (int st = admit(ctx, "fk_fp8_quantize", a, stream)) return st;
  const dim3 grid(block_groups(a->rows, a->k)), block(FK_FP8_THREADS);
  of_type(a->x_type, [&](auto t) {
    hipLaunchKernelGGL((op_fp8_quantize<decltype(t)::value>), grid, block, 0, stream_of(ctx, stream), *a);
  });
  return launched(ctx, "fk_fp8_quantize");
}

extern "C" int fk_fp8_dequantize(fk_ctx *ctx, const fk_fp8_dequantize_args *a, fk_stream *stream) {
  if (int st = admit(ctx, "fk_fp8_dequantize", a, stream)) return st;
  const dim3 grid(block_groups(a->rows, a->k)), block(FK_FP8_THREADS);
  of_type(a->y_type, [&](auto t) {
    hipLaunchKernelGGL((op_fp8_dequantize<decltype(t)::value>), grid, block, 0, stream_of(ctx, stream), *a);
  });
  return launched(ctx, "fk_fp8_dequantize");
}

extern "C" int fk_fp8_add_norm(fk_ctx *ctx, const fk_fp8_add_norm_args *a, fk_stream *stream) {
  if (int st = admit(ctx, "fk_fp8_add_norm", a, stream)) return st;
  const NormLaunch l = norm_launch(*a);
  const hipStream_t s = stream_of(ctx, stream);
  of_type(a->x_type, [&](auto t) {
    constexpr int T = decltype(t)::value;
    if (l.rows == 2) queue_norm<T, 2, 2>(*a, l, s);
    else if (l.held == 1) queue_norm<T, 1, 1>(*a, l, s);
    else if (l.held == 2) queue_norm<T, 1, 2>(*a, l, s);
    else queue_norm<T, 1, FK_FP8_NORM_HELD>(*a, l, s);
  });
  return launched(ctx, "fk_fp8_add_norm");
}

extern "C" const char *fk_fp8_gemm_form(uint32_t m, uint32_t n, uint32_t k, uint32_t c_type) {
  return !is_c(c_type) || refused(m, n, k, c_type) ? "" : forms[pick(m, n, k, c_type)].name;
}

extern "C" int fk_fp8_gemm(fk_ctx *ctx, const fk_fp8_gemm_args *a, fk_stream *stream) {
  if (int st = admit(ctx, "fk_fp8_gemm", a, stream)) return st;
  const hipStream_t s = stream_of(ctx, stream);
  const uint32_t form = pick(a->m, a->n, a->k, a->c_type);
  constexpr auto all = std::make_index_sequence<std::size(forms)>{};
  of_type(type_of(a->c_type), [&](auto t) {
    constexpr int T = decltype(t)::value;
    if constexpr (T == FK_T_F32) queue_picked<T, false>(form, *a, s, all);
    else if (is_cut(a->c_type)) queue_picked<T, true>(form, *a, s, all);
    else queue_picked<T, false>(form, *a, s, all);
  });
  return launched(ctx, "fk_fp8_gemm");
}
