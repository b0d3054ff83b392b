// fk_mx4.hip — the 4-bit microscaled matrices' operators as one C call each
// (include/fkrocm_mx4.h), their kernels compiled into the C ABI's library.

#include "../../include/fkrocm_mx4.h"

#include <hip/hip_runtime.h>

#include <cmath>
#include <iterator>
#include <utility>

#include "fk_admit.h"
#include "kernels/fk_mx4.h"
#include "kernels/fk_mx4_gemm.h"

using fk::admit;
using fk::launched;
using fk::Refusal;
using fk::Span;
using fk::stream_of;

namespace {

template <int T, bool ONCE>
__global__ void __launch_bounds__(FK_MX4_THREADS) op_mx4_quantize(fk_mx4_quantize_args a) {
  fk::mx4_quantize<T, ONCE>(a);
}

template <int T>
__global__ void __launch_bounds__(FK_MX4_THREADS) op_mx4_dequantize(fk_mx4_dequantize_args a) {
  fk::mx4_dequantize<T>(a);
}

// (two wavefronts a SIMD: 8 x 2 with two pairs in flight would take one's
// registers and its CU alone; 200 rows by 8192, k 2048 8.7 µs, so 7.0)
template <uint32_t MB, uint32_t NB, uint32_t W, int T>
__global__ void __launch_bounds__(64 * W, 2) op_mx4_gemm_few(fk_mx4_gemm_args a) {
  fk::mx4_gemm_few<MB, NB, W, T>(a);
}

template <int T>
__global__ void __launch_bounds__(256, 1) op_mx4_gemm_many(fk_mx4_gemm_args a) {
  fk::mx4_gemm_many<T>(a);
}

template <uint32_t GM, uint32_t GN, int T>
__global__ void __launch_bounds__(256, 3) op_mx4_gemm_mid(fk_mx4_gemm_args a) {
  fk::mx4_gemm_mid<GM, GN, T>(a);
}

uint64_t codes_bytes(uint32_t rows, uint32_t k) { return (uint64_t)fk::mx4_row_tiles(rows) * fk::mx4_pairs(k) * 2048; }
uint64_t scales_bytes(uint32_t rows, uint32_t k) { return (uint64_t)fk::mx4_row_tiles(rows) * fk::mx4_pairs(k) * 128; }

// A matrix that one launch of a wavefront a tile makes: fewer than 2^25 - 1 pairs
// of tiles (1.4 10^11 elements), 2^32 threads in whole threadgroups.
bool matrix(uint32_t rows, uint32_t k) {
  return rows > 0 && k > 0 && rows <= 1u << 30 && k <= 1u << 30 &&
         (uint64_t)fk::mx4_row_tiles(rows) * fk::mx4_pairs(k) < (1ull << 25) - 1;
}

// Rows of `type`, `stride` elements apart, aligned to their elements.
int check_rows(Refusal &no, const char *name, uint64_t stride, uint64_t width, uint32_t type) {
  if (type > FK_T_BF16) return no(FK_ERR_ARG, "%s of type %u", name, type);
  if (stride < width || stride >= 1ull << 40)
    return no(FK_ERR_ARG, "%s's rows of %llu, %llu apart", name, (unsigned long long)width, (unsigned long long)stride);
  return FK_OK;
}
Span rows_of(const char *name, uint64_t addr, uint64_t rows, uint64_t stride, uint64_t width, uint32_t type) {
  const uint32_t bytes = fk::mx4_bytes_of((int)type);
  return {name, addr, fk::rows_span(rows, stride, width, bytes), bytes};
}

// Threadgroups of a wavefront a tile.
uint32_t tile_groups(uint32_t rows, uint32_t k) {
  const uint64_t tiles = 2ull * fk::mx4_row_tiles(rows) * fk::mx4_pairs(k), w = FK_MX4_THREADS / FK_WAVE;
  return (uint32_t)((tiles + w - 1) / w);
}

// Rows that pass the caches by: many, and in whole 16 bytes.  µs plain and so,
// out of memory each time, and with the codes read back behind it: 100 x 3080
// bf16 3.7 4.0, 512 x 2048 3.8 4.5; 1024 x 4096 5.4 5.4, 4.8 4.6; 4096 x 4096
// 11.0 10.1, 10.7 9.4; 8192 x 8192 35.3 33.0, 34.2 30.6, f32 58.3 56.9, 68.2
// 56.8; rows of 8191 48.4 50.1.
bool passes_by(const fk_mx4_quantize_args &a) {
  const uint64_t bytes = fk::mx4_bytes_of((int)a.x_type);
  return (uint64_t)a.rows * a.k * bytes >= 1ull << 23 && a.x % 16 == 0 && a.x_stride * bytes % 16 == 0;
}

template <typename F>
void of_type(uint32_t type, F &&f) {
  if (type == FK_T_F32) f(std::integral_constant<int, FK_T_F32>{});
  else if (type == FK_T_F16) f(std::integral_constant<int, FK_T_F16>{});
  else f(std::integral_constant<int, FK_T_BF16>{});
}

// The forms of the product: blocks of 16 of a threadgroup's tile, the
// wavefronts that share a tile's k (few) or the threadgroups the chip holds at
// once (mid, many).
enum Kind { FEW, MID, MANY };
struct Form {
  const char *name;
  Kind kind;
  uint32_t mb, nb, by;
  double base, step, turn, work;
};
// What each costs, in µs, fitted to its times on 229 products (1 to 8192 rows
// by 512 to 16384, k of 2048 to 8192, the operands from memory each time):
//   few         base, for each pair of tiles of k a wavefront takes `step` and
//               `turn` for every threadgroup of its CU, and `work` for a
//               thousand KB that all threadgroups read (mb + nb blocks a pair
//               each: what a tile reads again, others read too)
//   mid, many   `step` a pair, `work` for 10^5 blocks times pairs, and `base`
//               for every time the tiles fill the chip
// The form of the least cost takes 1.003 times the fastest one's time on
// average over them, at most 1.18 (512 rows by 5000, k 2048: 14.6 µs, mid
// 12.4).  Between 64 x 16 and 128 x 32 blocks, 32 x 32 ones would be 0.5 %
// faster on average.
constexpr Form forms[] = {
    {"few 1x1", FEW, 1, 1, 8, 2.598, 0.129, 0.091, 0.160}, {"few 4x1", FEW, 4, 1, 8, 2.587, 0.182, 0.512, 0.074},
    {"few 4x2", FEW, 4, 2, 4, 2.558, 0, 0.580, 0.060},     {"few 8x2", FEW, 8, 2, 4, 2.743, 0, 1.047, 0.025},
    {"mid 8x8", MID, 8, 8, 768, 5.416, 0.467, 0, 2.579},   {"many 16x16", MANY, 16, 16, 256, 11.667, 0.763, 0, 1.376},
};

uint64_t tiles_of(const Form &f, uint32_t m, uint32_t n) {
  return (uint64_t)((fk::mx4_row_tiles(m) + f.mb - 1) / f.mb) * ((fk::mx4_row_tiles(n) + f.nb - 1) / f.nb);
}

double cost(const Form &f, uint32_t m, uint32_t n, uint32_t k) {
  const double t = (double)tiles_of(f, m, n), pairs = fk::mx4_pairs(k);
  if (f.kind == FEW)
    return f.base + std::ceil(pairs / f.by) * (f.step + f.turn * std::ceil(t / 256)) +
           f.work * 1e-3 * t * pairs * (f.mb + f.nb);
  return f.base * std::ceil(t / f.by) + f.step * pairs + f.work * 1e-5 * t * f.mb * f.nb * pairs;
}

// mid and many address a tile's slab with 32 bits.
bool takes(const Form &f, uint32_t k) { return f.kind == FEW || fk::mx4_pairs(k) < 1u << 16; }

uint32_t pick(uint32_t m, uint32_t n, uint32_t k) {
  uint32_t best = 0;
  for (uint32_t i = 1; i < std::size(forms); i++)
    if (takes(forms[i], k) && cost(forms[i], m, n, k) < cost(forms[best], m, n, k)) best = i;
  return best;
}

// Why the kernels do not take a product of these sizes; null if they do.
const char *refused(uint32_t m, uint32_t n, uint32_t k) {
  if (!matrix(m, k) || !matrix(n, k)) return "no such matrices";
  if ((uint64_t)fk::mx4_row_tiles(m) * fk::mx4_row_tiles(n) >= 1ull << 31) return "2^31 tiles and more";
  const Form &f = forms[pick(m, n, k)];
  if (f.kind != MANY && tiles_of(f, m, n) >= 1ull << 23)  // a launch of 2^32 threads
    return "2^23 threadgroups and more";
  return nullptr;
}

template <uint32_t I, int T>
void queue_form(const fk_mx4_gemm_args &a, hipStream_t s) {
  constexpr Form f = forms[I];
  const uint32_t tiles = (uint32_t)tiles_of(f, a.m, a.n);
  if constexpr (f.kind == FEW)
    hipLaunchKernelGGL((op_mx4_gemm_few<f.mb, f.nb, f.by, T>), dim3(tiles), dim3(64 * f.by), 0, s, a);
  else if constexpr (f.kind == MID)
    hipLaunchKernelGGL((op_mx4_gemm_mid<f.mb / 4, f.nb / 4, T>), dim3(tiles), dim3(256),
                       (fk::mx4_mid_lds<f.mb / 4, f.nb / 4>()), s, a);
  else
    hipLaunchKernelGGL((op_mx4_gemm_many<T>), dim3(tiles < f.by ? tiles : f.by), dim3(256), fk::mx4_many_lds, s, a);
}

template <int T, size_t... I>
void queue_picked(uint32_t form, const fk_mx4_gemm_args &a, hipStream_t s, std::index_sequence<I...>) {
  ((form == I ? queue_form<I, T>(a, s) : void()), ...);
}

}  // namespace

namespace fk {

int check(const fk_mx4_quantize_args &a, Refusal &no) {
  if (!matrix(a.rows, a.k)) return no(FK_ERR_RANGE, "no matrix of %u rows of %u", a.rows, a.k);
  if (int st = check_rows(no, "x", a.x_stride, a.k, a.x_type)) return st;
  const Span reads[] = {rows_of("x", a.x, a.rows, a.x_stride, a.k, a.x_type)};
  const Span writes[] = {{"codes", a.codes, codes_bytes(a.rows, a.k)}, {"scales", a.scales, scales_bytes(a.rows, a.k)}};
  return check_spans(no, reads, 1, writes, 2);
}

int check(const fk_mx4_dequantize_args &a, Refusal &no) {
  if (!matrix(a.rows, a.k)) return no(FK_ERR_RANGE, "no matrix of %u rows of %u", a.rows, a.k);
  if (int st = check_rows(no, "y", a.y_stride, a.k, a.y_type)) return st;
  const Span reads[] = {{"codes", a.codes, codes_bytes(a.rows, a.k)}, {"scales", a.scales, scales_bytes(a.rows, a.k)}};
  const uint64_t blocks = (a.k >> 5) + ((a.k & 31u) != 0);
  const Span writes[] = {rows_of("y", a.y, a.rows, a.y_stride, a.k, a.y_type),
                         {"scales_out", a.scales_out, a.scales_out ? 4ull * a.rows * blocks : 0, 4}};
  return check_spans(no, reads, 2, writes, 2);
}

int check(const fk_mx4_gemm_args &a, Refusal &no) {
  if (const char *why = refused(a.m, a.n, a.k))
    return no(FK_ERR_RANGE, "a product of %u by %u rows of %u: %s", a.m, a.n, a.k, why);
  if (int st = check_rows(no, "c", a.c_stride, a.n, a.c_type)) return st;
  const Span reads[] = {{"a_codes", a.a_codes, codes_bytes(a.m, a.k)},
                        {"a_scales", a.a_scales, scales_bytes(a.m, a.k)},
                        {"b_codes", a.b_codes, codes_bytes(a.n, a.k)},
                        {"b_scales", a.b_scales, scales_bytes(a.n, a.k)}};
  const Span writes[] = {rows_of("c", a.c, a.m, a.c_stride, a.n, a.c_type)};
  return check_spans(no, reads, 4, writes, 1);
}

}  // namespace fk

extern "C" size_t fk_mx4_codes_bytes(uint32_t rows, uint32_t k) { return matrix(rows, k) ? codes_bytes(rows, k) : 0; }
extern "C" size_t fk_mx4_scales_bytes(uint32_t rows, uint32_t k) { return matrix(rows, k) ? scales_bytes(rows, k) : 0; }

extern "C" int fk_mx4_quantize(fk_ctx *ctx, const fk_mx4_quantize_args *a, fk_stream *stream) {
  if (int st = admit(ctx, "fk_mx4_quantize", a, stream)) return st;
  const dim3 grid(tile_groups(a->rows, a->k)), block(FK_MX4_THREADS);
  const hipStream_t s = stream_of(ctx, stream);
  of_type(a->x_type, [&](auto t) {
    if (passes_by(*a)) hipLaunchKernelGGL((op_mx4_quantize<decltype(t)::value, true>), grid, block, 0, s, *a);
    else hipLaunchKernelGGL((op_mx4_quantize<decltype(t)::value, false>), grid, block, 0, s, *a);
  });
  return launched(ctx, "fk_mx4_quantize");
}

extern "C" int fk_mx4_dequantize(fk_ctx *ctx, const fk_mx4_dequantize_args *a, fk_stream *stream) {
  if (int st = admit(ctx, "fk_mx4_dequantize", a, stream)) return st;
  const dim3 grid(tile_groups(a->rows, a->k)), block(FK_MX4_THREADS);
  const hipStream_t s = stream_of(ctx, stream);
  of_type(a->y_type, [&](auto t) {
    hipLaunchKernelGGL((op_mx4_dequantize<decltype(t)::value>), grid, block, 0, s, *a);
  });
  return launched(ctx, "fk_mx4_dequantize");
}

extern "C" const char *fk_mx4_gemm_form(uint32_t m, uint32_t n, uint32_t k) {
  return refused(m, n, k) ? "" : forms[pick(m, n, k)].name;
}

extern "C" int fk_mx4_gemm(fk_ctx *ctx, const fk_mx4_gemm_args *a, fk_stream *stream) {
  if (int st = admit(ctx, "fk_mx4_gemm", a, stream)) return st;
  const hipStream_t s = stream_of(ctx, stream);
  of_type(a->c_type, [&](auto t) {
    queue_picked<decltype(t)::value>(pick(a->m, a->n, a->k), *a, s, std::make_index_sequence<std::size(forms)>{});
  });
  return launched(ctx, "fk_mx4_gemm");
}
