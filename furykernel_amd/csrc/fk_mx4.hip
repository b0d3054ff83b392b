// fk_mx4.hip — the 4-bit microscaled matrices' operators as one C call each
// (include/fkrocm_mx4.h), their kernels compiled into the C ABI's library.

#include "../../include/fkrocm_mx4.h"

#include <hip/hip_runtime.h>
#include <cstdlib>

#include "fk_admit.h"
#include "kernels/fk_mx4.h"
#include "kernels/fk_mx4_gemm.h"

using fk::admit;
using fk::launched;
using fk::Refusal;
using fk::Span;
using fk::stream_of;

namespace {

template <int T, bool WIDE>
__global__ void __launch_bounds__(FK_MX4_THREADS) op_mx4_quantize(fk_mx4_quantize_args a) {
  fk::mx4_quantize<T, WIDE>(a);
}

template <int T, bool WIDE>
__global__ void __launch_bounds__(FK_MX4_THREADS) op_mx4_dequantize(fk_mx4_dequantize_args a) {
  fk::mx4_dequantize<T, WIDE>(a);
}

template <uint32_t MB, uint32_t NB, uint32_t W, int T>
__global__ void __launch_bounds__(64 * W) op_mx4_gemm_few(fk_mx4_gemm_args a) {
  fk::mx4_gemm_few<MB, NB, W, T>(a);
}

template <uint32_t GB, int T>
__global__ void __launch_bounds__(256, GB == 4 ? 1 : 2) op_mx4_gemm_many(fk_mx4_gemm_args a) {
  fk::mx4_gemm_many<GB, T>(a);
}

uint64_t codes_bytes(uint32_t rows, uint32_t k) { return (uint64_t)fk::mx4_row_tiles(rows) * fk::mx4_pairs(k) * 2048; }
uint64_t scales_bytes(uint32_t rows, uint32_t k) { return (uint64_t)fk::mx4_row_tiles(rows) * fk::mx4_pairs(k) * 128; }

// A matrix the kernels' 32-bit counts of tiles hold.
bool matrix(uint32_t rows, uint32_t k) {
  return rows > 0 && k > 0 && rows <= 1u << 30 && k <= 1u << 30 &&
         (uint64_t)fk::mx4_row_tiles(rows) * fk::mx4_pairs(k) < 1ull << 31;
}

// Rows of `type` from `addr` on, `stride` elements apart: aligned to their
// elements, and to 16 bytes if whole eights go at a time.
int check_rows(Refusal &no, const char *name, uint64_t addr, uint64_t stride, uint64_t width, uint32_t type) {
  if (type > FK_T_BF16) return no(FK_ERR_ARG, "%s of type %u", name, type);
  if (stride < width || stride >= 1ull << 40)
    return no(FK_ERR_ARG, "%s's rows of %llu, %llu apart", name, (unsigned long long)width, (unsigned long long)stride);
  if (addr == 0 || addr % fk::mx4_bytes_of((int)type))
    return no(FK_ERR_ARG, "%s is null or not aligned to its elements", name);
  return FK_OK;
}
bool wide_rows(uint64_t addr, uint64_t stride, uint64_t k, uint32_t type) {
  return addr % 16 == 0 && k % 8 == 0 && stride * fk::mx4_bytes_of((int)type) % 16 == 0;
}
uint64_t rows_bytes(uint64_t rows, uint64_t stride, uint64_t width, uint32_t type) {
  return ((rows - 1) * stride + width) * fk::mx4_bytes_of((int)type);
}

// A threadgroup a FK_MX4_THREADS / 64 pairs of tiles.
uint32_t pair_groups(uint32_t rows, uint32_t k) {
  const uint64_t pairs = (uint64_t)fk::mx4_row_tiles(rows) * fk::mx4_pairs(k), w = FK_MX4_THREADS / FK_WAVE;
  return (uint32_t)((pairs + w - 1) / w);
}

template <typename F>
void of_type(uint32_t type, F &&f) {
  if (type == FK_T_F32) f(std::integral_constant<int, FK_T_F32>{});
  else if (type == FK_T_F16) f(std::integral_constant<int, FK_T_F16>{});
  else f(std::integral_constant<int, FK_T_BF16>{});
}

template <uint32_t MB, uint32_t NB, uint32_t W, int T>
void queue_few(const fk_mx4_gemm_args &a, hipStream_t s) {
  const uint32_t tm = (fk::mx4_row_tiles(a.m) + MB - 1) / MB, tn = (fk::mx4_row_tiles(a.n) + NB - 1) / NB;
  hipLaunchKernelGGL((op_mx4_gemm_few<MB, NB, W, T>), dim3(tm * tn), dim3(64 * W), 0, s, a);
}

template <uint32_t GB, int T>
void queue_many(const fk_mx4_gemm_args &a, hipStream_t s) {
  constexpr uint32_t side = fk::mx4_many_tiles<GB>();
  const uint32_t tm = (fk::mx4_row_tiles(a.m) + side - 1) / side, tn = (fk::mx4_row_tiles(a.n) + side - 1) / side;
  const uint32_t most = GB == 4 ? 256 : 512;  // as many as the chip holds at once
  hipLaunchKernelGGL((op_mx4_gemm_many<GB, T>), dim3(tm * tn < most ? tm * tn : most), dim3(256), fk::mx4_many_lds<GB>(), s, a);
}

}  // namespace

namespace fk {

int check(const fk_mx4_quantize_args &a, Refusal &no) {
  if (!matrix(a.rows, a.k)) return no(FK_ERR_RANGE, "no matrix of %u rows of %u", a.rows, a.k);
  if (int st = check_rows(no, "x", a.x, a.x_stride, a.k, a.x_type)) return st;
  const Span x = {"x", a.x, rows_bytes(a.rows, a.x_stride, a.k, a.x_type)};
  const Span writes[] = {{"codes", a.codes, codes_bytes(a.rows, a.k)}, {"scales", a.scales, scales_bytes(a.rows, a.k)}};
  for (const Span &w : writes)
    if (meets(w, x)) return no(FK_ERR_ARG, "%s overlaps x", w.name);
  return check_spans(no, nullptr, 0, writes, 2, 16);
}

int check(const fk_mx4_dequantize_args &a, Refusal &no) {
  if (!matrix(a.rows, a.k)) return no(FK_ERR_RANGE, "no matrix of %u rows of %u", a.rows, a.k);
  if (int st = check_rows(no, "y", a.y, a.y_stride, a.k, a.y_type)) return st;
  const Span reads[] = {{"codes", a.codes, codes_bytes(a.rows, a.k)}, {"scales", a.scales, scales_bytes(a.rows, a.k)}};
  const Span y = {"y", a.y, rows_bytes(a.rows, a.y_stride, a.k, a.y_type)};
  const Span out = {"scales_out", a.scales_out, a.scales_out ? 4ull * a.rows * ((a.k >> 5) + ((a.k & 31u) != 0)) : 0};
  if (a.scales_out % 4) return no(FK_ERR_ARG, "scales_out is not 4-byte aligned");
  for (const Span &w : {y, out})
    for (const Span &r : reads)
      if (meets(w, r)) return no(FK_ERR_ARG, "%s overlaps %s", w.name, r.name);
  if (meets(y, out)) return no(FK_ERR_ARG, "scales_out overlaps y");
  return check_spans(no, reads, 2, nullptr, 0, 16);
}

int check(const fk_mx4_gemm_args &a, Refusal &no) {
  if (!matrix(a.m, a.k) || !matrix(a.n, a.k)) return no(FK_ERR_RANGE, "no product of %u and %u rows of %u", a.m, a.n, a.k);
  if ((uint64_t)mx4_row_tiles(a.m) * mx4_row_tiles(a.n) >= 1ull << 31)
    return no(FK_ERR_RANGE, "a product of %u by %u: 2^31 tiles and more", a.m, a.n);
  if (int st = check_rows(no, "c", a.c, a.c_stride, a.n, a.c_type)) return st;
  const Span reads[] = {{"a_codes", a.a_codes, codes_bytes(a.m, a.k)},
                        {"a_scales", a.a_scales, scales_bytes(a.m, a.k)},
                        {"b_codes", a.b_codes, codes_bytes(a.n, a.k)},
                        {"b_scales", a.b_scales, scales_bytes(a.n, a.k)}};
  const Span c = {"c", a.c, rows_bytes(a.m, a.c_stride, a.n, a.c_type)};
  for (const Span &r : reads)
    if (meets(c, r)) return no(FK_ERR_ARG, "c overlaps %s", r.name);
  return check_spans(no, reads, 4, nullptr, 0, 16);
}

}  // namespace fk

extern "C" size_t fk_mx4_codes_bytes(uint32_t rows, uint32_t k) { return matrix(rows, k) ? codes_bytes(rows, k) : 0; }
extern "C" size_t fk_mx4_scales_bytes(uint32_t rows, uint32_t k) { return matrix(rows, k) ? scales_bytes(rows, k) : 0; }

extern "C" int fk_mx4_quantize(fk_ctx *ctx, const fk_mx4_quantize_args *a, fk_stream *stream) {
  if (int st = admit(ctx, "fk_mx4_quantize", a)) return st;
  const dim3 grid(pair_groups(a->rows, a->k)), block(FK_MX4_THREADS);
  const hipStream_t s = stream_of(ctx, stream);
  of_type(a->x_type, [&](auto t) {
    if (wide_rows(a->x, a->x_stride, a->k, a->x_type))
      hipLaunchKernelGGL((op_mx4_quantize<decltype(t)::value, true>), grid, block, 0, s, *a);
    else
      hipLaunchKernelGGL((op_mx4_quantize<decltype(t)::value, false>), grid, block, 0, s, *a);
  });
  return launched(ctx, "fk_mx4_quantize");
}

extern "C" int fk_mx4_dequantize(fk_ctx *ctx, const fk_mx4_dequantize_args *a, fk_stream *stream) {
  if (int st = admit(ctx, "fk_mx4_dequantize", a)) return st;
  const dim3 grid(pair_groups(a->rows, a->k)), block(FK_MX4_THREADS);
  const hipStream_t s = stream_of(ctx, stream);
  of_type(a->y_type, [&](auto t) {
    if (wide_rows(a->y, a->y_stride, a->k, a->y_type))
      hipLaunchKernelGGL((op_mx4_dequantize<decltype(t)::value, true>), grid, block, 0, s, *a);
    else
      hipLaunchKernelGGL((op_mx4_dequantize<decltype(t)::value, false>), grid, block, 0, s, *a);
  });
  return launched(ctx, "fk_mx4_dequantize");
}

extern "C" int fk_mx4_gemm(fk_ctx *ctx, const fk_mx4_gemm_args *a, fk_stream *stream) {
  if (int st = admit(ctx, "fk_mx4_gemm", a)) return st;
  const hipStream_t s = stream_of(ctx, stream);
  of_type(a->c_type, [&](auto t) {
    constexpr int T = decltype(t)::value;
    const char *f = getenv("FK_MX4_FORM");
    const int form = f ? atoi(f) : (a->m <= 16 ? 0 : a->m <= 128 ? 3 : 5);
    switch (form) {
      case 0: queue_few<1, 1, 8, T>(*a, s); break;
      case 1: queue_few<1, 2, 8, T>(*a, s); break;
      case 2: queue_few<2, 2, 8, T>(*a, s); break;
      case 3: queue_few<4, 4, 4, T>(*a, s); break;
      case 4: queue_many<2, T>(*a, s); break;
      case 6: queue_few<4, 2, 8, T>(*a, s); break;
      case 7: queue_few<4, 1, 8, T>(*a, s); break;
      case 8: queue_few<2, 1, 8, T>(*a, s); break;
      case 9: queue_few<8, 2, 4, T>(*a, s); break;
      default: queue_many<4, T>(*a, s);
    }
  });
  return launched(ctx, "fk_mx4_gemm");
}
