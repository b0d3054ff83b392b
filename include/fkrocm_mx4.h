/*
 * fkrocm_mx4.h — 4-bit microscaled matrices (the OCP MX format MXFP4): made,
 * read back and multiplied, one C call each over device buffers the caller
 * holds.  For a served model's linears: the weights kept at 4.25 bits an
 * element, the activations brought to the same form as they come, the product
 * on the matrix cores' scaled 4-bit operations.
 *
 * A row's elements go by blocks of 32.  A block has one scale, a power of two
 * (e8m0: a byte b stands for 2^(b - 127), 255 for NaN), and each element a
 * sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (e2m1) times the scale.
 *
 *   scale    2^(floor(log2 max |x|) - 2), at least 2^-127; 1 for a block of
 *            zeros; NaN for a block with a value that is not finite
 *   element  x / scale to the nearest, halfway cases to the even code; 6 for
 *            what is larger
 *
 * A matrix [rows, k] is held in the order the matrix operations take it: rows
 * by 16 and elements by 128 (4 blocks), such a tile's 64 blocks (block j of
 * row r at 16 j + r) as 16 bytes of codes each, element 2 i of a block the low
 * half of its byte i; tiles of one 16 rows in the order of k, which counts up
 * to a multiple of 256.  The scales lie apart, two bytes a block place: those
 * of a tile and of the next, for every pair of tiles.  Rows past the last to a
 * multiple of 16, and elements past k, are codes 0 of scale 1.
 *
 * The calls queue on the stream (NULL: the context's), allocate nothing and
 * may be captured.  Arguments the kernels do not take are refused before
 * anything is queued (fk_serve_check of fkrocm_serve.h knows these entries
 * too).
 */
#ifndef FKROCM_MX4_H
#define FKROCM_MX4_H

#include "fkrocm.h"
#include "fkrocm_serve.h"

#ifdef __cplusplus
extern "C" {
#endif

/* The bytes of a matrix's codes and of its scales. */
size_t fk_mx4_codes_bytes(uint32_t rows, uint32_t k);
size_t fk_mx4_scales_bytes(uint32_t rows, uint32_t k);

/* x [rows][k], x_stride elements from row to row, to 4 bits. */
typedef struct fk_mx4_quantize_args {
  uint64_t x;
  uint64_t codes;
  uint64_t scales;
  uint64_t x_stride;
  uint32_t rows;
  uint32_t k;
  uint32_t x_type; /* FK_T_* */
} fk_mx4_quantize_args;

/* x is aligned to its elements, codes and scales to 16 bytes. */
int fk_mx4_quantize(fk_ctx *ctx, const fk_mx4_quantize_args *args, fk_stream *stream);

/* The values that a matrix stands for, each rounded once to y's type, and its
 * scales. */
typedef struct fk_mx4_dequantize_args {
  uint64_t codes;
  uint64_t scales;
  uint64_t y;          /* [rows][k], y_stride elements from row to row */
  uint64_t scales_out; /* f32 [rows][ceil(k / 32)], or 0 */
  uint64_t y_stride;
  uint32_t rows;
  uint32_t k;
  uint32_t y_type; /* FK_T_* */
} fk_mx4_dequantize_args;

int fk_mx4_dequantize(fk_ctx *ctx, const fk_mx4_dequantize_args *args, fk_stream *stream);

/* C [m][n] = A Bᵀ of A [m][k] and B [n][k], products exact, sums binary32 in
 * the matrix operations' order (the same for every run of one shape), rounded
 * once to c's type. */
typedef struct fk_mx4_gemm_args {
  uint64_t a_codes, a_scales;
  uint64_t b_codes, b_scales;
  uint64_t c;
  uint64_t c_stride; /* elements from row to row */
  uint32_t m;
  uint32_t n;
  uint32_t k;
  uint32_t c_type; /* FK_T_* */
} fk_mx4_gemm_args;

int fk_mx4_gemm(fk_ctx *ctx, const fk_mx4_gemm_args *args, fk_stream *stream);

/* The name of the kernel form that a product of these sizes takes ("" for one
 * that is refused); for profiles and tests. */
const char *fk_mx4_gemm_form(uint32_t m, uint32_t n, uint32_t k);

#ifdef __cplusplus
}
#endif

#endif /* FKROCM_MX4_H */
