// fk_admit.h — what the one-call operators' entries share: the checks of their
// arguments, made on the host before anything is queued, and their refusals.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdio>
#include <type_traits>

#include "../../include/fkrocm_fp8.h"
#include "../../include/fkrocm_mx4.h"
#include "../../include/fkrocm_paged8.h"
#include "fk_internal.h"

namespace fk {

// The context's device, and nothing left of what an earlier call on this
// thread (a refused allocation, another library's) failed with: `launched`
// would take it for the launch's.
inline int use_device(fk_ctx *ctx) {
  const hipError_t e = hipSetDevice(ctx->device);
  (void)hipGetLastError();
  return e == hipSuccess ? FK_OK : fk_fail(ctx, FK_ERR_HIP, "hipSetDevice: %s", hipGetErrorString(e));
}

inline int launched(fk_ctx *ctx, const char *what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? FK_OK : fk_fail(ctx, FK_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

inline hipStream_t stream_of(fk_ctx *ctx, fk_stream *s) { return s ? s->stream : ctx->stream; }

// What a check of a call's arguments finds: FK_OK, or a status and the reason.
struct Refusal {
  char text[512] = "";
  __attribute__((format(printf, 3, 4))) int operator()(int status, const char *fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(text, sizeof text, fmt, ap);
    va_end(ap);
    return status;
  }
};

// A span of device memory a call reads or writes, aligned to `align` bytes.
struct Span {
  const char *name;
  uint64_t addr, bytes;
  uint32_t align = 16;
};

// The bytes from the first to the last of `rows` rows, `stride` elements of
// `bytes` apart; what no memory holds as 2^62.
inline uint64_t rows_span(uint64_t rows, uint64_t stride, uint64_t width, uint64_t bytes) {
  const __uint128_t span = rows ? ((__uint128_t)(rows - 1) * stride + width) * bytes : 0;
  return span < 1ull << 62 ? (uint64_t)span : 1ull << 62;
}

inline bool meets(const Span &a, const Span &b) {
  return a.bytes && b.bytes && a.addr < b.addr + b.bytes && b.addr < a.addr + a.bytes;
}

// Every span there, aligned and within 2^48 bytes; no output over another span.
inline int check_spans(Refusal &no, const Span *reads, size_t n_reads, const Span *writes, size_t n_writes) {
  for (size_t i = 0; i < n_reads + n_writes; i++) {
    const Span &s = i < n_reads ? reads[i] : writes[i - n_reads];
    if (s.bytes && (s.addr == 0 || s.addr % s.align))
      return no(FK_ERR_ARG, "%s is null or not %u-byte aligned", s.name, s.align);
    if (s.bytes >= 1ull << 48 || s.addr > UINT64_MAX - s.bytes)
      return no(FK_ERR_RANGE, "%s spans 2^48 bytes and more", s.name);
  }
  for (size_t i = 0; i < n_writes; i++) {
    for (size_t j = 0; j < n_reads; j++)
      if (meets(writes[i], reads[j])) return no(FK_ERR_ARG, "%s overlaps %s", writes[i].name, reads[j].name);
    for (size_t j = 0; j < i; j++)
      if (meets(writes[i], writes[j])) return no(FK_ERR_ARG, "%s overlaps %s", writes[i].name, writes[j].name);
  }
  return FK_OK;
}

// Rows of an FK_T_* type, `stride` elements apart, aligned to their elements.
inline uint32_t type_bytes(uint32_t type) { return type == FK_T_F32 ? 4 : 2; }
inline int check_rows(Refusal &no, const char *name, uint64_t stride, uint64_t width, uint32_t type) {
  if (type > FK_T_BF16) return no(FK_ERR_ARG, "%s of type %u", name, type);
  if (stride < width || stride >= 1ull << 40)
    return no(FK_ERR_ARG, "%s's rows of %llu, %llu apart", name, (unsigned long long)width, (unsigned long long)stride);
  return FK_OK;
}
inline Span rows_of(const char *name, uint64_t addr, uint64_t rows, uint64_t stride, uint64_t width, uint32_t type) {
  return {name, addr, rows_span(rows, stride, width, type_bytes(type)), type_bytes(type)};
}

// f with an FK_T_* type as a constant.
template <typename F>
void of_type(uint32_t type, F &&f) {
  if (type == FK_T_F32) f(std::integral_constant<int, FK_T_F32>{});
  else if (type == FK_T_F16) f(std::integral_constant<int, FK_T_F16>{});
  else f(std::integral_constant<int, FK_T_BF16>{});
}

// A call's arguments as its entry takes them, or the refusal on the context.
template <typename Args, typename... More>
int admit(fk_ctx *ctx, const char *what, const Args *a, fk_stream *stream, const More &...more) {
  if (!ctx || !a) return fk_fail(ctx, FK_ERR_ARG, "%s: null argument", what);
  if (stream && stream->ctx->device != ctx->device)
    return fk_fail(ctx, FK_ERR_ARG, "%s: a stream of device %d on device %d", what, stream->ctx->device, ctx->device);
  Refusal no;
  if (int st = check(*a, more..., no)) return fk_fail(ctx, st, "%s: %s", what, no.text);
  return use_device(ctx);
}

}  // namespace fk

// The checks of the other files' entries, for fk_serve_check.
namespace fk {
int check(const fk_mx4_quantize_args &a, Refusal &no);
int check(const fk_mx4_dequantize_args &a, Refusal &no);
int check(const fk_mx4_gemm_args &a, Refusal &no);
int check(const fk_fp8_quantize_args &a, Refusal &no);
int check(const fk_fp8_dequantize_args &a, Refusal &no);
int check(const fk_fp8_add_norm_args &a, Refusal &no);
int check(const fk_fp8_gemm_args &a, Refusal &no);
int check(const fk_paged_store8_args &a, Refusal &no);
int check(const fk_paged_load8_args &a, Refusal &no);
int check(const fk_paged_attend8_args &a, Refusal &no);
}  // namespace fk
