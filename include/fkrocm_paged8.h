/*
 * fkrocm_paged8.h — paged KV caches held in 8 bits: rows stored, read back and
 * attended to, one C call each over device buffers the caller holds.  The
 * 8-bit counterparts of fkrocm_serve.h's calls, for the same page plan.
 *
 * A pool is [blocks][kv_heads][block_size][head_dim] of e4m3 (448 the largest,
 * no infinity), and each block and head has a scale for its keys and one for
 * its values: scales f32 [blocks][kv_heads][2] (k's, v's), powers of two.  A
 * value is its code times its scale.
 *
 * What fkrocm_serve.h says of streams, graphs, refusals and workspaces holds
 * here too (fk_serve_check knows these entries).
 */
#ifndef FKROCM_PAGED8_H
#define FKROCM_PAGED8_H

#include "fkrocm.h"
#include "fkrocm_serve.h"

#ifdef __cplusplus
extern "C" {
#endif

/* A step's rows into the caches: for each token t with a slot below blocks *
 * block_size, q and k turned by RoPE as fk_paged_store does, q rounded once
 * into qr (f16 or bf16), k and v to 8 bits.  Tokens without a slot leave
 * everything as it was.
 *
 * The tokens of a block follow one another, in the order of their places (as a
 * plan's do): they are its run.  A block's needed scale is the smallest power of
 * two, from 2^-126 on, that keeps the run's largest finite magnitude within
 * 448.  A run that begins at place 0 begins the block: the needed scale is its
 * scale.  Another run's block takes the larger of its scale and the needed one,
 * and where that grew, the codes at the places before the run are brought to it
 * (each rounded to the nearest, halfway cases to the even code); what lies
 * behind the run keeps its bytes.  Elements are x / scale, rounded likewise; NaN
 * where not finite.  (Two runs of one block in a call: its bytes mean nothing.) */
typedef struct fk_paged_store8_args {
  uint64_t q, k, v;   /* rows of rows_type; q may be 0: no queries */
  uint64_t slots;     /* u32 [tokens] */
  uint64_t positions; /* u32 [tokens] (read when rotated) */
  uint64_t rope;      /* f32 [rope_rows][rotated][2] (read when rotated); positions past it take its last row */
  uint64_t qr;        /* out: [tokens][heads][head_dim], f16 or bf16 */
  uint64_t kpool, vpool;
  uint64_t scales;    /* f32 [blocks][kv_heads][2] */
  uint64_t q_stride, k_stride, v_stride; /* elements from row to row */
  uint32_t tokens;
  uint32_t heads;     /* of q */
  uint32_t kv_heads;
  uint32_t head_dim;  /* a multiple of 16, at most 256 */
  uint32_t block_size; /* a multiple of 8 */
  uint32_t blocks;
  uint32_t rotated;   /* pairs turned: 0 (no RoPE) to head_dim / 2 */
  uint32_t rope_rows;
  uint32_t rows_type; /* FK_T_* of q, k and v */
  uint32_t q_bf16;    /* qr holds bf16 (else f16) */
} fk_paged_store8_args;

/* Addresses are 16-byte aligned, rows too (strides); slots and positions 4-byte,
 * scales 8-byte. */
int fk_paged_store8(fk_ctx *ctx, const fk_paged_store8_args *args, fk_stream *stream);

/* Cached positions as rows: for each t with a slot below blocks * block_size,
 * the keys and values at it into row t of k and v, [kv_heads][head_dim] of
 * rows_type, each rounded once.  Rows without a slot stay as they were. */
typedef struct fk_paged_load8_args {
  uint64_t slots; /* u32 [tokens] */
  uint64_t kpool, vpool;
  uint64_t scales;
  uint64_t k, v;  /* out */
  uint64_t k_stride, v_stride; /* elements from row to row */
  uint32_t tokens;
  uint32_t kv_heads;
  uint32_t head_dim;   /* a multiple of 16, at most 256 */
  uint32_t block_size; /* a multiple of 8 */
  uint32_t blocks;
  uint32_t rows_type;  /* FK_T_* of k and v */
} fk_paged_load8_args;

/* Alignment as fk_paged_store8's. */
int fk_paged_load8(fk_ctx *ctx, const fk_paged_load8_args *args, fk_stream *stream);

/* Attention of one new token a request, as fk_paged_attend's, over 8-bit pools:
 * the requests, tables, lengths, starts, windows and empty rows are as there.
 * q and out are f16 or bf16 (out also f32).  A table entry past `blocks` reads
 * the pool's last block; what lies behind a length, and what entries behind it
 * hold, does not matter.
 *
 * Scores, the running maximum, the sums and the weighted values are binary32,
 * rounded once on the way out (probabilities go to the matrix cores as three
 * bf16 parts, which hold all their bits; of values below 2^-126 what bfloat16
 * holds, or nothing).  The same lengths give the same bits, whatever else the pool
 * holds. */
typedef struct fk_paged_attend8_args {
  uint64_t q;         /* rows of [heads][head_dim], f16 or bf16: a request's each, or with starts q_rows */
  uint64_t kpool, vpool;
  uint64_t scales;    /* f32 [blocks][kv_heads][2] */
  uint64_t table;     /* u32 [requests][table_len] */
  uint64_t lengths;   /* u32 [requests] */
  uint64_t starts;    /* u32 [requests + 1], or 0: q has a row a request */
  uint64_t out;       /* [requests] rows of [heads][head_dim], q's type or f32 */
  uint64_t workspace; /* fk_paged_attend8_workspace bytes; need not be cleared */
  uint64_t workspace_bytes;
  uint64_t q_stride, out_stride; /* elements from row to row */
  uint32_t requests;
  uint32_t heads;
  uint32_t kv_heads;
  uint32_t head_dim;  /* a multiple of 16, at most 256 */
  uint32_t block_size; /* a multiple of 8 */
  uint32_t blocks;
  uint32_t table_len;
  uint32_t window;    /* 0: none */
  uint32_t q_rows;    /* with starts: the rows of q */
  uint32_t q_bf16;    /* q holds bf16 (else f16) */
  uint32_t out_f32;
  float scale;
} fk_paged_attend8_args;

/* As fk_paged_attend_workspace and fk_paged_attend_form. */
size_t fk_paged_attend8_workspace(const fk_paged_attend8_args *args);
const char *fk_paged_attend8_form(const fk_paged_attend8_args *args);
/* Addresses are 16-byte aligned (table, lengths and starts 4-byte, scales
 * 8-byte); q_stride a multiple of 8. */
int fk_paged_attend8(fk_ctx *ctx, const fk_paged_attend8_args *args, fk_stream *stream);

#ifdef __cplusplus
}
#endif

#endif /* FKROCM_PAGED8_H */
