/*
 * fkrocm_serve.h — the operators of a served batch, one C call each over
 * device buffers the caller holds: what a step over paged KV caches does
 * beside the model's own launches.
 *
 *   fk_page_plan       block tables and slot maps from the requests' lengths
 *   fk_paged_store     q, k, v rows: RoPE, k and v into the pools at their slots
 *   fk_paged_attend    attention of one new token a request over its pages
 *
 * The pools are the program layer's paged caches (src/FuryKernel/Program/
 * Graph.hs:144-152): [blocks][kv_heads][block_size][head_dim] of f16 or bf16,
 * position p of a request at p mod block_size of block table[p / block_size].
 * The reference plans such a step's shapes ahead; requests that come and go,
 * with lengths of their own, are this target's addition.
 *
 * Every call queues its kernels on the stream (NULL: the context's) and
 * returns; it allocates nothing, keeps nothing, and may be captured into a
 * graph.  Arguments that the kernels do not take are refused before anything
 * is queued (FK_ERR_ARG, FK_ERR_RANGE; fk_last_error says what).  Two calls
 * that may run at the same time must not share outputs or a workspace.
 */
#ifndef FKROCM_SERVE_H
#define FKROCM_SERVE_H

#include "fkrocm.h"

#ifdef __cplusplus
extern "C" {
#endif

/* A slot map's entry of a token that is stored nowhere. */
#define FK_NO_SLOT 0xFFFFFFFFu

/* Element types. */
enum { FK_T_F32 = 0, FK_T_F16 = 1, FK_T_BF16 = 2 };

/* The page plan of a step.  Request r holds `cached[r]` positions in the
 * first ceil(cached[r] / block_size) blocks of its table row and brings
 * fresh[r] new tokens (0: none this step).  The tokens are numbered request by
 * request (starts: the prefix sums of fresh); each new block that a request
 * needs is the free list's next, from entry *head on, in the order of the
 * requests, and is written into its table row.
 *
 * Token t < counts[0] of request r: owner[t] = r, positions[t] = cached[r] + t
 * - starts[r], slots[t] = its block times block_size plus its position mod
 * block_size.  Tokens behind the last: owner and slot FK_NO_SLOT, position 0.
 *
 * A request does not fit if cached + fresh passes table_len * block_size, if
 * its tokens (or those of one before it) end past `tokens`, or if it needs new
 * blocks and those that the requests up to it need pass the free list (one
 * whose tokens all go into blocks it holds fits whatever the list holds); it
 * takes no block, its length stays cached, its tokens' slots are FK_NO_SLOT (so
 * what a step makes of them means nothing: it goes into a later step). */
typedef struct fk_page_plan_args {
  uint64_t cached;      /* u32 [requests] */
  uint64_t fresh;       /* u32 [requests] */
  uint64_t free_blocks; /* u32 [free_len] */
  uint64_t head;        /* u32 [1]: the free list's first entry not taken */
  uint64_t table;       /* u32 [requests][table_len]: read, and new blocks written */
  uint64_t lengths;     /* out: u32 [requests]: cached + fresh */
  uint64_t starts;      /* out: u32 [requests + 1] */
  uint64_t slots;       /* out: u32 [tokens] */
  uint64_t positions;   /* out: u32 [tokens] */
  uint64_t owner;       /* out: u32 [tokens] */
  uint64_t counts;      /* out: u32 [4]: tokens, blocks taken, requests that do not fit, the next step's head */
  uint32_t requests;    /* at least 1 */
  uint32_t tokens;      /* the step's tokens, padding included */
  uint32_t table_len;
  uint32_t block_size;
  uint32_t free_len;
} fk_page_plan_args;

/* Addresses are 4-byte aligned; no output overlaps an input or another
 * output (head is none of counts). */
int fk_page_plan(fk_ctx *ctx, const fk_page_plan_args *args, fk_stream *stream);

/* A step's rows into the caches: for each token t with a slot below blocks *
 * block_size, q and k turned by RoPE (src/FuryKernel/Program/Eval.hs:372-383,
 * NeoX halves, in binary32 by the table's cosines and sines at positions[t]),
 * q rounded once into qr, k and v rounded once into the pools.  Tokens without
 * a slot leave everything as it was.  Slots are distinct, as a plan's are (of
 * two tokens with one slot, each element is one's or the other's). */
typedef struct fk_paged_store_args {
  uint64_t q, k, v;   /* rows of rows_type; q may be 0: no queries */
  uint64_t slots;     /* u32 [tokens] */
  uint64_t positions; /* u32 [tokens] (read when rotated) */
  uint64_t rope;      /* f32 [rope_rows][rotated][2] (read when rotated); positions past it take its last row */
  uint64_t qr;        /* out: [tokens][heads][head_dim] of the caches' type */
  uint64_t kpool, vpool;
  uint64_t q_stride, k_stride, v_stride; /* elements from row to row */
  uint32_t tokens;
  uint32_t heads;     /* of q */
  uint32_t kv_heads;
  uint32_t head_dim;  /* a multiple of 16, at most 256 */
  uint32_t block_size;
  uint32_t blocks;
  uint32_t rotated;   /* pairs turned: 0 (no RoPE) to head_dim / 2 */
  uint32_t rope_rows;
  uint32_t rows_type; /* FK_T_* of q, k and v */
  uint32_t cache_bf16; /* the pools and qr hold bf16 (else f16) */
} fk_paged_store_args;

/* Addresses are 16-byte aligned, rows too (strides); slots and positions 4-byte. */
int fk_paged_store(fk_ctx *ctx, const fk_paged_store_args *args, fk_stream *stream);

/* Attention of one new token a request: out[r] = softmax(scale q[r] Kᵀ) V
 * (src/FuryKernel/Program/Eval.hs:474-527) over positions 0 .. lengths[r] - 1
 * of the request (with a window its last `window`), query head h over kv head
 * h / (heads / kv_heads).  With `starts` (a plan's) the query of request r is
 * that of its last new token, row starts[r + 1] - 1 of q_rows, and a request
 * without a new token (or with tokens past q_rows) counts as empty.  A length
 * of 0 gives a row of zeros; a length past table_len * block_size counts as
 * that.  A table entry past `blocks` reads the pool's last block; what entries
 * behind a length hold does not matter.
 *
 * Scores, the running maximum, the sums and the weighted values are binary32
 * (probabilities go to the matrix cores as 16-bit parts, which hold 24 bits of
 * them with bf16 caches, 21 with f16 ones), rounded once on the way out.  The
 * same lengths give the same bits, whatever else the pool holds.  An infinite
 * value gives infinity whatever its key's finite score. */
typedef struct fk_paged_attend_args {
  uint64_t q;         /* rows of [heads][head_dim], the caches' type: a request's each, or with starts q_rows */
  uint64_t kpool, vpool;
  uint64_t table;     /* u32 [requests][table_len] */
  uint64_t lengths;   /* u32 [requests] */
  uint64_t starts;    /* u32 [requests + 1], or 0: q has a row a request */
  uint64_t out;       /* [requests] rows of [heads][head_dim], the caches' type or f32 */
  uint64_t workspace; /* fk_paged_attend_workspace bytes; need not be cleared */
  uint64_t workspace_bytes;
  uint64_t q_stride, out_stride; /* elements from row to row */
  uint32_t requests;
  uint32_t heads;
  uint32_t kv_heads;
  uint32_t head_dim;  /* a multiple of 8, at most 256 */
  uint32_t block_size;
  uint32_t blocks;
  uint32_t table_len;
  uint32_t window;    /* 0: none */
  uint32_t q_rows;    /* with starts: the rows of q */
  uint32_t cache_bf16;
  uint32_t out_f32;
  float scale;
} fk_paged_attend_args;

/* The workspace's bytes for these sizes (addresses, scale and strides are not
 * looked at); 0 if the sizes are refused. */
size_t fk_paged_attend_workspace(const fk_paged_attend_args *args);
/* How a call of these sizes is shared out: "split" (runs of keys, and a second
 * launch that joins them), "whole 4" or "whole 8" (each request and kv head to
 * one threadgroup of as many wavefronts), "" if the sizes are refused; for
 * profiles and tests. */
const char *fk_paged_attend_form(const fk_paged_attend_args *args);
/* Addresses are 16-byte aligned (table, lengths and starts 4-byte); q_stride a
 * multiple of 8. */
int fk_paged_attend(fk_ctx *ctx, const fk_paged_attend_args *args, fk_stream *stream);

/* The checks that an entry makes of its arguments before it queues anything,
 * on the host alone (no GPU, no context): FK_OK, or the status it would return
 * with the reason in `err`.  `args` is the entry's struct, of args_bytes. */
int fk_serve_check(const char *entry, const void *args, size_t args_bytes, char *err, size_t err_cap);

#ifdef __cplusplus
}
#endif

#endif /* FKROCM_SERVE_H */
