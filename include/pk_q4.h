/*
 * pk_q4.h - C ABI of the product with 4-bit weights and group scales on
 * gfx950, from one row (a token) to many. Same library, contexts, streams,
 * events and status codes as pk_palette.h. No counterpart in the reference,
 * whose packed weights are 5- and 6-bit palette codes (gemm.ts:621-704);
 * pk_gemm_* is that product.
 *
 *   w[k, n]   = scale[k / G, n] * (code[k, n] - 8) + offset[k / G, n]
 *   out[m, n] = residual + residual_scale * activation(sum_k a[m, k] w[k, n]
 *               + bias[n])
 *
 * with the reference's epilogue order (gemm.ts:2006-2044); SiLU is
 * v / (1 + exp(-v)) without the reference's clamp. Products and sums are f32
 * in both profiles (f16: f16 operands in exact products; f32: f32 operands),
 * scales are applied to each group's sum in f32, and an output is rounded
 * once. A group's sums of a (code - 8) and, for its offset, of a have to stay
 * within f32: they do where the magnitudes of `a` add up to less than 2^125
 * over a group (f16: always). Where they do not, or an activation is an
 * infinity or a NaN, outputs of that row are infinities or NaN, NaN also where
 * the formula has an infinity (with offsets the two sums may be opposite
 * ones), and no other row is touched.
 */
#ifndef PK_Q4_H
#define PK_Q4_H

#include "pk_palette.h"

#ifdef __cplusplus
extern "C" {
#endif

#define PK_Q4_MAX_ROWS 1048560u
#define PK_Q4_MAX_STRIDE 16777216u

typedef struct pk_q4_op pk_q4_op;

typedef struct pk_q4_desc {
  uint32_t struct_size;          /* sizeof(pk_q4_desc) */
  const char *label;
  int32_t precision;             /* pk_precision of a, scales, offsets, residual and output */
  uint32_t rows;                 /* M capacity, 1 to PK_Q4_MAX_ROWS */
  uint32_t inner;                /* K, 1 to PK_Q4_MAX_STRIDE */
  uint32_t columns;              /* N; ceil(K / 128) * ceil(N / 16) below 2^24, M * N at most 2^35 */
  uint32_t group_size;           /* G: a power of two from 32 on, or 0 (one group: G = K);
                                    the last group may be short */
  const void *a;                 /* [rows, inner], rows a_stride elements apart (0: inner) */
  uint64_t a_bytes;
  uint32_t a_stride;             /* at most PK_Q4_MAX_STRIDE */
  const uint32_t *packed;        /* codes of [inner, columns], K-major, 8 per word, LSB first */
  uint64_t packed_bytes;         /* exactly 4 * ceil(inner * columns / 8) */
  const void *scales;            /* [ceil(inner / G), columns] */
  uint64_t scales_bytes;         /* exactly */
  const void *offsets;           /* like scales, or NULL: zero */
  uint64_t offsets_bytes;
  void *output;                  /* [rows, columns], rows output_stride elements apart (0: columns) */
  uint64_t output_bytes;
  uint32_t output_stride;
  const float *bias;             /* [columns] f32, or NULL */
  uint64_t bias_bytes;           /* exactly 4 * columns */
  const void *residual;          /* like output, or NULL */
  uint64_t residual_bytes;
  uint32_t residual_stride;
  int32_t has_residual_scale;    /* 0: scale 1 when a residual is given */
  float residual_scale;
  int32_t activation;            /* pk_activation */
} pk_q4_desc;

/* a, output and residual may start at any address that fits their elements
   and have any stride. The output may be the residual (the same
   pointer and stride); any other overlap with a or the residual is refused,
   where columns of one buffer (the same stride) do not overlap if their
   columns do not. */
int pk_q4_validate(const pk_q4_desc *desc);
/* Lays the codes, scales and offsets out once in memory of the op, on
   `stream`, and returns when that is done: the bindings may be freed or
   changed then. Refused on a stream that is capturing a graph. */
int pk_q4_create(pk_context *ctx, const pk_q4_desc *desc, void *stream, pk_q4_op **out);
/* The first `active_rows` rows (0 = all); rows behind them are left as they
   were. A row's outputs may differ in their last bits between row counts
   (another order of the sum over K), never from launch to launch of one
   count. May be captured into graphs. Few tiles of a long K are split along
   it and meet in memory of the op: launches of one op, eager or replayed,
   must be ordered by the caller, as their outputs ask for anyway. */
int pk_q4_enqueue(pk_q4_op *op, uint32_t active_rows, void *stream);
int pk_q4_enqueue_timed(pk_q4_op *op, uint32_t active_rows, void *stream, void *start_event, void *end_event);
/* Device bytes of the weight in the op: half a byte per weight (K padded to
   128, N to 16) and its scales and offsets. A split K takes up to 16 MiB
   more. */
int pk_q4_weight_bytes(const pk_q4_op *op, uint64_t *bytes);
int pk_q4_destroy(pk_q4_op *op);
int pk_q4_release(pk_q4_op *op);

#ifdef __cplusplus
}
#endif

#endif
