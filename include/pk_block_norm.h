/*
 * pk_block_norm.h - C ABI of the fused norms around a block on gfx950: the
 * norm of a block's output, its gate and residual, and the norm that feeds
 * the next block, in one pass over the rows. Same library, contexts, streams,
 * events and status codes as pk_palette.h. No counterpart in the reference,
 * whose graph runs a LayerNorm dispatch (layernorm.ts:29-240) on each side of
 * a GEMM with a residual epilogue; pk_layernorm.h is that dispatch.
 *
 *   v      = input, or norm(input; gamma, beta) with gamma set
 *   y      = residual + residual_scale * gate * v
 *   output = y rounded to the profile's type
 *   next_output = norm(y; next_gamma, next_beta) rounded likewise
 *
 * A missing gate counts as one, a missing residual as zero. Over the C
 * channels of a row, PK_NORM_LAYER is
 *   (x - mean) / sqrt(mean((x - mean)^2) + epsilon) * gamma + beta
 * and PK_NORM_RMS x / sqrt(mean(x^2) + epsilon) * gamma + beta, a missing
 * beta counting as zero. Everything between loading and storing is f32: the
 * second norm sees y before its rounding. The squares that a norm adds up have
 * to stay within f32: they do where its operands, the input or y, lie below
 * 2^56 in magnitude. A row with an infinity or a NaN has NaN where the formula
 * has it and touches no other row.
 */
#ifndef PK_BLOCK_NORM_H
#define PK_BLOCK_NORM_H

#include "pk_palette.h"

#ifdef __cplusplus
extern "C" {
#endif

#define PK_BLOCK_NORM_MAX_CHANNELS 16384u
#define PK_BLOCK_NORM_MAX_ROWS 4194303u

typedef enum pk_norm_kind {
  PK_NORM_LAYER = 0,
  PK_NORM_RMS = 1,
} pk_norm_kind;

typedef struct pk_block_norm_op pk_block_norm_op;

/* Matrices are rows of `channels` elements of the profile's type, each row
   `*_stride` elements after the one before (0: channels), at any address
   that fits their elements; `*_bytes` is the capacity from the pointer on
   and must reach the end of the last row. */
typedef struct pk_block_norm_desc {
  uint32_t struct_size;          /* sizeof(pk_block_norm_desc) */
  const char *label;
  int32_t precision;             /* pk_precision of every matrix */
  int32_t kind;                  /* pk_norm_kind of both norms */
  uint32_t rows;                 /* 1 to PK_BLOCK_NORM_MAX_ROWS */
  uint32_t channels;             /* 1 to PK_BLOCK_NORM_MAX_CHANNELS */
  const void *input;             /* the block's output */
  uint64_t input_bytes;
  uint32_t input_stride;
  const float *gamma;            /* [channels] f32, NULL: no norm after the block */
  uint64_t gamma_bytes;          /* exactly 4 * channels */
  const float *beta;             /* [channels] f32 or NULL; needs gamma */
  uint64_t beta_bytes;
  const void *gate;              /* NULL: none */
  uint64_t gate_bytes;
  uint32_t gate_stride;
  uint32_t gate_rows;            /* row r takes gate row r / gate_rows; 0: gate row 0 for all */
  const void *residual;          /* NULL: none */
  uint64_t residual_bytes;
  uint32_t residual_stride;
  int32_t has_residual_scale;    /* 0: scale 1 */
  float residual_scale;          /* finite */
  void *output;
  uint64_t output_bytes;
  uint32_t output_stride;
  const float *next_gamma;       /* [channels] f32, with next_output */
  uint64_t next_gamma_bytes;
  const float *next_beta;        /* [channels] f32 or NULL */
  uint64_t next_beta_bytes;
  void *next_output;             /* NULL: none */
  uint64_t next_output_bytes;
  uint32_t next_output_stride;
  int32_t has_epsilon;           /* 0: epsilon 1e-5 */
  float epsilon;                 /* finite, >= 0 */
} pk_block_norm_desc;

/* Both outputs may be the input or the residual (the same pointer and
   stride), but not each other; any other overlap of an output with what the
   op reads is refused. Columns of one buffer (the same stride) do not
   overlap where their columns do not. */
int pk_block_norm_validate(const pk_block_norm_desc *desc);
int pk_block_norm_create(pk_context *ctx, const pk_block_norm_desc *desc, pk_block_norm_op **out);
/* The first `active_rows` rows (0 = all); rows behind them are left as they
   were. The op holds no workspace: it may be captured into graphs, and
   launches of it may overlap where their rows may. */
int pk_block_norm_enqueue(pk_block_norm_op *op, uint32_t active_rows, void *stream);
int pk_block_norm_enqueue_timed(pk_block_norm_op *op, uint32_t active_rows, void *stream, void *start_event,
                                void *end_event);
int pk_block_norm_destroy(pk_block_norm_op *op);
int pk_block_norm_release(pk_block_norm_op *op);

#ifdef __cplusplus
}
#endif

#endif
