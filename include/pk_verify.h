/*
 * pk_verify.h - C ABI of the verification of drafted tokens on gfx950: from
 * the target model's rows of logits for a chunk of drafted tokens, how many
 * of them stand and which token follows. Same library, contexts, streams,
 * events and status codes as pk_palette.h. No counterpart in the reference,
 * whose decoder takes one token at a time (tdt-decoder.ts:1740-2010). The
 * caller brings the logits, of a head product (pk_q4.h, pk_palette.h) over the
 * rows of pk_cache.h's attention for instance; pk_score.h scores them.
 *
 * Sequence s has the rows [row_starts[s], row_starts[s + 1]) of the batch:
 * tokens[row] is the token that was fed at a row, and each row but a
 * sequence's last judges the draft d = tokens[row + 1]. A draft that is no
 * column (PK_VERIFY_NO_TOKEN for instance) is none: its row is the
 * sequence's last, and what follows it is not read.
 *
 * PK_VERIFY_SAMPLE: with p = softmax(target / temperature) and q =
 * softmax(draft / temperature) of a row, or q = 1 at d and 0 elsewhere without
 * draft logits, d is accepted if uniforms[row] * q(d) < p(d). The next token
 * is drawn at the first row whose draft is not accepted from w = max(p - q, 0),
 * or at the last row from w = p: the first whose running sum of w, in the order
 * of the columns, exceeds draws[s] times the whole sum. So drafts that were
 * drawn from q give tokens distributed as p. Probabilities and their sums are
 * f64, so that these decisions do not hang on the order of the sums. A
 * probability under 2^-990 counts as 0.
 * PK_VERIFY_GREEDY: d is accepted if it is the row's best logit, the lowest
 * of equal ones, and the next token is the best of the row that ends; draft
 * logits, the temperature, uniforms and draws are not read.
 */
#ifndef PK_VERIFY_H
#define PK_VERIFY_H

#include "pk_palette.h"

#ifdef __cplusplus
extern "C" {
#endif

#define PK_VERIFY_NO_TOKEN 0xffffffffu
#define PK_VERIFY_MAX_ROWS 1048576u
#define PK_VERIFY_MAX_SEQUENCES 65535u
#define PK_VERIFY_MAX_COLUMNS 16777216u

typedef enum pk_verify_mode {
  PK_VERIFY_SAMPLE = 0,
  PK_VERIFY_GREEDY = 1,
} pk_verify_mode;

typedef struct pk_verify_op pk_verify_op;

typedef struct pk_verify_desc {
  uint32_t struct_size;          /* sizeof(pk_verify_desc) */
  const char *label;
  int32_t precision;             /* pk_precision of both logits */
  int32_t mode;                  /* pk_verify_mode */
  uint32_t rows;                 /* that the bindings hold: 1 to PK_VERIFY_MAX_ROWS */
  uint32_t sequences;            /* 1 to PK_VERIFY_MAX_SEQUENCES */
  uint32_t columns;              /* V, 1 to PK_VERIFY_MAX_COLUMNS; logits may start at any element */
  const void *target;            /* [rows, columns] */
  uint64_t target_bytes;         /* capacity from the pointer to the end of the last row */
  uint32_t target_stride;        /* elements from row to row (0: columns) */
  const void *draft;             /* [rows, columns], what row + 1's token was drawn from; NULL: none */
  uint64_t draft_bytes;
  uint32_t draft_stride;
  int32_t has_temperature;       /* 0: temperature 1 */
  float temperature;             /* 2^-20 to 2^20 */
  const uint32_t *row_starts;    /* [sequences + 1], cut to `rows`; should not decrease */
  uint64_t row_starts_bytes;
  const uint32_t *tokens;        /* [rows] */
  uint64_t tokens_bytes;
  const float *uniforms;         /* [rows] of [0, 1); may be NULL if greedy */
  uint64_t uniforms_bytes;
  const float *draws;            /* [sequences] of [0, 1); likewise */
  uint64_t draws_bytes;
  uint32_t *accepted;            /* [sequences] */
  uint64_t accepted_bytes;
  uint32_t *next_tokens;         /* [sequences] */
  uint64_t next_tokens_bytes;
} pk_verify_desc;

/* What the formulas do not say:
   - a logit of minus infinity has probability 0;
   - w that is 0 everywhere (p nowhere above q, by rounding) is replaced by p;
   - a row of the target with a NaN, plus infinity or only minus infinities
     accepts nothing and gives PK_VERIFY_NO_TOKEN, and so does such a row of
     the draft if its sequence gets to it; greedy leaves out NaN and takes
     plus infinity as the best, and a row without another number gives
     PK_VERIFY_NO_TOKEN;
   - uniforms and draws outside [0, 1) or NaN: a uniform accepts or refuses as
     the formula says, NaN refuses; a draw of 1 or more, or NaN, gives the last
     token with w above 0, a negative one the first;
   - a sequence without rows accepts 0 and gives PK_VERIFY_NO_TOKEN.
   Outputs must not overlap each other or the inputs. */
int pk_verify_validate(const pk_verify_desc *desc);
int pk_verify_create(pk_context *ctx, const pk_verify_desc *desc, pk_verify_op **out);
/* The first `active_sequences` sequences (0 = all); outputs of the others are
   left as they were. May be captured into graphs. Rows meet in memory of the
   op: launches of one op, eager or replayed, must be ordered by the caller, as
   their outputs ask for anyway. */
int pk_verify_enqueue(pk_verify_op *op, uint32_t active_sequences, void *stream);
int pk_verify_enqueue_timed(pk_verify_op *op, uint32_t active_sequences, void *stream, void *start_event,
                            void *end_event);
int pk_verify_destroy(pk_verify_op *op);
int pk_verify_release(pk_verify_op *op);

#ifdef __cplusplus
}
#endif

#endif
