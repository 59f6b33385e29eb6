/*
 * pk_score.h - C ABI of token scores on gfx950: from rows of logits the log
 * probability of a given token, the entropy of the row and its best
 * alternatives, in one pass over the logits. Same library, contexts, streams,
 * events and status codes as pk_palette.h. No counterpart in the reference,
 * whose decoder returns the tokens it chose and no measure of how sure it was
 * (tdt-decoder.ts:84-130). The caller brings the logits, of a head product
 * (pk_q4.h, pk_palette.h) for instance: pk_tdt.h keeps those of its decoder to
 * itself. Token and duration columns of one head row are two bindings.
 *
 * With z = logits / temperature over the V columns of a row,
 *   log p = z - log(sum exp z),   entropy = -sum p log p   (nats),
 * in f32 from the stored logits: with m = max z and r the sum of exp(z - m)
 * over all columns but one of value m, log(sum exp z) = m + log1p(r), and the
 * entropy log1p(r) + sum exp(z - m) (m - z) / (1 + r) adds two terms that
 * are not negative, so both keep their digits where one token is certain.
 */
#ifndef PK_SCORE_H
#define PK_SCORE_H

#include "pk_palette.h"

#ifdef __cplusplus
extern "C" {
#endif

#define PK_SCORE_NO_TOKEN 0xffffffffu
#define PK_SCORE_MAX_ALTERNATIVES 32u
#define PK_SCORE_MAX_ROWS 4194303u
#define PK_SCORE_MAX_COLUMNS 1073741824u

typedef struct pk_score_op pk_score_op;

typedef struct pk_score_desc {
  uint32_t struct_size;          /* sizeof(pk_score_desc) */
  const char *label;
  int32_t precision;             /* pk_precision of the logits */
  uint32_t rows;                 /* 1 to PK_SCORE_MAX_ROWS */
  uint32_t columns;              /* V, 1 to PK_SCORE_MAX_COLUMNS; the logits may start at any element */
  uint32_t row_stride;           /* elements from row to row (0: columns) */
  const void *logits;
  uint64_t logits_bytes;         /* capacity from the pointer to the end of the last row */
  int32_t has_temperature;       /* 0: temperature 1 */
  float temperature;             /* 2^-20 to 2^20 */
  const uint32_t *tokens;        /* [rows], with log_probs */
  uint64_t tokens_bytes;
  float *log_probs;              /* [rows], or NULL */
  uint64_t log_probs_bytes;
  float *entropies;              /* [rows], or NULL */
  uint64_t entropies_bytes;
  uint32_t alternatives;         /* 0 to PK_SCORE_MAX_ALTERNATIVES */
  uint32_t *top_tokens;          /* [rows, alternatives], best first, equal logits by index */
  uint64_t top_tokens_bytes;
  float *top_log_probs;          /* [rows, alternatives] */
  uint64_t top_log_probs_bytes;
} pk_score_desc;

/* What a row gives where the formulas do not say:
   - a token of PK_SCORE_NO_TOKEN (a padded position) has log probability 0,
     any other token of `columns` or more NaN; neither is read;
   - a logit of minus infinity (a masked token) has probability 0: its log
     probability is minus infinity and it is never an alternative. Places
     beyond the last possible alternative hold PK_SCORE_NO_TOKEN and minus
     infinity. The type's lowest number masks too, but counts as an
     alternative, and rows that it leaves few others take several times as
     long;
   - a row of minus infinities has entropy 0, no alternatives, and log
     probability minus infinity for every token;
   - a row with a NaN or plus infinity has NaN for its entropy and every log
     probability (PK_SCORE_NO_TOKEN: 0); its alternatives are ordered by
     their logits without the NaNs.
   Outputs must not overlap each other or the inputs. */
int pk_score_validate(const pk_score_desc *desc);
int pk_score_create(pk_context *ctx, const pk_score_desc *desc, pk_score_op **out);
/* The first `active_rows` rows (0 = all); outputs of the rows behind them are
   left as they were. May be captured into graphs. Rows split over several
   workgroups (long ones, when there are few) meet in memory of the op:
   launches of one op, eager or replayed, must be ordered by the caller, as
   their outputs ask for anyway. */
int pk_score_enqueue(pk_score_op *op, uint32_t active_rows, void *stream);
int pk_score_enqueue_timed(pk_score_op *op, uint32_t active_rows, void *stream, void *start_event, void *end_event);
int pk_score_destroy(pk_score_op *op);
int pk_score_release(pk_score_op *op);

#ifdef __cplusplus
}
#endif

#endif
