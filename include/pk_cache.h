/*
 * pk_cache.h - C ABI of a paged cache of keys and values on gfx950: the
 * append of new tokens with the rotation of their positions, and the attention
 * of new tokens over the cache. Same library, contexts, streams, events and
 * status codes as pk_palette.h. No counterpart in the reference, whose
 * attention (attention.ts:418-727; pk_attention.h) sees one window of frames
 * and keeps nothing.
 *
 * Sequence s has the rows [row_starts[s], row_starts[s + 1]) of the batch,
 * n of them: its newest tokens. lengths[s] counts its tokens with these, so
 * that row i of the n has the position lengths[s] - n + i. Token t lies in
 * place t mod page_size of page page_table[s][t / page_size]. A cache is
 * [pages][kv_heads][page_size][head_dim] of the profile's type, page_stride
 * elements from page to page; keys and values may be halves of the pages of
 * one buffer. A page may stand in several tables, or several times in one, as
 * long as no two new tokens go to the same place of it.
 *
 * These arrays lie on the device and are read by every launch: a replayed
 * graph follows what they hold then. What they hold is kept within the
 * bindings: row_starts are cut to `rows` and should not decrease; a row before
 * position 0 (n above the length) is neither appended nor rotated, its query
 * output is left as it was, and it attends to nothing if causal, or else, as
 * all rows of its sequence, to what that holds; a token whose page is
 * PK_CACHE_NO_PAGE or any other number of `pages` or more, or that lies behind
 * pages_per_sequence pages, is not stored and is hidden from every row.
 *
 * cache append: with j < rotary_dim / 2 and the angle a = position *
 * frequencies[j], the elements x, y of a head of the queries and keys that lie
 * at j and rotary_dim / 2 + j (PK_ROTARY_HALVES) or at 2j and 2j + 1
 * (PK_ROTARY_NEIGHBOURS) become
 *   x cos a - y sin a,  y cos a + x sin a
 * in f32, rounded once; the angle is reduced exactly, at any position and for
 * frequencies of up to 2^36 in magnitude. The other elements, and the values,
 * are copied.
 *
 * cache attention: head h reads the kv head h / (heads / kv_heads);
 *   z = scale * q . k, or cap * tanh(scale * q . k / cap),
 *   output = sum exp(z) v / sum exp(z)
 * over the tokens that the row sees: of the first lengths[s], those up to its
 * own position if causal, and of these the last `window`. Sums, maxima and
 * exponentials are f32; f16 rows round the exponentials to f16 for their
 * product with the values, where those below 2^-32 of the largest so far
 * are 0, in the sum they are not. A row that sees
 * nothing, or only scores of minus infinity, gives zeros. What a row does not
 * see, infinities and NaN included, does not touch it; values that it does see
 * and that are infinite or NaN, and scores beyond 2^23, make its block of rows
 * many times slower.
 * Scores beyond f32 and sums of f32 values beyond 2^119 overflow.
 * How the work is shared out follows the op's rows over the launch's active
 * sequences, which the host knows, and not row_starts: hold one op for single
 * tokens and one for chunks.
 */
#ifndef PK_CACHE_H
#define PK_CACHE_H

#include "pk_palette.h"

#ifdef __cplusplus
extern "C" {
#endif

#define PK_CACHE_NO_PAGE 0xffffffffu
#define PK_CACHE_MAX_ROWS 1048576u
#define PK_CACHE_MAX_SEQUENCES 4096u
#define PK_CACHE_MAX_HEADS 1024u
#define PK_CACHE_MAX_HEAD_DIM 256u
#define PK_CACHE_MAX_PAGE_SIZE 65536u
#define PK_CACHE_MAX_TOKENS 1073741824u           /* page_size * pages_per_sequence */
#define PK_CACHE_MAX_BYTES (64ull << 30)          /* of one cache binding's extent */
#define PK_CACHE_MAX_UNITS 4000000u               /* attention: rows * heads / 16 + kv_heads * min(sequences, rows) */

typedef enum pk_rotary_kind {
  PK_ROTARY_HALVES = 0,
  PK_ROTARY_NEIGHBOURS = 1,
} pk_rotary_kind;

typedef struct pk_cache_append_op pk_cache_append_op;
typedef struct pk_cache_attention_op pk_cache_attention_op;

/* Rows of queries, keys, values and outputs are [heads][head_dim] elements, a
   row `*_stride` elements after the one before (0: packed), at any address
   that fits their elements; `*_bytes` is the capacity from the pointer on and
   must reach the end of the last row, or of the last page. */
typedef struct pk_cache_append_desc {
  uint32_t struct_size;          /* sizeof(pk_cache_append_desc) */
  const char *label;
  int32_t precision;             /* pk_precision of rows and caches */
  uint32_t rows;                 /* that the bindings hold: 1 to PK_CACHE_MAX_ROWS */
  uint32_t sequences;            /* 1 to PK_CACHE_MAX_SEQUENCES */
  uint32_t heads;                /* of the queries; 0: no queries */
  uint32_t kv_heads;             /* 1 to PK_CACHE_MAX_HEADS */
  uint32_t head_dim;             /* a multiple of 8 up to PK_CACHE_MAX_HEAD_DIM */
  const void *queries;           /* with query_output, or NULL */
  uint64_t queries_bytes;
  uint32_t query_stride;
  void *query_output;            /* may be the queries (the same pointer and stride) */
  uint64_t query_output_bytes;
  uint32_t query_output_stride;
  const void *keys;
  uint64_t keys_bytes;
  uint32_t key_stride;
  const void *values;
  uint64_t values_bytes;
  uint32_t value_stride;
  uint32_t rotary_dim;           /* even, up to head_dim; 0: no rotation */
  int32_t rotary;                /* pk_rotary_kind */
  const float *frequencies;      /* [rotary_dim / 2] radians per position, with rotary_dim; up to 2^36 */
  uint64_t frequencies_bytes;
  const uint32_t *positions;     /* [rows] of the rotation, NULL: those in the sequence */
  uint64_t positions_bytes;
  const uint32_t *row_starts;    /* [sequences + 1] */
  uint64_t row_starts_bytes;
  const uint32_t *lengths;       /* [sequences] */
  uint64_t lengths_bytes;
  const uint32_t *page_table;    /* [sequences, pages_per_sequence] */
  uint64_t page_table_bytes;
  uint32_t pages_per_sequence;
  uint32_t pages;                /* of a cache */
  uint32_t page_size;            /* tokens, 1 to PK_CACHE_MAX_PAGE_SIZE */
  uint64_t page_stride;          /* elements from page to page, a multiple of 8 (0: packed) */
  void *key_cache;               /* aligned to 16 bytes */
  uint64_t key_cache_bytes;
  void *value_cache;
  uint64_t value_cache_bytes;
} pk_cache_append_desc;

/* Outputs and caches must not overlap each other or what the op reads, but
   for query_output on the queries' own rows. */
int pk_cache_append_validate(const pk_cache_append_desc *desc);
int pk_cache_append_create(pk_context *ctx, const pk_cache_append_desc *desc, pk_cache_append_op **out);
/* The rows of the first `active_sequences` sequences (0 = all); rows behind
   them, and places of the caches that no row goes to, are left as they were.
   The op holds no workspace and may be captured into graphs. */
int pk_cache_append_enqueue(pk_cache_append_op *op, uint32_t active_sequences, void *stream);
int pk_cache_append_enqueue_timed(pk_cache_append_op *op, uint32_t active_sequences, void *stream, void *start_event,
                                  void *end_event);
int pk_cache_append_destroy(pk_cache_append_op *op);
int pk_cache_append_release(pk_cache_append_op *op);

typedef struct pk_cache_attention_desc {
  uint32_t struct_size;          /* sizeof(pk_cache_attention_desc) */
  const char *label;
  int32_t precision;             /* pk_precision of rows and caches */
  uint32_t rows;                 /* that the bindings hold: 1 to PK_CACHE_MAX_ROWS */
  uint32_t sequences;            /* 1 to PK_CACHE_MAX_SEQUENCES */
  uint32_t heads;                /* a multiple of kv_heads up to PK_CACHE_MAX_HEADS */
  uint32_t kv_heads;
  uint32_t head_dim;             /* a multiple of 8 up to PK_CACHE_MAX_HEAD_DIM */
  const void *queries;
  uint64_t queries_bytes;
  uint32_t query_stride;
  void *output;
  uint64_t output_bytes;
  uint32_t output_stride;
  int32_t causal;                /* 1: a row sees tokens up to its own position; 0: all */
  uint32_t window;               /* causal: the last so many tokens, its own among them; 0: all */
  int32_t has_scale;             /* 0: scale 1 / sqrt(head_dim) */
  float scale;                   /* -2^60 to 2^60 */
  float score_cap;               /* 0: none; 2^-20 to 2^20 */
  const uint32_t *row_starts;    /* [sequences + 1] */
  uint64_t row_starts_bytes;
  const uint32_t *lengths;       /* [sequences] */
  uint64_t lengths_bytes;
  const uint32_t *page_table;    /* [sequences, pages_per_sequence] */
  uint64_t page_table_bytes;
  uint32_t pages_per_sequence;
  uint32_t pages;                /* of a cache */
  uint32_t page_size;            /* tokens, 1 to PK_CACHE_MAX_PAGE_SIZE */
  uint64_t page_stride;          /* elements from page to page, a multiple of 8 (0: packed) */
  const void *key_cache;         /* aligned to 16 bytes */
  uint64_t key_cache_bytes;
  const void *value_cache;
  uint64_t value_cache_bytes;
} pk_cache_attention_desc;

/* The output must not overlap what the op reads. */
int pk_cache_attention_validate(const pk_cache_attention_desc *desc);
int pk_cache_attention_create(pk_context *ctx, const pk_cache_attention_desc *desc, pk_cache_attention_op **out);
/* The rows of the first `active_sequences` sequences (0 = all); rows behind
   them are left as they were. May be captured into graphs. Long sequences
   are split over workgroups, which meet in memory of the op, where lists of
   more than 64 sequences lie as well: launches of one op, eager or replayed,
   must be ordered by the caller, as their outputs ask for anyway. */
int pk_cache_attention_enqueue(pk_cache_attention_op *op, uint32_t active_sequences, void *stream);
int pk_cache_attention_enqueue_timed(pk_cache_attention_op *op, uint32_t active_sequences, void *stream,
                                     void *start_event, void *end_event);
int pk_cache_attention_destroy(pk_cache_attention_op *op);
int pk_cache_attention_release(pk_cache_attention_op *op);

#ifdef __cplusplus
}
#endif

#endif
