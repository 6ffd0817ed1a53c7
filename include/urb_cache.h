/*
 * urb_cache.h -- C ABI of paged key-value caches: the pages and slots of a step's new tokens, writing
 * keys and values into pages, attention of a request's new tokens over its pages, and the pages that
 * follow the beams of a search (urb_beams_select, urb_step.h).
 *
 * The reference (inspirewind/Urbilateria) keeps its caches on the CPU inside its model adapters; none
 * of the entry points mirrors one of its interfaces.  The conventions are urb_step.h's: every pointer
 * not named "host" is HBM memory on the current HIP device, calls only enqueue, a context belongs to
 * the device that was current when it was created (others return URB_ERR_ARGUMENT) and its calls are
 * stream-ordered and must not overlap on different streams.  Nothing is allocated by a call, so all of
 * them but the _create, _destroy and _sync functions may be captured into a HIP graph.  Graphs that
 * hold calls of one context must not run at the same time.
 */
#ifndef URB_CACHE_H
#define URB_CACHE_H

#include "urb_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- the cache of one layer ----
 *
 * `pages` pages of page_size tokens.  The values of key (value) head h of token i of page p start at
 * k (v) + p * page_stride + h * head_stride + i * token_stride values and are contiguous; K and V have
 * the same strides, so either may be a part of a wider buffer.  Slot s is token s % page_size of page
 * s / page_size.
 *
 * BF16 values, or E4M3 codes with one E8M0 scale for each token and head, [pages, heads, page_size]
 * contiguous: a value is its code times 2^(scale - 127).  Scales of 0 and 255 must not be used.
 *
 * pages 1 .. 2^24, heads 1 .. 1024, page_size 1 .. 1024, head_dim a multiple of 16 in 16 .. 256, less
 * than 2^36 bytes from the first value of K (of V) to the last, each stride (of an axis of more than one) at
 * least what the axes of smaller strides span, else URB_ERR_SHAPE; rows that start at multiples of 16 bytes,
 * BF16 or E4M3, scales with E4M3 and only there, else URB_ERR_ARGUMENT. */
typedef struct {
  void *k, *v;
  uint8_t *k_scales, *v_scales; /* E4M3 alone */
  urb_dtype dtype;              /* BF16, F8_E4M3 */
  uint32_t pages, heads, page_size, head_dim;
  uint64_t page_stride, head_stride, token_stride; /* in values */
} urb_kv_cache;

/* Rows of new keys and values, [tokens, heads, head_dim] each, in BF16 or f32: strides in values from
 * token to token and head to head, heads at multiples of 16 bytes (URB_ERR_ARGUMENT). */
typedef struct {
  const void *k, *v;
  urb_dtype dtype;
  uint64_t k_token_stride, k_head_stride, v_token_stride, v_head_stride;
} urb_kv_rows;

/* Writes token t's keys and values into slot slots[t] (i64); a slot that is not in the cache, such as
 * -1, skips its token.  Slots must differ from each other.  f32 values are rounded once to BF16.  In an
 * E4M3 cache a head's row is stored by the least power of two s >= 2^-100 with max |x| <= 448 s, its
 * codes x / s rounded to nearest even; a row that holds an infinity or a NaN is stored as NaN.
 * cache, rows: host structs, read by the call.  1 <= tokens < 2^24, else URB_ERR_SHAPE. */
urb_status urb_kv_append(const urb_kv_cache *cache, const urb_kv_rows *rows, const int64_t *slots,
                         uint32_t tokens, void *stream);

/* ---- pages ----
 *
 * A pager knows `pages` pages of page_size tokens, tables of up to max_rows rows of up to max_blocks
 * pages, and steps of up to max_tokens tokens (0: no plans).  The free pages are a stack that the
 * caller owns: free_pages [pages] (i32), of which the first *free_count are free; the last of them is
 * taken first.  Table row r holds in its column j the page of tokens j * page_size .. of row r; columns
 * past a row's length are neither read nor written.
 *
 * pages 1 .. 2^24, page_size 1 .. 1024, max_rows 1 .. 2^20, max_blocks 1 .. 2^20, max_tokens < 2^30,
 * max_rows * max_blocks < 2^31, max_blocks * page_size < 2^30, else URB_ERR_SHAPE. */
typedef struct {
  uint32_t pages, page_size, max_rows, max_blocks, max_tokens;
} urb_pager_desc;

typedef struct urb_pager urb_pager;

urb_status urb_pager_create(const urb_pager_desc *desc, urb_pager **out);
void urb_pager_destroy(urb_pager *pager);

/* The pages and slots of a step in which row r, of lengths[r] tokens so far, gets added[r] more (NULL:
 * one each).  Its missing pages are taken off the stack in the order of rows and columns and entered in
 * the table.  The new tokens lie behind each other in the order of the rows, starts[r] being the first
 * of row r and starts[rows] their number; for token t: token_rows[t] its row, positions[t] its place
 * in the row, slots[t] its slot.  Behind the last token, up to `tokens`: row -1, position 0, slot -1.
 *
 * A row for which pages are missing keeps its length and takes none, its tokens have slot -1, and the
 * next urb_pager_sync returns URB_ERR_OUT_OF_MEMORY (rows behind it that need no page are served).  A
 * row with a negative length or number, or of more than max_blocks pages, has no tokens in the step; a
 * row whose tokens do not all lie below `tokens` keeps those that do, with slot -1; an entry of the
 * table or the stack that is needed and is no page gives slot -1: URB_ERR_ARGUMENT by the next sync.  A
 * *free_count that is negative or above `pages` counts as 0 and is returned so, too.
 *
 * lengths_out may be lengths and free_count_out free_count; no other output may overlap anything.
 * starts, token_rows and positions may be NULL.  1 <= rows <= max_rows, 1 <= tokens <= max_tokens,
 * table_stride >= max_blocks, else URB_ERR_SHAPE. */
typedef struct {
  uint32_t rows, tokens;
  uint64_t table_stride; /* entries from row to row */
  const int32_t *lengths, *added;
  int32_t *tables;
  const int32_t *free_pages, *free_count;
  int32_t *lengths_out;    /* [rows] */
  int32_t *starts;         /* [rows + 1] */
  int32_t *token_rows;     /* [tokens] */
  int64_t *positions;      /* [tokens] */
  int64_t *slots;          /* [tokens] */
  int32_t *free_count_out; /* [1] */
} urb_page_plan;

urb_status urb_pager_plan(urb_pager *pager, const urb_page_plan *plan, void *stream);

/* Beams take over their parents' pages: of each request's `width` rows, row i becomes a copy of the
 * request's row parents[i] (0 .. width - 1) as it was, or ends with length 0 (negative).  Whole pages
 * are shared between rows of the same parent.  A page that its row fills in part stays with the lowest
 * of the parent's children; the others get a page of their own, with a copy of its tokens in each of the
 * caches.  Pages that no row of the request holds any more are put on the stack, in the order of
 * requests, columns and rows, before the new ones are taken off it, in the order of rows.  With all
 * parents negative a request ends and its pages are free.
 *
 * A page may stand in several rows of one request, in the same column, and in no two requests; one that
 * is filled in part in a row that has children (a prompt's last page in all the rows of a search that begins)
 * in no other row that has: such rows go on sharing it, and URB_ERR_ARGUMENT is returned by the next
 * sync.  A row for which no page is left ends with length 0, and the next urb_pager_sync returns
 * URB_ERR_OUT_OF_MEMORY.  A length that is negative or above max_blocks * page_size counts as 0, a parent
 * of `width` or more as negative, an entry that is no page is neither put on the stack nor copied, pages
 * beyond a full stack are left out, a *free_count out of range counts as 0: URB_ERR_ARGUMENT by the next
 * sync.
 *
 * The first max_blocks columns of tables_out must not overlap those of tables (URB_ERR_ARGUMENT);
 * lengths_out may be lengths, free_count_out free_count.  caches (host array) have the pager's pages and
 * page_size.  requests, width >= 1, width <= 64, requests * width <= max_rows, requests <= 4096, n_caches
 * <= 4096, both table strides >= max_blocks, else URB_ERR_SHAPE. */
typedef struct {
  uint32_t requests, width;
  uint64_t table_stride, table_out_stride;
  const int32_t *parents; /* [requests, width] */
  const int32_t *tables, *lengths;
  int32_t *tables_out, *lengths_out;
  int32_t *free_pages;
  const int32_t *free_count;
  int32_t *free_count_out;
  const urb_kv_cache *caches;
  uint32_t n_caches;
} urb_page_fork;

urb_status urb_pager_fork(urb_pager *pager, const urb_page_fork *fork, void *stream);

/* Waits for `stream` and returns the first of the failures latched since the previous urb_pager_sync
 * (URB_ERR_ARGUMENT before URB_ERR_OUT_OF_MEMORY; URB_OK if none), then clears them. */
urb_status urb_pager_sync(urb_pager *pager, void *stream);

/* ---- attention of new tokens ----
 *
 * For row r of lengths[r] cached tokens, its last `queries` ones among them, and query token i of them:
 *   e_j = exp(scale q . k_j),  o = sum_j e_j v_j / (exp(sink) + sum_j e_j)
 * over j < n = lengths[r] - (queries - 1 - i), and j >= n - window if window > 0; without sinks that
 * term is 0 (as with one of -inf; one of +inf leaves 0 of the values).  Query head h reads cache head
 * h / (q_heads / heads).  lse is the logarithm of the denominator; where that is 0, as with no j in reach, o
 * is 0 and lse -inf.  Tokens that no query of the row reaches are not used, whatever the cache holds there;
 * an infinity or a NaN that one of its queries reaches may come out of all of them, and either may come out
 * where queries, cached values, products q . k_j (before the scale) or sums e_j v_j reach 2^127.
 *
 * The products, sums and statistics are f32; the weights e are multiplied with 16 bits for BF16 rows and
 * with 24 for f32 rows, whose queries keep their 24 bits too.  A row's result may differ in its last bits
 * with the other rows of a call (they decide how its length is shared out), not between equal calls.
 *
 * A row's pages are read once for every sixteen queries of a cache head (queries * q_heads / heads of them).
 *
 * q_heads a multiple of heads, q_heads <= 8192, queries 1 .. 16, max_rows 1 .. 2^20, max_length
 * 1 .. 2^24, heads, page_size and head_dim as in urb_kv_cache, else URB_ERR_SHAPE; a scale that is not
 * finite, <= 0 or above 2^127 -> URB_ERR_INVALID_GEOMETRY. */
typedef struct {
  uint32_t q_heads, heads, head_dim, page_size;
  urb_dtype dtype;       /* of queries and outputs: BF16, F32 */
  urb_dtype cache_dtype; /* BF16, F8_E4M3 */
  uint32_t queries;      /* new tokens per row */
  uint32_t window;       /* 0: off */
  float scale;
  uint32_t max_rows, max_length;
} urb_attention_desc;

typedef struct urb_attention urb_attention;

urb_status urb_attention_create(const urb_attention_desc *desc, urb_attention **out);
void urb_attention_destroy(urb_attention *attention);

/* Queries and outputs, [rows, queries, q_heads, head_dim] each: strides in values; a head's values are
 * contiguous and start at a multiple of 16 bytes (URB_ERR_ARGUMENT).  out may be q itself (same address
 * and strides) and must not overlap it otherwise; strides of the output that are less than what the axes of
 * smaller strides span -> URB_ERR_SHAPE. */
typedef struct {
  uint32_t rows;
  const void *q;
  void *out;
  uint64_t q_row_stride, q_token_stride, q_head_stride;
  uint64_t out_row_stride, out_token_stride, out_head_stride;
  const int32_t *tables; /* [rows, >= the pages of max_length] */
  uint64_t table_stride;
  const int32_t *lengths; /* [rows] */
  const float *sinks;     /* [q_heads], or NULL */
  float *lse;             /* [rows, queries, q_heads], or NULL */
} urb_attention_call;

/* One call.  A length that is negative or above max_length counts as 0, and a table entry in reach that
 * is no page of the cache as tokens out of reach: URB_ERR_ARGUMENT by the next urb_attention_sync.
 * 1 <= rows <= max_rows, table_stride >= the pages of max_length, a cache of the context's heads,
 * head_dim, page_size and type, else URB_ERR_SHAPE. */
urb_status urb_attend(urb_attention *attention, const urb_kv_cache *cache,
                      const urb_attention_call *call, void *stream);

/* Waits for `stream` and returns the failure latched since the previous urb_attention_sync (URB_OK if
 * none), then clears it. */
urb_status urb_attention_sync(urb_attention *attention, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* URB_CACHE_H */
