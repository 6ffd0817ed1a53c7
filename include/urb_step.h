/*
 * urb_step.h -- C ABI of the steps of a decoder on either side of the MoE block call
 * (urb_moe_forward_block, urb_moe.h): projections with low-rank adapters of many requests, the
 * norm of every query and key head with the position rotation, sampling from logits, and beam search's
 * selection.  The cache between them and its attention: urb_cache.h.
 *
 * The reference (inspirewind/Urbilateria) runs these steps on the CPU inside its model adapters;
 * none of the entry points mirrors one of its interfaces.  The conventions are urb_moe.h's: plain
 * pointers and sizes, every pointer not named "host" is HBM memory on the current HIP device,
 * `stream` is a hipStream_t passed as void* (NULL = the default stream), calls only enqueue, and
 * a context's calls are stream-ordered and must not overlap on different streams.  A context
 * belongs to the device that was current when it was created; a call made while another device
 * is current returns URB_ERR_ARGUMENT.  Nothing is allocated by a call, so all of them but the
 * _create, _destroy and _sync functions and urb_proj_set_adapter from host memory may be captured
 * into a HIP graph.
 *
 * Rows are BF16 or f32 (urb_dtype's URB_DTYPE_BF16 and URB_DTYPE_F32; others return
 * URB_ERR_ARGUMENT); sums and intermediate values are f32 or wider and are rounded once, to the
 * output's type.  Values are not checked for being finite: a row with an infinity or a NaN has
 * such outputs, and no other row is touched by it.
 */
#ifndef URB_STEP_H
#define URB_STEP_H

#include "urb_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- projections with low-rank adapters ----
 *
 * y[t] = W x[t] + scale_a B_a (A_a x[t]),  a = adapter_ids[t]
 *
 * W [rows, cols] is one packed matrix for all tokens (urb_format; kept in the panel layout of
 * urb_pack_matrix), A_a [rank_a, cols] and B_a [rows, rank_a] are BF16 and live in numbered slots
 * of the context, in HBM from urb_proj_set_adapter on.  A x is carried in f32.  f32 values and A x
 * are multiplied with all their 24 bits, as far as these lie at 2^-133 (BF16's least) or above.
 *
 * rows % 16 == 0 and cols % 128 == 0 (the panel layout), rows <= 2^20, cols <= 32768, max_tokens
 * 1 .. 2^30, adapter_slots <= 4096 and max_rank <= 256 (both 0, or neither), else URB_ERR_SHAPE. */
typedef struct {
  uint32_t rows;          /* outputs per token */
  uint32_t cols;          /* inputs per token */
  urb_format format;      /* of the matrix */
  urb_dtype x_dtype;      /* of the tokens' rows: BF16, F32 */
  urb_dtype y_dtype;      /* of the outputs: BF16, F32 */
  uint32_t max_tokens;    /* the most that one call may pass */
  uint32_t adapter_slots; /* 0 = no adapters */
  uint32_t max_rank;      /* the largest rank that a slot can hold */
} urb_proj_desc;

typedef struct {
  const uint16_t *a; /* [rank, cols] BF16, row-major */
  const uint16_t *b; /* [rows, rank] BF16, row-major */
  uint32_t rank;     /* 1 .. max_rank */
  float scale;       /* finite */
} urb_adapter;

typedef struct urb_proj_ctx urb_proj_ctx;

/* Builds a projection: the matrix is uploaded and laid out (HOST, DEVICE_COPY) or used in place
 * (DEVICE_BORROW: panel layout, must outlive the context) and its payload validated, as
 * urb_moe_create does: E8M0 0xFF -> URB_ERR_INVALID_SCALE, E4M3 NaN codes or non-finite BF16 ->
 * URB_ERR_NONFINITE. */
urb_status urb_proj_create(const urb_proj_desc *desc, const urb_matrix *weight,
                           urb_weight_source source, urb_proj_ctx **out);
void urb_proj_destroy(urb_proj_ctx *ctx);

/* Puts an adapter into a slot (in place of what is there), or empties it (adapter NULL).  The
 * change is ordered on `stream`: calls made before it there use the slot's previous content.  From
 * device memory (DEVICE_COPY) nothing waits, and a and b may be reused once the stream has passed;
 * HOST memory is uploaded before the call returns.  A non-finite value in a or b empties the slot
 * and is returned as URB_ERR_NONFINITE by the next urb_proj_sync.  A slot or rank out of range
 * -> URB_ERR_SHAPE; a scale that is not finite -> URB_ERR_NONFINITE; DEVICE_BORROW ->
 * URB_ERR_ARGUMENT (the slot has a layout of its own). */
urb_status urb_proj_set_adapter(urb_proj_ctx *ctx, uint32_t slot, const urb_adapter *adapter,
                                urb_weight_source source, void *stream);

/* One call over `tokens` rows: x [tokens, cols] with x_stride values from row to row, y [tokens,
 * rows] with y_stride.  adapter_ids [tokens] (i32): the slot of each row, negative = none; NULL =
 * none for all.  An id that names no filled slot gives the row W x alone and is returned as
 * URB_ERR_ARGUMENT by the next urb_proj_sync.  1 <= tokens <= max_tokens, x_stride >= cols,
 * y_stride >= rows, else URB_ERR_SHAPE.  x rows must start at multiples of 16 bytes (URB_ERR_
 * ARGUMENT); y may start at any value.  y must not overlap x. */
urb_status urb_proj_forward(urb_proj_ctx *ctx, const void *x, uint64_t x_stride,
                            const int32_t *adapter_ids, uint32_t tokens, void *y,
                            uint64_t y_stride, void *stream);

/* Waits for `stream` and returns the first of the failures latched since the previous
 * urb_proj_sync (URB_ERR_NONFINITE before URB_ERR_ARGUMENT; URB_OK if none), then clears them. */
urb_status urb_proj_sync(urb_proj_ctx *ctx, void *stream);

/* HBM bytes the context holds for the matrix (0 when borrowed), the adapter slots and workspace. */
urb_status urb_proj_memory(const urb_proj_ctx *ctx, size_t *weight_bytes, size_t *adapter_bytes,
                           size_t *workspace_bytes);

/* ---- norms of queries and keys with the position rotation ----
 *
 * For every token and head, with h the head's head_dim values:
 *   n_i = h_i / sqrt(mean(h^2) + eps) * w_i          (zero_centered: 1 + w_i, as in
 *                                                     urb_zc_rms_norm_bf16)
 * and the first rotary_dim values turned in pairs by angle = position * inv_freq[i]:
 *   (n_a, n_b) -> (n_a cos - n_b sin, n_b cos + n_a sin)
 * where pair i is values (i, i + rotary_dim / 2), or (2i, 2i + 1) if interleaved; the other values
 * are n_i.  The angle is an f64 product, so far positions keep their fraction; the norm is not
 * rounded before the rotation.  The squares are summed in f32 (values of 2^60 and more overflow it), and
 * |position * inv_freq| must stay below 2^40, where the product still has 2^-13 of a radian.
 *
 * head_dim 2 .. 1024 and even, rotary_dim even and <= head_dim (0 = no rotation), q_heads >= 1,
 * q_heads + k_heads <= 65535, tokens * (q_heads + k_heads) < 2^31, else URB_ERR_SHAPE; eps not finite or <= 0 ->
 * URB_ERR_INVALID_GEOMETRY.  Strides are in values, from token to token and head to head; a head's
 * values are contiguous.  Heads may be parts of a wider buffer (a fused q/k/v row); an output may
 * be its own input (same address and strides) and must not overlap an input or the other output
 * otherwise; strides by which the heads of an output overlap each other -> URB_ERR_SHAPE. */
typedef struct {
  urb_dtype dtype; /* of q, k and the outputs: BF16, F32 */
  uint32_t q_heads, k_heads;
  uint32_t head_dim, rotary_dim;
  int32_t interleaved;
  int32_t zero_centered;
  float eps;
  uint64_t q_token_stride, q_head_stride;
  uint64_t k_token_stride, k_head_stride;
  uint64_t q_out_token_stride, q_out_head_stride;
  uint64_t k_out_token_stride, k_out_head_stride;
} urb_qk_desc;

/* q, k, q_out, k_out as the descriptor (host memory, read by the call) says; q_weight, k_weight
 * [head_dim] f32; positions [tokens] i64; inv_freq [rotary_dim / 2] f32 (may be NULL with
 * rotary_dim 0, as positions).  k, k_weight and k_out are not read with k_heads 0.  tokens 0 ->
 * URB_ERR_SHAPE.  Heads that start at multiples of 16 bytes, with head_dim (and, unless
 * interleaved, rotary_dim) a multiple of 16, take a kernel of wide loads; others one of single
 * values. */
urb_status urb_qk_norm_rope(const urb_qk_desc *desc, const void *q, const void *k,
                            const float *q_weight, const float *k_weight,
                            const int64_t *positions, const float *inv_freq, uint32_t tokens,
                            void *q_out, void *k_out, void *stream);

/* ---- sampling ----
 *
 * For each row of logits l, with m its largest value, temperature tau and e_i = exp((l_i - m)/tau):
 *   1. the order is by descending logit, equal ones by ascending index;
 *   2. top_k > 0 keeps its first top_k tokens;
 *   3. top_p < 1 keeps the shortest beginning of those whose sum of e reaches top_p times theirs;
 *   4. min_p > 0 keeps of those the tokens with e_i >= min_p;
 *   5. the first token is always kept; the draw takes the smallest index i at which the sum of e
 *      over the kept tokens of index <= i exceeds uniform times the sum over all kept ones.
 * tau = 0 takes the lowest index of the largest logit.  NaN logits count as -inf and are never
 * drawn; a row with nothing above -inf gives id -1 and probability 0.  With logits of +inf the draw
 * is among those.  e is computed in f64 and enters the sums as the nearest multiple of 2^-min(51, 62 -
 * ceil(log2(vocab))): 2^-42 of the largest for 2^20 tokens, 2^-45 for 131072.  Sums of integers do
 * not depend on their order, so a result depends on nothing but the row and its parameters; tokens
 * below half of that unit are never drawn.
 *
 * vocab 1 .. 2^20, max_rows 1 .. 2^24, else URB_ERR_SHAPE. */
typedef struct {
  uint32_t vocab;
  uint32_t max_rows;
  urb_dtype dtype; /* of the logits: BF16, F32 */
} urb_sampler_desc;

/* One value per row, or NULL: temperature 1, top_k 0 (off), top_p 1 (off), min_p 0 (off). */
typedef struct {
  const float *temperature; /* finite, >= 0 */
  const int32_t *top_k;     /* <= 0 or >= vocab: off */
  const float *top_p;       /* > 0; >= 1: off */
  const float *min_p;       /* 0 .. 1 */
} urb_sample_params;

typedef struct urb_sampler urb_sampler;

urb_status urb_sampler_create(const urb_sampler_desc *desc, urb_sampler **out);
void urb_sampler_destroy(urb_sampler *sampler);

/* Draws one token per row of logits [rows, vocab] (row_stride values from row to row, any
 * alignment) with the given uniform [rows] f32 in [0, 1): ids [rows] i32 and, unless NULL, the
 * drawn tokens' probabilities among the kept ones [rows] f32.  params: host struct of device
 * pointers, or NULL for all defaults.  A row whose parameters or uniform are outside the ranges
 * above gives id -1 and probability 0 and is returned as URB_ERR_ARGUMENT by the next urb_sampler_
 * sync.  1 <= rows <= max_rows and row_stride >= vocab, else URB_ERR_SHAPE. */
urb_status urb_sample(urb_sampler *sampler, const void *logits, uint64_t row_stride, uint32_t rows,
                      const urb_sample_params *params, const float *uniform, int32_t *ids,
                      float *probs, void *stream);

/* Waits for `stream` and returns the failure latched since the previous urb_sampler_sync (URB_OK
 * if none), then clears it. */
urb_status urb_sampler_sync(urb_sampler *sampler, void *stream);

/* ---- beam search's selection ----
 *
 * For each request, over its `width` beams b with scores c_b and rows of logits l: the candidates (b, v)
 * of score
 *   c_b + ((l_v - m) - log(sum_i exp(l_i - m))),  m = the row's largest logit
 * (l_v - m is 0 where both are +inf), and of a beam that has ended only (b, end_token), of score c_b.  The
 * `picks` best are taken: by descending score, equal ones by ascending b * vocab + v.  Scores are compared
 * in f64, where those of different logits of a beam may be equal too (under a score of -1e12, or of logits of
 * nearly 0).  NaN logits count as -inf, and nothing of score -inf, or below f32's range, is taken: missing
 * picks have score -inf, token -1 and parent -1.  A beam of score -inf is not there (of a search that begins,
 * all but one are).
 *
 * vocab 1 .. 2^18, width 1 .. 32, picks 1 .. 64, max_requests 1 .. 65535, else URB_ERR_SHAPE. */
typedef struct {
  uint32_t vocab;
  uint32_t width;        /* beams of a request */
  uint32_t picks;
  uint32_t max_requests;
  urb_dtype dtype;       /* of the logits: BF16, F32 */
} urb_beams_desc;

typedef struct urb_beams urb_beams;

urb_status urb_beams_create(const urb_beams_desc *desc, urb_beams **out);
void urb_beams_destroy(urb_beams *beams);

/* logits [requests * width, vocab], row_stride values from row to row, any alignment; scores and ended
 * [requests, width] (ended NULL: none; else not 0 for a beam that has); scores_out, tokens, parents (0 ..
 * width - 1) and ended_out (NULL, or 1 where the parent had ended, the token is end_token or the pick is
 * missing) [requests, picks].  end_token 0 .. vocab - 1, or -1 for none where ended is NULL, else
 * URB_ERR_ARGUMENT.  With picks = width, scores_out may be scores and ended_out ended; no other output may
 * overlap anything.  A score that is NaN or +inf counts as -inf and is returned as URB_ERR_ARGUMENT by the
 * next urb_beams_sync.  1 <= requests <= max_requests, row_stride >= vocab, else URB_ERR_SHAPE. */
typedef struct {
  const void *logits;
  uint64_t row_stride;
  uint32_t requests;
  int32_t end_token;
  const float *scores;
  const int32_t *ended;
  float *scores_out;
  int32_t *tokens, *parents, *ended_out;
} urb_beams_call;

urb_status urb_beams_select(urb_beams *beams, const urb_beams_call *call, void *stream);

/* Waits for `stream` and returns the failure latched since the previous urb_beams_sync (URB_OK if
 * none), then clears it. */
urb_status urb_beams_sync(urb_beams *beams, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* URB_STEP_H */
