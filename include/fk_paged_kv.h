/*
 * fk_paged_kv.h -- C ABI of the operators around the paged KV cache for B200 (sm_100a): what fills
 * the pages that fk_page_decode.h reads.
 *
 * Page layouts are those of fk_page_decode.h:
 *
 *   key_pages    [pages, num_kv_heads, page_size, head_dim]          bf16 | e4m3 | int8
 *   value_pages  same shape and type as key_pages
 *   key_scales   [pages, num_kv_heads, head_dim / 64]                fp32, NULL for bf16 pages
 *   value_scales [pages, num_kv_heads, page_size, head_dim / 64]     fp32, NULL for bf16 pages
 *
 * head_dim is 64 or 128, page_size 16 or 32. All pointers are device pointers unless a comment says
 * otherwise. Calls are asynchronous on `stream`, which belongs to the current device. Plain C: no
 * C++ or framework types cross this boundary, and nothing is thrown through it.
 */
#ifndef FK_PAGED_KV_H_
#define FK_PAGED_KV_H_

#include <stddef.h>
#include <stdint.h>

#if defined(__GNUC__)
#define FK_PAGED_KV_API __attribute__((visibility("default")))
#else
#define FK_PAGED_KV_API
#endif

#ifdef __cplusplus
extern "C" {
#endif

#define FK_PAGED_KV_OK 0
#define FK_PAGED_KV_ERR_INVALID_ARGUMENT (-1) /* std::invalid_argument / ValueError */
#define FK_PAGED_KV_ERR_CUDA (-2)             /* a CUDA call failed: std::runtime_error */

/* The page formats, as in fk_page_decode.h. */
#define FK_PAGED_KV_BF16 0
#define FK_PAGED_KV_FP8_E4M3 1
#define FK_PAGED_KV_INT8 2

/* Writes the keys and values of new tokens into their pages.
 *
 * A segment is a run of consecutive new tokens that go to one page: `segments` holds
 * [num_segments][4] int32 = physical page, first slot | token count << 16, row of the first token in
 * `keys` / `values`, position of the first token. No two segments of a call name the same page. A
 * segment that does not fit the page, the pool or the rows is left out.
 *
 * With rotate_keys != 0 dimensions 2i and 2i + 1 of a key are turned by position * theta^(-2i/head_dim)
 * (the angle's fraction of a turn is taken in 64-bit fixed point, the turn is fp32).
 *   bf16 pages: the turned key is rounded once; values are copied.
 *   8-bit pages, L = 127 (int8) or 448 (e4m3): a value is stored as round(v / s) with
 *   s = max(max|v| / L, 1e-6) over the token's 64-dim block. A key block's scale belongs to the page:
 *   s' = max(s, max|k| / L, 1e-6), where s is the scale that the page holds, or 0 if the segment
 *   starts at slot 0 (whatever a reused page held is gone). Where s' > s, the elements q of the slots
 *   before the segment become round(q s / s'). Slots behind the segment are left as they are.
 *   Scales are fp32, rounding is to nearest even; keys and values must be finite. */
typedef struct fk_paged_kv_append_args {
  const void* keys;   /* bf16 rows [num_tokens][num_kv_heads][head_dim], strides below, 16-byte aligned rows */
  const void* values;
  int64_t key_token_stride; /* in elements, multiples of 8 */
  int64_t key_head_stride;
  int64_t value_token_stride;
  int64_t value_head_stride;
  void* key_pages;
  void* value_pages;
  float* key_scales;
  float* value_scales;
  const int32_t* segments;
  int32_t num_segments;
  int32_t num_tokens;
  int32_t num_pages;
  int32_t num_kv_heads;
  int32_t head_dim;
  int32_t page_size;
  int32_t kv_format;
  int32_t rotate_keys;
  float rope_theta;
  void* stream;
} fk_paged_kv_append_args;

/* Attention of query vectors over lists of pages, cut into items by the caller.
 *
 * A vector is one token's query: `vectors` holds [num_vectors][4] int32 = row in `query` and `output`,
 * position, first partial result, number of partial results. An item is a run of vectors and one kv
 * head over a range of tokens: `items` holds [num_items][8] int32 = first vector, number of vectors,
 * kv head, entry of `page_ids` that holds token 0, first token (a multiple of page_size), end token,
 * causal, partial result. Token t lies in page page_ids[entry + t / page_size], slot t % page_size. A
 * vector of the item sees tokens first .. end - 1, with causal != 0 only those at or before its
 * position:
 *     logit_t = softmax_scale * < R(position) q , k_t >,   sum_t softmax(logit)_t * v_t
 * The keys in the pages carry their rotation already; R turns dimensions 2i and 2i + 1 as in
 * fk_paged_kv_append. A vector that sees nothing gets zeros. number of vectors *
 * (num_q_heads / num_kv_heads) is at most FK_PAGED_KV_ITEM_ROWS.
 *
 * An item whose partial result is -1 writes its rows of `output` and must be the only one of its
 * vectors and kv head. Otherwise it leaves, per vector and query head, the weighted values, the
 * maximum of the logits in units of ln 2 and the denominator at
 *     partials[(first partial of the vector + partial result of the item) * num_q_heads + q_head]
 * (rows of head_dim + 4 floats: values, maximum, denominator, two unused; any number serves as the maximum
 * that values and denominator are relative to). With `combine` != 0 a second
 * kernel adds the partial results of every vector that has some, in order, into `output`; without it
 * the caller hands them to fk_page_decode_forward_merged.
 *
 * The positions of a causal item's vectors ascend. An item that does not fit the arrays, or ends behind
 * FK_PAGED_KV_MAX_TOKENS, is left out.
 *
 * Rounding. Logits, maxima, denominators and weighted values are fp32. bf16 pages: the turned query and the
 * probabilities are rounded to bf16 once. 8-bit pages: the turned query is rounded to fp16 behind an
 * exact power of two; keys and values are fp16 numbers, exact in the 64-dim block that has the page's
 * (token's) larger scale, the other block's times the ratio of the two scales (off by up to 2^-10 of itself down
 * to a ratio of 2^-21, by 2^-8 at 2^-24, and lost at 2^-32); a probability times its
 * token's larger value scale is rounded to fp16 relative to the row's heaviest, so that one below 2^-21
 * of it is off by up to 2^-32 of it. A non-finite key or value of a token that counts may reach every
 * vector of an item; what lies behind a request's last token is never used. Results do not depend on
 * timing. */
#define FK_PAGED_KV_ITEM_ROWS 256
#define FK_PAGED_KV_MAX_TOKENS (0x7fffffff - 127) /* of an item's end token */
typedef struct fk_paged_kv_attention_args {
  const void* query; /* bf16 rows [rows][num_q_heads][head_dim], strides below, 16-byte aligned rows */
  int64_t query_row_stride; /* in elements, multiples of 8 */
  int64_t query_head_stride;
  const void* key_pages;
  const void* value_pages;
  const float* key_scales;
  const float* value_scales;
  const int32_t* page_ids;
  const int32_t* vectors;
  const int32_t* items;
  void* output; /* bf16 [rows][num_q_heads][head_dim], contiguous */
  float* partials;
  int32_t num_rows; /* of query and output */
  int32_t num_page_ids;
  int32_t num_vectors;
  int32_t num_items;
  int32_t num_partials;
  int32_t num_pages;
  int32_t num_q_heads;
  int32_t num_kv_heads;
  int32_t head_dim;
  int32_t page_size;
  int32_t kv_format;
  int32_t combine;
  float softmax_scale;
  float rope_theta;
  void* stream;
} fk_paged_kv_attention_args;

FK_PAGED_KV_API const char* fk_paged_kv_last_error(void);

FK_PAGED_KV_API int fk_paged_kv_attention(const fk_paged_kv_attention_args* args);

/* Reads and clears the device status word of the current device: 0 = fine, 1 = a bounded wait inside a
 * kernel gave up (the outputs of that call are not valid). */
FK_PAGED_KV_API int fk_paged_kv_device_status(int* status);

FK_PAGED_KV_API int fk_paged_kv_append(const fk_paged_kv_append_args* args);

#ifdef __cplusplus
}
#endif

#endif /* FK_PAGED_KV_H_ */
