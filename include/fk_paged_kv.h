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
 * (the angle's fraction of a turn is taken in fp64, the turn is fp32).
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

FK_PAGED_KV_API const char* fk_paged_kv_last_error(void);

FK_PAGED_KV_API int fk_paged_kv_append(const fk_paged_kv_append_args* args);

#ifdef __cplusplus
}
#endif

#endif /* FK_PAGED_KV_H_ */
