// The paged-KV operators of this build behind the module's conventions: raw device addresses and a
// stream handle, std::invalid_argument for arguments, std::runtime_error for CUDA errors.
#pragma once

#include <cstdint>

namespace fast_kernels::paged_kv {

// New keys and values into their pages (fk_paged_kv_append in include/fk_paged_kv.h).
void paged_kv_append_forward(
    std::uintptr_t keys_ptr, std::uintptr_t values_ptr, std::int64_t key_token_stride, std::int64_t key_head_stride,
    std::int64_t value_token_stride, std::int64_t value_head_stride, std::uintptr_t key_pages_ptr,
    std::uintptr_t value_pages_ptr, std::uintptr_t key_scales_ptr, std::uintptr_t value_scales_ptr,
    std::uintptr_t segments_ptr, int num_segments, int num_tokens, int num_pages, int num_kv_heads, int head_dim,
    int page_size, int kv_format, int rotate_keys, float rope_theta, std::uintptr_t stream_ptr);

// Causal attention of prompt tokens over pages (fk_paged_kv_attention, partial results added up).
void paged_attention_forward(
    std::uintptr_t query_ptr, std::int64_t query_row_stride, std::int64_t query_head_stride, std::uintptr_t key_ptr,
    std::uintptr_t value_ptr, std::uintptr_t key_scales_ptr, std::uintptr_t value_scales_ptr,
    std::uintptr_t page_ids_ptr, std::uintptr_t vectors_ptr, std::uintptr_t items_ptr, std::uintptr_t output_ptr,
    std::uintptr_t partials_ptr, int num_rows, int num_page_ids, int num_vectors, int num_items, int num_partials,
    int num_pages, int num_q_heads, int num_kv_heads, int head_dim, int page_size, int kv_format, float softmax_scale,
    float rope_theta, std::uintptr_t stream_ptr);

// Decode behind shared runs of pages: the runs' items (fk_paged_kv_attention), then every request's own
// tokens merged with them (fk_page_decode_forward_merged). Uses no scratch of this layer's own: calls on several
// streams, and captured ones, do not share any.
void shared_prefix_decode_forward(
    std::uintptr_t query_ptr, std::uintptr_t key_ptr, std::uintptr_t value_ptr, std::uintptr_t key_scales_ptr,
    std::uintptr_t value_scales_ptr, std::uintptr_t page_ids_ptr, std::uintptr_t vectors_ptr, std::uintptr_t items_ptr,
    std::uintptr_t of_request_ptr, std::uintptr_t run_base_pages_ptr, std::uintptr_t run_page_counts_ptr,
    std::uintptr_t run_logical_starts_ptr, std::uintptr_t run_last_page_lens_ptr,
    std::uintptr_t request_run_offsets_ptr, std::uintptr_t seq_lens_ptr, std::uintptr_t output_ptr,
    std::uintptr_t partials_ptr, int batch, int num_page_ids, int num_items, int num_partials, int num_runs,
    int max_tail_pages, int num_pages, int num_q_heads, int num_kv_heads, int head_dim, int page_size, int kv_format,
    float softmax_scale, float rope_theta, std::uintptr_t stream_ptr);

int paged_kv_device_status();

}  // namespace fast_kernels::paged_kv
