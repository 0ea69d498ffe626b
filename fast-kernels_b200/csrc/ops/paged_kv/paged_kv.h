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

}  // namespace fast_kernels::paged_kv
