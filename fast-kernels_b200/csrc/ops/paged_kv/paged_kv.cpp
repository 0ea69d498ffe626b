// C++ launchers over the C ABI of libfk_paged_kv.so.
#include "ops/paged_kv/paged_kv.h"

#include <stdexcept>
#include <string>

#include "fk_page_decode.h"
#include "fk_paged_kv.h"

namespace fast_kernels::paged_kv {
namespace {

void raise_if_failed(int code) {
  if (code == FK_PAGED_KV_OK) {
    return;
  }
  const std::string message = fk_paged_kv_last_error();
  if (code == FK_PAGED_KV_ERR_INVALID_ARGUMENT) {
    throw std::invalid_argument(message);
  }
  throw std::runtime_error(message);
}

template <typename T>
T* as(std::uintptr_t value) {
  return reinterpret_cast<T*>(value);
}

}  // namespace

void paged_kv_append_forward(
    std::uintptr_t keys_ptr, std::uintptr_t values_ptr, std::int64_t key_token_stride, std::int64_t key_head_stride,
    std::int64_t value_token_stride, std::int64_t value_head_stride, std::uintptr_t key_pages_ptr,
    std::uintptr_t value_pages_ptr, std::uintptr_t key_scales_ptr, std::uintptr_t value_scales_ptr,
    std::uintptr_t segments_ptr, int num_segments, int num_tokens, int num_pages, int num_kv_heads, int head_dim,
    int page_size, int kv_format, int rotate_keys, float rope_theta, std::uintptr_t stream_ptr) {
  fk_paged_kv_append_args args{};
  args.keys = as<const void>(keys_ptr);
  args.values = as<const void>(values_ptr);
  args.key_token_stride = key_token_stride;
  args.key_head_stride = key_head_stride;
  args.value_token_stride = value_token_stride;
  args.value_head_stride = value_head_stride;
  args.key_pages = as<void>(key_pages_ptr);
  args.value_pages = as<void>(value_pages_ptr);
  args.key_scales = as<float>(key_scales_ptr);
  args.value_scales = as<float>(value_scales_ptr);
  args.segments = as<const int32_t>(segments_ptr);
  args.num_segments = num_segments;
  args.num_tokens = num_tokens;
  args.num_pages = num_pages;
  args.num_kv_heads = num_kv_heads;
  args.head_dim = head_dim;
  args.page_size = page_size;
  args.kv_format = kv_format;
  args.rotate_keys = rotate_keys;
  args.rope_theta = rope_theta;
  args.stream = as<void>(stream_ptr);
  raise_if_failed(fk_paged_kv_append(&args));
}

void paged_attention_forward(
    std::uintptr_t query_ptr, std::int64_t query_row_stride, std::int64_t query_head_stride, std::uintptr_t key_ptr,
    std::uintptr_t value_ptr, std::uintptr_t key_scales_ptr, std::uintptr_t value_scales_ptr,
    std::uintptr_t page_ids_ptr, std::uintptr_t vectors_ptr, std::uintptr_t items_ptr, std::uintptr_t output_ptr,
    std::uintptr_t partials_ptr, int num_rows, int num_page_ids, int num_vectors, int num_items, int num_partials,
    int num_pages, int num_q_heads, int num_kv_heads, int head_dim, int page_size, int kv_format, float softmax_scale,
    float rope_theta, std::uintptr_t stream_ptr) {
  fk_paged_kv_attention_args args{};
  args.query = as<const void>(query_ptr);
  args.query_row_stride = query_row_stride;
  args.query_head_stride = query_head_stride;
  args.key_pages = as<const void>(key_ptr);
  args.value_pages = as<const void>(value_ptr);
  args.key_scales = as<const float>(key_scales_ptr);
  args.value_scales = as<const float>(value_scales_ptr);
  args.page_ids = as<const int32_t>(page_ids_ptr);
  args.vectors = as<const int32_t>(vectors_ptr);
  args.items = as<const int32_t>(items_ptr);
  args.output = as<void>(output_ptr);
  args.partials = as<float>(partials_ptr);
  args.num_rows = num_rows;
  args.num_page_ids = num_page_ids;
  args.num_vectors = num_vectors;
  args.num_items = num_items;
  args.num_partials = num_partials;
  args.num_pages = num_pages;
  args.num_q_heads = num_q_heads;
  args.num_kv_heads = num_kv_heads;
  args.head_dim = head_dim;
  args.page_size = page_size;
  args.kv_format = kv_format;
  args.combine = 1;
  args.softmax_scale = softmax_scale;
  args.rope_theta = rope_theta;
  args.stream = as<void>(stream_ptr);
  raise_if_failed(fk_paged_kv_attention(&args));
}

void shared_prefix_decode_forward(
    std::uintptr_t query_ptr, std::uintptr_t key_ptr, std::uintptr_t value_ptr, std::uintptr_t key_scales_ptr,
    std::uintptr_t value_scales_ptr, std::uintptr_t page_ids_ptr, std::uintptr_t vectors_ptr, std::uintptr_t items_ptr,
    std::uintptr_t of_request_ptr, std::uintptr_t run_base_pages_ptr, std::uintptr_t run_page_counts_ptr,
    std::uintptr_t run_logical_starts_ptr, std::uintptr_t run_last_page_lens_ptr,
    std::uintptr_t request_run_offsets_ptr, std::uintptr_t seq_lens_ptr, std::uintptr_t output_ptr,
    std::uintptr_t partials_ptr, int batch, int num_page_ids, int num_items, int num_partials, int num_runs,
    int max_tail_pages, int num_pages, int num_q_heads, int num_kv_heads, int head_dim, int page_size, int kv_format,
    float softmax_scale, float rope_theta, std::uintptr_t stream_ptr) {
  if (num_items <= 0 || num_partials <= 0) {
    throw std::invalid_argument("shared_prefix_decode: items and partial results come together");
  }
  fk_page_decode_args tail{};
  tail.query = as<const void>(query_ptr);
  tail.key_pages = as<const void>(key_ptr);
  tail.value_pages = as<const void>(value_ptr);
  tail.key_scales = as<const float>(key_scales_ptr);
  tail.value_scales = as<const float>(value_scales_ptr);
  tail.run_base_pages = as<const int32_t>(run_base_pages_ptr);
  tail.run_page_counts = as<const int32_t>(run_page_counts_ptr);
  tail.run_logical_starts = as<const int32_t>(run_logical_starts_ptr);
  tail.run_last_page_lens = as<const int32_t>(run_last_page_lens_ptr);
  tail.request_run_offsets = as<const int32_t>(request_run_offsets_ptr);
  tail.seq_lens = as<const int32_t>(seq_lens_ptr);
  tail.output = as<void>(output_ptr);
  tail.batch = batch;
  tail.num_runs = num_runs;
  tail.num_q_heads = num_q_heads;
  tail.num_kv_heads = num_kv_heads;
  tail.head_dim = head_dim;
  tail.page_size = page_size;
  tail.kv_format = kv_format;
  tail.keys_are_rotated = 1;
  tail.splits = 0;  // without a workspace: what merges through shared memory
  tail.max_pages_hint = max_tail_pages;
  tail.softmax_scale = softmax_scale;
  tail.rope_theta = rope_theta;
  tail.stream = as<void>(stream_ptr);

  fk_paged_kv_attention_args args{};
  args.query = tail.query;
  args.query_row_stride = static_cast<int64_t>(num_q_heads) * head_dim;
  args.query_head_stride = head_dim;
  args.key_pages = tail.key_pages;
  args.value_pages = tail.value_pages;
  args.key_scales = tail.key_scales;
  args.value_scales = tail.value_scales;
  args.page_ids = as<const int32_t>(page_ids_ptr);
  args.vectors = as<const int32_t>(vectors_ptr);
  args.items = as<const int32_t>(items_ptr);
  args.output = tail.output;
  args.partials = as<float>(partials_ptr);
  args.num_rows = batch;
  args.num_page_ids = num_page_ids;
  args.num_vectors = batch;
  args.num_items = num_items;
  args.num_partials = num_partials;
  args.num_pages = num_pages;
  args.num_q_heads = num_q_heads;
  args.num_kv_heads = num_kv_heads;
  args.head_dim = head_dim;
  args.page_size = page_size;
  args.kv_format = kv_format;
  args.softmax_scale = softmax_scale;
  args.rope_theta = rope_theta;
  args.stream = tail.stream;
  raise_if_failed(fk_paged_kv_attention(&args));
  const fk_page_decode_prior prior{as<const float>(partials_ptr), as<const int32_t>(of_request_ptr)};
  const int code = fk_page_decode_forward_merged(&tail, &prior);
  if (code == FK_PAGE_DECODE_ERR_INVALID_ARGUMENT) {
    throw std::invalid_argument(fk_page_decode_last_error());
  }
  if (code != FK_PAGE_DECODE_OK) {
    throw std::runtime_error(fk_page_decode_last_error());
  }
}

int paged_kv_device_status() {
  int status = 0;
  raise_if_failed(fk_paged_kv_device_status(&status));
  return status;
}

}  // namespace fast_kernels::paged_kv
