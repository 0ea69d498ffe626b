// C++ launchers over the C ABI of libfk_paged_kv.so.
#include "ops/paged_kv/paged_kv.h"

#include <stdexcept>
#include <string>

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

}  // namespace fast_kernels::paged_kv
