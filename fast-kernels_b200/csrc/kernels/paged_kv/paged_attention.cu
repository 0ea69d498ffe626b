// extern "C" entry points of the attention over lists of pages: validation, launch.
#include <algorithm>
#include <cmath>
#include <mutex>

#include "paged_attention.cuh"

namespace fk_paged_kv {

__device__ int g_paged_kv_status = 0;

namespace {

constexpr int kMaxDevices = 64;

// Address of the status word on the current device; asked for once per device.
int status_word(int** out) {
  static std::mutex mutex;
  static int* table[kMaxDevices];
  int device = 0;
  cudaError_t err = cudaGetDevice(&device);
  if (err != cudaSuccess) {
    return fail_cuda("cudaGetDevice", err);
  }
  if (device < 0 || device >= kMaxDevices) {
    return fail(FK_PAGED_KV_ERR_CUDA, "device ordinal out of range");
  }
  std::lock_guard<std::mutex> lock(mutex);
  if (table[device] == nullptr) {
    void* address = nullptr;
    err = cudaGetSymbolAddress(&address, g_paged_kv_status);
    if (err != cudaSuccess) {
      return fail_cuda("cudaGetSymbolAddress", err);
    }
    table[device] = static_cast<int*>(address);
  }
  *out = table[device];
  return FK_PAGED_KV_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

cudaError_t launch_items(const AttentionParams& params, int head_dim, int kv_format, int num_items, cudaStream_t stream) {
  if (head_dim == 64) {
    return kv_format == kKvBf16 ? launch_attention_d64_bf16(params, num_items, stream)
           : kv_format == kKvFp8 ? launch_attention_d64_fp8(params, num_items, stream)
                                 : launch_attention_d64_int8(params, num_items, stream);
  }
  return kv_format == kKvBf16 ? launch_attention_d128_bf16(params, num_items, stream)
         : kv_format == kKvFp8 ? launch_attention_d128_fp8(params, num_items, stream)
                               : launch_attention_d128_int8(params, num_items, stream);
}

cudaError_t launch_combine(const AttentionParams& params, int head_dim, cudaStream_t stream) {
  cudaLaunchConfig_t config{};
  const long long warps = static_cast<long long>(params.num_vectors) * params.num_q_heads;
  config.gridDim = dim3(static_cast<unsigned>((warps + 7) / 8), 1, 1);
  config.blockDim = dim3(256, 1, 1);
  config.stream = stream;
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attribute;
  config.numAttrs = 1;
  return head_dim == 64 ? cudaLaunchKernelEx(&config, combine_partials_kernel<64>, params)
                        : cudaLaunchKernelEx(&config, combine_partials_kernel<128>, params);
}

}  // namespace
}  // namespace fk_paged_kv

using namespace fk_paged_kv;

extern "C" {

FK_PAGED_KV_API int fk_paged_kv_attention(const fk_paged_kv_attention_args* args) {
  if (args == nullptr) {
    return fail(FK_PAGED_KV_ERR_INVALID_ARGUMENT, "args must not be NULL");
  }
  const fk_paged_kv_attention_args& a = *args;
  if (a.head_dim != 64 && a.head_dim != 128) {
    return fail(FK_PAGED_KV_ERR_INVALID_ARGUMENT, "paged attention only supports head_dim 64 or 128");
  }
  if (a.page_size != 16 && a.page_size != 32) {
    return fail(FK_PAGED_KV_ERR_INVALID_ARGUMENT, "paged attention only supports page_size 16 or 32");
  }
  if (a.kv_format != kKvBf16 && a.kv_format != kKvFp8 && a.kv_format != kKvInt8) {
    return fail(FK_PAGED_KV_ERR_INVALID_ARGUMENT, "unsupported kv_format");
  }
  if (a.num_q_heads <= 0 || a.num_kv_heads <= 0 || a.num_q_heads % a.num_kv_heads != 0) {
    return fail(FK_PAGED_KV_ERR_INVALID_ARGUMENT, "num_q_heads must be divisible by num_kv_heads");
  }
  if (a.num_q_heads / a.num_kv_heads > FK_PAGED_KV_ITEM_ROWS) {
    return fail(FK_PAGED_KV_ERR_INVALID_ARGUMENT, "more than 256 query heads per kv head");
  }
  if (a.num_rows < 0 || a.num_page_ids < 0 || a.num_vectors < 0 || a.num_items < 0 || a.num_partials < 0 ||
      a.num_pages < 0) {
    return fail(FK_PAGED_KV_ERR_INVALID_ARGUMENT, "counts must be non-negative");
  }
  if (!std::isfinite(a.softmax_scale) || !(a.rope_theta > 0.0f) || !std::isfinite(a.rope_theta)) {
    return fail(FK_PAGED_KV_ERR_INVALID_ARGUMENT, "softmax_scale must be finite and rope_theta positive");
  }
  if (a.num_vectors == 0 || a.num_items == 0) {
    return FK_PAGED_KV_OK;
  }
  if (a.query == nullptr || a.key_pages == nullptr || a.value_pages == nullptr || a.page_ids == nullptr ||
      a.vectors == nullptr || a.items == nullptr || a.output == nullptr) {
    return fail(FK_PAGED_KV_ERR_INVALID_ARGUMENT, "query, pages, page_ids, vectors, items and output must not be NULL");
  }
  if (a.num_pages == 0 || static_cast<long long>(a.num_pages) * a.num_kv_heads * a.page_size > 0x7fffffffLL) {
    return fail(FK_PAGED_KV_ERR_INVALID_ARGUMENT, "num_pages * num_kv_heads * page_size must be positive and fit 31 bits");
  }
  if (static_cast<long long>(a.num_vectors) * a.num_q_heads > 0x7fffffffLL) {
    return fail(FK_PAGED_KV_ERR_INVALID_ARGUMENT, "num_vectors * num_q_heads must fit 31 bits");
  }
  if (a.num_partials > 0 && a.partials == nullptr) {
    return fail(FK_PAGED_KV_ERR_INVALID_ARGUMENT, "partials must not be NULL when num_partials > 0");
  }
  if (a.kv_format != kKvBf16 && (a.key_scales == nullptr || a.value_scales == nullptr)) {
    return fail(FK_PAGED_KV_ERR_INVALID_ARGUMENT, "quantised pages need key_scales and value_scales");
  }
  if (!aligned16(a.query) || !aligned16(a.key_pages) || !aligned16(a.value_pages) || !aligned16(a.vectors) ||
      !aligned16(a.items) || !aligned16(a.output) || !aligned16(a.partials) ||
      (a.kv_format != kKvBf16 && !aligned16(a.value_scales))) {
    return fail(FK_PAGED_KV_ERR_INVALID_ARGUMENT,
                "query, pages, value_scales, vectors, items, output and partials must be 16-byte aligned");
  }
  // (a page's key scales are one load; a cache that starts inside another one's scales has no more alignment than that)
  const uintptr_t scale_bytes = sizeof(float) * (a.head_dim / 64);
  if (a.kv_format != kKvBf16 && (reinterpret_cast<uintptr_t>(a.key_scales) & (scale_bytes - 1)) != 0) {
    return fail(FK_PAGED_KV_ERR_INVALID_ARGUMENT, "key_scales must be aligned to the head_dim / 64 scales of a page");
  }
  if (((a.query_row_stride | a.query_head_stride) & 7) != 0) {
    return fail(FK_PAGED_KV_ERR_INVALID_ARGUMENT, "strides of the query must be multiples of 8 elements");
  }
  AttentionParams params{};
  if (const int code = status_word(&params.status); code != FK_PAGED_KV_OK) {
    return code;
  }
  params.query = static_cast<const uint16_t*>(a.query);
  params.query_row_stride = a.query_row_stride;
  params.query_head_stride = a.query_head_stride;
  params.key_pages = static_cast<const uint8_t*>(a.key_pages);
  params.value_pages = static_cast<const uint8_t*>(a.value_pages);
  params.key_scales = a.key_scales;
  params.value_scales = a.value_scales;
  params.page_ids = a.page_ids;
  params.vectors = reinterpret_cast<const int4*>(a.vectors);
  params.items = reinterpret_cast<const int4*>(a.items);
  params.output = static_cast<uint16_t*>(a.output);
  params.partials = a.partials;
  params.num_rows = a.num_rows;
  params.num_page_ids = a.num_page_ids;
  params.num_vectors = a.num_vectors;
  params.num_partials = a.num_partials;
  params.num_pages = a.num_pages;
  params.num_q_heads = a.num_q_heads;
  params.num_kv_heads = a.num_kv_heads;
  params.group = a.num_q_heads / a.num_kv_heads;
  params.page_size = a.page_size;
  params.scale_log2e = static_cast<float>(static_cast<double>(a.softmax_scale) * 1.4426950408889634);
  fill_rope_table(&params.rope, a.head_dim, a.rope_theta);
  const cudaStream_t stream = static_cast<cudaStream_t>(a.stream);
  cudaError_t err = launch_items(params, a.head_dim, a.kv_format, a.num_items, stream);
  if (err == cudaSuccess && a.combine != 0 && a.num_partials > 0) {
    err = launch_combine(params, a.head_dim, stream);
  }
  return err == cudaSuccess ? FK_PAGED_KV_OK : fail_cuda("paged attention launch", err);
}

FK_PAGED_KV_API int fk_paged_kv_device_status(int* status) {
  if (status == nullptr) {
    return fail(FK_PAGED_KV_ERR_INVALID_ARGUMENT, "status must not be NULL");
  }
  int* word = nullptr;
  if (const int code = status_word(&word); code != FK_PAGED_KV_OK) {
    return code;
  }
  int value = 0;
  cudaError_t err = cudaMemcpy(&value, word, sizeof value, cudaMemcpyDeviceToHost);
  if (err == cudaSuccess && value != 0) {
    err = cudaMemset(word, 0, sizeof value);
  }
  if (err != cudaSuccess) {
    return fail_cuda("device status", err);
  }
  *status = value;
  return FK_PAGED_KV_OK;
}

}  // extern "C"
