// extern "C" entry points of include/fk_paged_kv.h that every operator of the library uses, and the
// append: validation, launch.
#include <cmath>

#include "paged_kv_append.cuh"

namespace fk_paged_kv {
namespace {
thread_local std::string t_last_error;

cudaError_t launch(const void* kernel, int blocks, void** arguments, cudaStream_t stream) {
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(blocks), 1, 1);
  config.blockDim = dim3(kAppendWarps * 32, 1, 1);
  config.stream = stream;
  // Programmatic dependent launch: the kernel waits for its predecessor before it reads memory.
  cudaLaunchAttribute attribute{};
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attribute;
  config.numAttrs = 1;
  return cudaLaunchKernelExC(&config, kernel, arguments);
}

template <int D, int PS, int KV>
const void* kernel_for(bool rotate) {
  return rotate ? reinterpret_cast<const void*>(paged_kv_append_kernel<D, PS, KV, true>)
                : reinterpret_cast<const void*>(paged_kv_append_kernel<D, PS, KV, false>);
}
template <int D, int PS>
const void* kernel_for(int kv_format, bool rotate) {
  return kv_format == kKvBf16 ? kernel_for<D, PS, kKvBf16>(rotate)
         : kv_format == kKvFp8 ? kernel_for<D, PS, kKvFp8>(rotate) : kernel_for<D, PS, kKvInt8>(rotate);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace

int fail(int code, const std::string& message) {
  t_last_error = message;
  return code;
}
int fail_cuda(const char* what, cudaError_t err) {
  return fail(FK_PAGED_KV_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(err));
}

}  // namespace fk_paged_kv

using namespace fk_paged_kv;

extern "C" {

FK_PAGED_KV_API const char* fk_paged_kv_last_error(void) { return t_last_error.c_str(); }

FK_PAGED_KV_API int fk_paged_kv_append(const fk_paged_kv_append_args* args) {
  if (args == nullptr) {
    return fail(FK_PAGED_KV_ERR_INVALID_ARGUMENT, "args must not be NULL");
  }
  const fk_paged_kv_append_args& a = *args;
  if (a.head_dim != 64 && a.head_dim != 128) {
    return fail(FK_PAGED_KV_ERR_INVALID_ARGUMENT, "paged_kv_append only supports head_dim 64 or 128");
  }
  if (a.page_size != 16 && a.page_size != 32) {
    return fail(FK_PAGED_KV_ERR_INVALID_ARGUMENT, "paged_kv_append only supports page_size 16 or 32");
  }
  if (a.kv_format != kKvBf16 && a.kv_format != kKvFp8 && a.kv_format != kKvInt8) {
    return fail(FK_PAGED_KV_ERR_INVALID_ARGUMENT, "unsupported kv_format");
  }
  if (a.num_kv_heads <= 0 || a.num_segments < 0 || a.num_tokens < 0 || a.num_pages < 0) {
    return fail(FK_PAGED_KV_ERR_INVALID_ARGUMENT, "num_kv_heads must be positive, the other counts non-negative");
  }
  if (a.rotate_keys != 0 && (!(a.rope_theta > 0.0f) || !std::isfinite(a.rope_theta))) {
    return fail(FK_PAGED_KV_ERR_INVALID_ARGUMENT, "rope_theta must be positive and finite");
  }
  if (a.num_segments == 0) {
    return FK_PAGED_KV_OK;
  }
  if (a.keys == nullptr || a.values == nullptr || a.key_pages == nullptr || a.value_pages == nullptr ||
      a.segments == nullptr) {
    return fail(FK_PAGED_KV_ERR_INVALID_ARGUMENT, "keys, values, pages and segments must not be NULL");
  }
  if (a.kv_format != kKvBf16 && (a.key_scales == nullptr || a.value_scales == nullptr)) {
    return fail(FK_PAGED_KV_ERR_INVALID_ARGUMENT, "quantised pages need key_scales and value_scales");
  }
  if (!aligned16(a.keys) || !aligned16(a.values) || !aligned16(a.key_pages) || !aligned16(a.value_pages) ||
      !aligned16(a.segments)) {
    return fail(FK_PAGED_KV_ERR_INVALID_ARGUMENT, "keys, values, pages and segments must be 16-byte aligned");
  }
  if ((reinterpret_cast<uintptr_t>(a.key_scales) & 3u) != 0 || (reinterpret_cast<uintptr_t>(a.value_scales) & 3u) != 0) {
    return fail(FK_PAGED_KV_ERR_INVALID_ARGUMENT, "scales must be 4-byte aligned");
  }
  if (((a.key_token_stride | a.key_head_stride | a.value_token_stride | a.value_head_stride) & 7) != 0) {
    return fail(FK_PAGED_KV_ERR_INVALID_ARGUMENT, "strides of keys and values must be multiples of 8 elements");
  }
  AppendParams params{};
  params.keys = static_cast<const uint16_t*>(a.keys);
  params.values = static_cast<const uint16_t*>(a.values);
  params.key_token_stride = a.key_token_stride;
  params.key_head_stride = a.key_head_stride;
  params.value_token_stride = a.value_token_stride;
  params.value_head_stride = a.value_head_stride;
  params.key_pages = static_cast<uint8_t*>(a.key_pages);
  params.value_pages = static_cast<uint8_t*>(a.value_pages);
  params.key_scales = a.key_scales;
  params.value_scales = a.value_scales;
  params.segments = reinterpret_cast<const int4*>(a.segments);
  params.num_tokens = a.num_tokens;
  params.num_pages = a.num_pages;
  params.num_kv_heads = a.num_kv_heads;
  const bool rotate = a.rotate_keys != 0;
  if (rotate) {
    fill_rope_table(&params.rope, a.head_dim, a.rope_theta);
  }
  const void* kernel = a.head_dim == 64 ? (a.page_size == 16 ? kernel_for<64, 16>(a.kv_format, rotate)
                                                             : kernel_for<64, 32>(a.kv_format, rotate))
                                        : (a.page_size == 16 ? kernel_for<128, 16>(a.kv_format, rotate)
                                                             : kernel_for<128, 32>(a.kv_format, rotate));
  void* arguments[] = {&params};
  const cudaError_t err = launch(kernel, a.num_segments, arguments, static_cast<cudaStream_t>(a.stream));
  return err == cudaSuccess ? FK_PAGED_KV_OK : fail_cuda("paged_kv_append launch", err);
}

}  // extern "C"
