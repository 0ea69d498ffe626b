// What the paged-KV operators share: page formats, checks of arguments.
#pragma once

#include <cuda_fp8.h>

#include <cstdint>
#include <string>

#include "../decode_quant_linear/w4a16_common.cuh"
#include "fk_paged_kv.h"
#include "rope_turns.cuh"

namespace fk_paged_kv {

using fk_rope::fill_rope_table;
using fk_rope::rope_cos_sin;
using fk_rope::rope_cos_sin_quick;
using fk_rope::RopeTable;
using fk_rope::share_rope_table;

constexpr int kKvBf16 = FK_PAGED_KV_BF16;
constexpr int kKvFp8 = FK_PAGED_KV_FP8_E4M3;
constexpr int kKvInt8 = FK_PAGED_KV_INT8;
constexpr int kScaleBlock = 64;  // dimensions that share a scale

__device__ __forceinline__ float bf16_low(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_high(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Host: the thread's last error message, and the codes that go with it.
int fail(int code, const std::string& message);
int fail_cuda(const char* what, cudaError_t err);

}  // namespace fk_paged_kv
