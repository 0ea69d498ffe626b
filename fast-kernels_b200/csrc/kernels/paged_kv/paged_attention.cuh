// Attention of query vectors over lists of pages: what the kernels are given, and the kernel that adds
// partial results.
#pragma once

#include "paged_kv_common.cuh"

namespace fk_paged_kv {

struct AttentionParams {
  const uint16_t* query;
  long long query_row_stride, query_head_stride;
  const uint8_t* key_pages;
  const uint8_t* value_pages;
  const float* key_scales;
  const float* value_scales;
  const int* page_ids;
  const int4* vectors;
  const int4* items;  // two per item
  uint16_t* output;
  float* partials;
  int* status;
  int num_rows;
  int num_page_ids;
  int num_vectors;
  int num_partials;
  int num_pages;
  int num_q_heads;
  int num_kv_heads;
  int group;
  int page_size;
  float scale_log2e;
  RopeTable rope;
};

struct Item {
  int first_vector, vectors, kv_head, entry, first_token, end_token, causal, partial;
};
__device__ __forceinline__ Item load_item(const AttentionParams& p, int index) {
  const int4 a = p.items[2 * index], b = p.items[2 * index + 1];
  return Item{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
}
// What the caller's tables may not make the kernels do: leave the arrays, or count past 31 bits (the kernel counts
// whole tiles of up to 128 tokens).
__device__ __forceinline__ bool item_fits(const AttentionParams& p, const Item& item) {
  return item.first_vector >= 0 && item.vectors > 0 && item.vectors <= FK_PAGED_KV_ITEM_ROWS / p.group &&
         item.first_vector <= p.num_vectors - item.vectors && item.kv_head >= 0 && item.kv_head < p.num_kv_heads &&
         item.entry >= 0 && item.first_token >= 0 && item.first_token % p.page_size == 0 && item.partial >= -1 &&
         item.end_token >= item.first_token && item.end_token <= FK_PAGED_KV_MAX_TOKENS &&
         static_cast<long long>(item.entry) + (static_cast<long long>(item.end_token) + p.page_size - 1) / p.page_size <=
             p.num_page_ids;
}

// Partial results of a vector, in order, into its row: one warp per (vector, query head).
template <int D>
__global__ void __launch_bounds__(256) combine_partials_kernel(const __grid_constant__ AttentionParams p) {
  constexpr int kPer = D / 32;
  const long long index = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  fk_w4a16::pdl_launch_dependents();
  fk_w4a16::pdl_wait_for_prerequisites();
  if (index >= static_cast<long long>(p.num_vectors) * p.num_q_heads) {
    return;
  }
  const int4 vector = p.vectors[index / p.num_q_heads];
  const int head = static_cast<int>(index % p.num_q_heads);
  if (vector.w <= 0 || vector.z < 0 || vector.z > p.num_partials - vector.w || vector.x < 0 || vector.x >= p.num_rows) {
    return;
  }
  const int lane = threadIdx.x & 31;
  const float* src = p.partials + (static_cast<size_t>(vector.z) * p.num_q_heads + head) * (D + 4);
  const size_t step = static_cast<size_t>(p.num_q_heads) * (D + 4);
  float m = -INFINITY;
  for (int s = 0; s < vector.w; ++s) {
    m = fmaxf(m, __ldcg(src + s * step + D));
  }
  const float ref = m == -INFINITY ? 0.0f : m;
  float l = 0.0f, o[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    o[e] = 0.0f;
  }
#pragma unroll 4
  for (int s = 0; s < vector.w; ++s) {
    const float2 ml = __ldcg(reinterpret_cast<const float2*>(src + s * step + D));
    const float weight = exp2f(ml.x - ref);
    l += weight * ml.y;
    float v[kPer];
    if constexpr (kPer == 4) {
      const float4 x = __ldcg(reinterpret_cast<const float4*>(src + s * step + lane * 4));
      v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
    } else {
      const float2 x = __ldcg(reinterpret_cast<const float2*>(src + s * step + lane * 2));
      v[0] = x.x, v[1] = x.y;
    }
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      o[e] = fmaf(weight, v[e], o[e]);
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  uint16_t* out = p.output + (static_cast<size_t>(vector.x) * p.num_q_heads + head) * D + lane * kPer;
#pragma unroll
  for (int e = 0; e < kPer; e += 2) {
    *reinterpret_cast<uint32_t*>(out + e) = pack_bf16(o[e] * inv, o[e + 1] * inv);
  }
}

// The tensor-core kernel (paged_attention_tc.cuh), one translation unit per (head_dim, page format).
#define FK_PAGED_ATTENTION_DECLARE(NAME) \
  cudaError_t launch_attention_##NAME(const AttentionParams& params, int num_items, cudaStream_t stream);
FK_PAGED_ATTENTION_DECLARE(d64_bf16)
FK_PAGED_ATTENTION_DECLARE(d64_fp8)
FK_PAGED_ATTENTION_DECLARE(d64_int8)
FK_PAGED_ATTENTION_DECLARE(d128_bf16)
FK_PAGED_ATTENTION_DECLARE(d128_fp8)
FK_PAGED_ATTENTION_DECLARE(d128_int8)
#undef FK_PAGED_ATTENTION_DECLARE

}  // namespace fk_paged_kv
