// Attention of query vectors over lists of pages: the item's descriptors, a plain kernel for it, and the
// kernel that adds partial results.
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
// What the caller's tables may not make the kernels do: leave the arrays.
__device__ __forceinline__ bool item_fits(const AttentionParams& p, const Item& item) {
  return item.first_vector >= 0 && item.vectors > 0 && item.vectors <= FK_PAGED_KV_ITEM_ROWS / p.group &&
         item.first_vector <= p.num_vectors - item.vectors && item.kv_head >= 0 && item.kv_head < p.num_kv_heads &&
         item.entry >= 0 && item.first_token >= 0 && item.first_token % p.page_size == 0 && item.partial >= -1 &&
         item.end_token >= item.first_token &&
         static_cast<long long>(item.entry) + (static_cast<long long>(item.end_token) + p.page_size - 1) / p.page_size <=
             p.num_page_ids;
}

template <int KV>
__device__ __forceinline__ float element(const uint8_t* pages, size_t at) {
  if constexpr (KV == kKvBf16) {
    return __uint_as_float(static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(pages)[at]) << 16);
  } else if constexpr (KV == kKvInt8) {
    return static_cast<float>(static_cast<int8_t>(pages[at]));
  } else {
    const __half_raw h = __nv_cvt_fp8_to_halfraw(pages[at], __NV_E4M3);
    return __half2float(*reinterpret_cast<const __half*>(&h));
  }
}

// One warp per row, one token at a time; lane l holds dimensions 2l, 2l + 1 (and 64 more).
template <int D, int KV>
__global__ void __launch_bounds__(256) paged_attention_rows_kernel(const __grid_constant__ AttentionParams p) {
  constexpr int kPairs = D / 64;
  const Item item = load_item(p, blockIdx.x);
  if (!item_fits(p, item)) {
    return;
  }
  const int lane = threadIdx.x & 31;
  for (int r = threadIdx.x >> 5; r < item.vectors * p.group; r += 8) {
    const int4 vector = p.vectors[item.first_vector + r / p.group];
    const int head = item.kv_head * p.group + r % p.group;
    if (vector.x < 0 || vector.x >= p.num_rows) {
      continue;
    }
    float q[2 * kPairs], o[2 * kPairs];
    for (int i = 0; i < kPairs; ++i) {
      const int pair = lane + 32 * i;
      const float2 cs = rope_cos_sin(p.rope.turns[pair], vector.y);
      const uint32_t w = *reinterpret_cast<const uint32_t*>(p.query + vector.x * p.query_row_stride +
                                                            head * p.query_head_stride + 2 * pair);
      q[2 * i] = (bf16_low(w) * cs.x - bf16_high(w) * cs.y) * p.scale_log2e;
      q[2 * i + 1] = (bf16_low(w) * cs.y + bf16_high(w) * cs.x) * p.scale_log2e;
      o[2 * i] = o[2 * i + 1] = 0.0f;
    }
    float m = -INFINITY, l = 0.0f;
    const int end = item.causal ? min(item.end_token, vector.y + 1) : item.end_token;
    for (int t = item.first_token; t < end; ++t) {
      const int page = p.page_ids[item.entry + t / p.page_size];
      if (page < 0 || page >= p.num_pages) {
        continue;
      }
      const size_t page_head = static_cast<size_t>(page) * p.num_kv_heads + item.kv_head;
      const size_t row = page_head * p.page_size + t % p.page_size;
      float s = 0.0f;
      for (int i = 0; i < kPairs; ++i) {
        const float scale = KV == kKvBf16 ? 1.0f : p.key_scales[page_head * kPairs + i];
        for (int e = 0; e < 2; ++e) {
          s += q[2 * i + e] * (element<KV>(p.key_pages, row * D + 64 * i + 2 * lane + e) * scale);
        }
      }
      s = fk_w4a16::warp_sum(s);
      const float m_new = fmaxf(m, s);
      const float alpha = exp2f(m - m_new), prob = exp2f(s - m_new);
      l = l * alpha + prob;
      m = m_new;
      for (int i = 0; i < kPairs; ++i) {
        const float scale = KV == kKvBf16 ? 1.0f : p.value_scales[row * kPairs + i];
        for (int e = 0; e < 2; ++e) {
          o[2 * i + e] = o[2 * i + e] * alpha + prob * (element<KV>(p.value_pages, row * D + 64 * i + 2 * lane + e) * scale);
        }
      }
    }
    if (item.partial < 0) {
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      uint16_t* out = p.output + (static_cast<size_t>(vector.x) * p.num_q_heads + head) * D;
      for (int i = 0; i < kPairs; ++i) {
        *reinterpret_cast<uint32_t*>(out + 64 * i + 2 * lane) = pack_bf16(o[2 * i] * inv, o[2 * i + 1] * inv);
      }
    } else if (item.partial < vector.w && vector.z >= 0 && vector.z + item.partial < p.num_partials) {
      float* out = p.partials + (static_cast<size_t>(vector.z + item.partial) * p.num_q_heads + head) * (D + 4);
      for (int i = 0; i < kPairs; ++i) {
        *reinterpret_cast<float2*>(out + 64 * i + 2 * lane) = make_float2(o[2 * i], o[2 * i + 1]);
      }
      if (lane == 0) {
        *reinterpret_cast<float2*>(out + D) = make_float2(m, l);
      }
    }
  }
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

}  // namespace fk_paged_kv
