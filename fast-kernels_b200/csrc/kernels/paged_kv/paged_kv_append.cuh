// New keys and values into their pages, the keys turned on the way.
//
// One block per segment (consecutive tokens of one page), one warp per kv head of it: the keys of a
// (segment, head) are a few KB that the warp holds in registers as they came, so the one pass over
// them that finds the page's scale and the one that quantises read memory once. The cosines and sines
// of the segment's tokens are computed once per block and shared by its heads. Lane l of a step takes
// 16 bytes (8 dimensions, four rotary pairs): loads are whole rows, stores whole rows of the page, and
// the eight lanes of a 64-dim block reduce its maximum by shuffles.
//
// What bounds it: memory. All loads of a warp are issued before the first use.
#pragma once

#include "paged_kv_common.cuh"

namespace fk_paged_kv {

constexpr int kAppendWarps = 8;

struct AppendParams {
  const uint16_t* keys;
  const uint16_t* values;
  long long key_token_stride, key_head_stride, value_token_stride, value_head_stride;
  uint8_t* key_pages;
  uint8_t* value_pages;
  float* key_scales;
  float* value_scales;
  const int4* segments;
  int num_tokens;
  int num_pages;
  int num_kv_heads;
  RopeTable rope;
};

template <int KV>
struct Quantiser;
template <>
struct Quantiser<kKvInt8> {
  static constexpr float kLimit = 127.0f;
  static __device__ __forceinline__ uint32_t one(float x) {  // x within [-127.0001, 127.0001]
    return static_cast<uint32_t>(__float2int_rn(fminf(fmaxf(x, -127.0f), 127.0f))) & 0xffu;
  }
  static __device__ __forceinline__ uint32_t four(float a, float b, float c, float d) {
    return one(a) | (one(b) << 8) | (one(c) << 16) | (one(d) << 24);
  }
  static __device__ __forceinline__ void back(uint32_t w, float (&x)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = static_cast<float>(static_cast<int8_t>((w >> (8 * i)) & 0xffu));
    }
  }
};
template <>
struct Quantiser<kKvFp8> {
  static constexpr float kLimit = 448.0f;
  static __device__ __forceinline__ uint32_t four(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | (hi << 16);
  }
  static __device__ __forceinline__ void back(uint32_t w, float (&x)[4]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const __half2_raw h =
          __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>((w >> (16 * i)) & 0xffffu), __NV_E4M3);
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
};

__device__ __forceinline__ void unpack8(const uint4& w, float (&x)[8]) {
  const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = bf16_low(words[i]);
    x[2 * i + 1] = bf16_high(words[i]);
  }
}
// Four rotary pairs; `cs_sn` points at the first pair's (cos, sin).
__device__ __forceinline__ void rotate8(float (&x)[8], const float2* cs_sn) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float even = x[2 * i], odd = x[2 * i + 1];
    x[2 * i] = even * cs_sn[i].x - odd * cs_sn[i].y;
    x[2 * i + 1] = even * cs_sn[i].y + odd * cs_sn[i].x;
  }
}
__device__ __forceinline__ float largest8(const float (&x)[8]) {
  float m = fabsf(x[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    m = fmaxf(m, fabsf(x[i]));
  }
  return m;
}
// x / s, rounded as a division rounds it, from r = 1 / s rounded: one Newton step on the quotient (Markstein,
// "Computation of elementary functions on the IBM RISC System/6000 processor", 1990). Sixteen divisions
// a step were most of the kernel's instructions.
__device__ __forceinline__ float quotient(float x, float s, float r) {
  const float q = x * r;
  return fmaf(fmaf(-q, s, x), r, q);
}
// Maximum over the eight lanes that hold one token's 64-dim block.
__device__ __forceinline__ float largest_of_block(float m) {
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) {
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  }
  return m;
}

template <int D, int PS, int KV, bool ROT>
__global__ void __launch_bounds__(kAppendWarps * 32) paged_kv_append_kernel(const __grid_constant__ AppendParams p) {
  constexpr bool QUANT = KV != kKvBf16;
  constexpr int kLanesPerRow = D / 8;
  constexpr int kRowsPerStep = 32 / kLanesPerRow;
  constexpr int kSteps = PS / kRowsPerStep;
  constexpr int kBlocks = D / kScaleBlock;
  __shared__ float2 table[ROT ? PS * (D / 2) : 1];  // [token][pair]: cos, sin
  __shared__ uint64_t turns[ROT ? D / 2 : 1];

  fk_w4a16::pdl_launch_dependents();
  if constexpr (ROT) {
    if (threadIdx.x < 32) {
      share_rope_table(p.rope, turns, D / 2, threadIdx.x);
    }
    __syncthreads();
  }
  fk_w4a16::pdl_wait_for_prerequisites();
  const int4 segment = p.segments[blockIdx.x];
  const int page = segment.x;
  const int slot = segment.y & 0xffff;
  const int count = segment.y >> 16;
  const int token = segment.z;
  if (page < 0 || page >= p.num_pages || count <= 0 || slot + count > PS || token < 0 ||
      token > p.num_tokens - count) {
    return;
  }
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int row = lane / kLanesPerRow;              // token of a step
  const int dim = (lane % kLanesPerRow) * 8;
  const int block = dim / kScaleBlock;

  for (int head0 = 0; head0 < p.num_kv_heads; head0 += kAppendWarps) {
    const int head = head0 + warp;
    const bool active = head < p.num_kv_heads;
    uint4 k[kSteps], v[kSteps];
    float held = 0.0f;  // the page's scale of this lane's block
    const size_t page_head = static_cast<size_t>(page) * p.num_kv_heads + head;
    if (active) {
      const uint16_t* key_row = p.keys + static_cast<long long>(token + row) * p.key_token_stride +
                                static_cast<long long>(head) * p.key_head_stride + dim;
      const uint16_t* value_row = p.values + static_cast<long long>(token + row) * p.value_token_stride +
                                  static_cast<long long>(head) * p.value_head_stride + dim;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        k[s] = v[s] = make_uint4(0u, 0u, 0u, 0u);
        if (s * kRowsPerStep + row < count) {
          k[s] = __ldg(reinterpret_cast<const uint4*>(key_row + s * kRowsPerStep * p.key_token_stride));
          v[s] = __ldg(reinterpret_cast<const uint4*>(value_row + s * kRowsPerStep * p.value_token_stride));
        }
      }
      if (QUANT && slot > 0) {
        held = p.key_scales[page_head * kBlocks + block];
      }
    }
    if (ROT && head0 == 0) {
      for (int i = threadIdx.x; i < count * (D / 2); i += kAppendWarps * 32) {
        table[i] = rope_cos_sin(turns[i % (D / 2)], segment.w + i / (D / 2));
      }
      __syncthreads();
    }
    if (!active) {
      continue;
    }
    const size_t first = (page_head * PS + slot + row) * D + dim;  // element of step 0
    if constexpr (!QUANT) {
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const int t = s * kRowsPerStep + row;
        if (t < count) {
          uint4 out = k[s];
          if constexpr (ROT) {
            float x[8];
            unpack8(k[s], x);
            rotate8(x, &table[t * (D / 2) + dim / 2]);
            out = make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
          }
          const size_t at = (first + static_cast<size_t>(s) * kRowsPerStep * D) * 2;
          *reinterpret_cast<uint4*>(p.key_pages + at) = out;
          *reinterpret_cast<uint4*>(p.value_pages + at) = v[s];
        }
      }
    } else {
      using Q = Quantiser<KV>;
      // keys: the largest magnitude of the segment's block, then the page's scale
      float largest = 0.0f;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const int t = s * kRowsPerStep + row;
        if (t < count) {
          float x[8];
          unpack8(k[s], x);
          if constexpr (ROT) {
            rotate8(x, &table[t * (D / 2) + dim / 2]);
          }
          largest = fmaxf(largest, largest8(x));
        }
      }
      largest = largest_of_block(largest);
#pragma unroll
      for (int o = kLanesPerRow; o < 32; o <<= 1) {  // the other tokens' lanes
        largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o));
      }
      const float scale = fmaxf(held, fmaxf(largest / Q::kLimit, 1e-6f));
      const float key_inverse = __frcp_rn(scale);
      if (scale > held) {  // (the same on all lanes of the block)
        // what the page holds already, brought to the larger scale
        for (int t = row; t < slot; t += kRowsPerStep) {
          uint2* at = reinterpret_cast<uint2*>(p.key_pages + (page_head * PS + t) * D + dim);
          const uint2 old = *at;
          float a[4], b[4];
          Q::back(old.x, a);
          Q::back(old.y, b);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            a[i] = a[i] * held / scale;
            b[i] = b[i] * held / scale;
          }
          *at = make_uint2(Q::four(a[0], a[1], a[2], a[3]), Q::four(b[0], b[1], b[2], b[3]));
        }
        if (row == 0 && dim % kScaleBlock == 0) {
          p.key_scales[page_head * kBlocks + block] = scale;
        }
      }
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const int t = s * kRowsPerStep + row;
        float x[8], y[8];
        unpack8(v[s], y);  // (zeros past the segment: every lane takes part in the shuffles)
        const float value_scale = fmaxf(largest_of_block(largest8(y)) / Q::kLimit, 1e-6f);
        const float value_inverse = __frcp_rn(value_scale);
        if (t < count) {
          unpack8(k[s], x);
          if constexpr (ROT) {
            rotate8(x, &table[t * (D / 2) + dim / 2]);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            x[i] = quotient(x[i], scale, key_inverse);
            y[i] = quotient(y[i], value_scale, value_inverse);
          }
          const size_t at = first + static_cast<size_t>(s) * kRowsPerStep * D;
          *reinterpret_cast<uint2*>(p.key_pages + at) =
              make_uint2(Q::four(x[0], x[1], x[2], x[3]), Q::four(x[4], x[5], x[6], x[7]));
          *reinterpret_cast<uint2*>(p.value_pages + at) =
              make_uint2(Q::four(y[0], y[1], y[2], y[3]), Q::four(y[4], y[5], y[6], y[7]));
          if (dim % kScaleBlock == 0) {
            p.value_scales[(page_head * PS + slot + t) * kBlocks + block] = value_scale;
          }
        }
      }
    }
  }
}

}  // namespace fk_paged_kv
