// Rotary angles in 64-bit fixed point: the keys of paged_kv_append, and the queries that meet them.
#pragma once

#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

namespace fk_rope {

constexpr int kMaxPairs = 64;

// Turns per position of every rotary pair, theta^(-2i/d) / (2 pi), in units of 2^-64: a position times
// this, modulo 2^64, is the angle with the whole turns taken off, off by at most 2^-34 turns at any
// 31-bit position (an fp32 product is off by up to 2^-8 radians at position 131072).
struct RopeTable {
  uint64_t turns[kMaxPairs];
};

// The table from the kernel's parameters to shared memory, by one warp: a parameter indexed by the lane is
// read one lane at a time (3000 clocks for the four pairs of 256 threads).
__device__ __forceinline__ void share_rope_table(const RopeTable& table, uint64_t* shared, int pairs, int lane) {
#pragma unroll 8
  for (int i = 0; i < pairs; ++i) {
    const uint64_t turns = table.turns[i];
    if (lane == (i & 31)) {
      shared[i] = turns;
    }
  }
}
// The nearest quarter turn comes off in integers, so that what is left, at most an eighth of a turn, loses no more than
// 2^-28 of a turn to fp32: an error of 2.3e-8 at most. (Rounding the whole angle loses up to 9.4e-8, rms twice that of an
// fp32 cosine; a correction behind the cosine is lost in its rounding.)
__device__ __forceinline__ float2 rope_cos_sin(uint64_t turns_per_position, int position) {
  const uint32_t turns = static_cast<uint32_t>((turns_per_position * static_cast<uint32_t>(position)) >> 32);
  const uint32_t quarters = (turns + 0x20000000u) >> 30;
  const float half_turns = static_cast<float>(static_cast<int32_t>(turns - (quarters << 30))) * 0x1p-31f;  // in [-1/4, 1/4]
  float sn, cs;
  sincospif(half_turns, &sn, &cs);
  const uint32_t c = __float_as_uint((quarters & 1u) != 0 ? sn : cs);
  const uint32_t s = __float_as_uint((quarters & 1u) != 0 ? cs : sn);
  return make_float2(__uint_as_float(c ^ (((quarters + 1u) & 2u) << 30)), __uint_as_float(s ^ ((quarters & 2u) << 30)));
}

// The same, off by up to 2^-20.5: for a query that is rounded to 16 bits behind it.
__device__ __forceinline__ float2 rope_cos_sin_quick(uint64_t turns_per_position, int position) {
  const uint64_t turns = turns_per_position * static_cast<uint32_t>(position);
  const float angle = static_cast<float>(static_cast<int32_t>(turns >> 32)) * (0x1p-32f * 6.2831853071795865f);
  return make_float2(__cosf(angle), __sinf(angle));
}

// Host.
inline void fill_rope_table(RopeTable* table, int head_dim, float theta) {
  // 64 powers take longer than the rest of a call; a thread's calls have the same ones nearly always
  thread_local RopeTable kept;
  thread_local int kept_dim = 0;
  thread_local float kept_theta = 0.0f;
  if (kept_dim != head_dim || kept_theta != theta) {
    for (int i = 0; i < head_dim / 2; ++i) {
      // long double: 64 bits of mantissa, so that far positions lose nothing (a theta below 1 turns pairs by
      // more than a turn per position; the whole turns do not matter)
      const long double turns =
          std::pow(static_cast<long double>(theta), -2.0L * i / head_dim) / 6.283185307179586476925286766559L;
      const long double fraction = turns - std::floor(turns);
      const long double scaled = std::round(fraction * 18446744073709551616.0L);
      kept.turns[i] = scaled >= 18446744073709551616.0L ? 0 : static_cast<uint64_t>(scaled);
    }
    kept_dim = head_dim;
    kept_theta = theta;
  }
  *table = kept;
}

}  // namespace fk_rope
