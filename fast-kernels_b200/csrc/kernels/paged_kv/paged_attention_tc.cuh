// Attention of up to 256 query rows of one kv head over a list of pages, on the fifth-generation
// tensor cores: both products as tcgen05.mma with the logits, the probabilities and the weighted
// values in tensor memory.
//
// One block per item. Its rows (vectors x query heads of the kv head) are two tiles, X = 0 and 1, of
// 128 rows; tokens come in tiles of 128. Per token tile j:
//     S_X = Q_X K_j^T          128 x 128, fp32, tensor memory     (A, B from shared memory)
//     P_X = 2^(S_X - m_X)      bf16, over S_X's own columns       (one thread per row)
//     O_X += P_X V_j           128 x head_dim, fp32               (A from tensor memory, B from shared memory)
// While the softmax warps of one row tile work, the tensor core multiplies for the other. The softmax
// scale times log2(e) rides on the query, so the exponential is one ex2.
//
// The logits are read from tensor memory twice, 32 columns at a time: once for the row's maximum, once
// for the probabilities. A row of 128 kept in registers in between left the compiler too few of them to
// overlap one exponential with the next.
//
// The running maximum is kept lazily: O is multiplied by 2^(old - new) only when a row's maximum has
// grown by more than kGrowth since the last time. The tensor core is done with O whenever a tile's logits
// are: their commit follows the previous tile's second product.
//
// What the roles of a block execute side by side has to stay near the instruction cache: with the 8-bit pages'
// conversion and the first pass for the maximum unrolled, 32768 tokens of fp8 took 449 us instead of 427, of
// which a tenth of all issue slots' waits were for instructions. The exponentials are unrolled all the same
// (rolled: no gain with 8-bit pages, 594 us instead of 577 with bf16).
//
// The exponentials are what the softmax warps are bound by (16 a clock and SM: 2048 clocks per token tile
// and 256 rows, the two products take as long).
//
// Roles (warps): 0-3 and 4-7 softmax of the two row tiles (they also turn and store the queries, and
// write the results), 8 and 11 issue the two tiles' MMAs, 9 the copies, 10 clears the value
// rows behind the end (a probability of 0 times whatever a page holds there would not be 0). 8-bit pages:
// 12-15 convert. Every wait is bounded, and a warp's lanes give up together (wait_all): what they do next
// needs all of them. Barriers that have no limit (bar.sync) are reached on every path.
//
// Operands in shared memory are rows of 128 bytes (64 16-bit elements) under the 128-byte swizzle; a
// tile of 128-dimensional rows is two such halves. bf16 pages are copied there by TMA, one box of
// page_size rows per page and half. 8-bit pages are copied as they are and converted by four warps to
// fp16, exactly for the 64-dim block with the page's (keys) or token's (values) larger scale, the other
// block times the ratio of the two scales. Where there are two blocks both are multiplied by 2^7 (e4m3's 448
// becomes 57344), which leaves the smaller one all 11 bits down to a ratio of 2^-21, and those of a bf16 result down
// to 2^-24; it comes off in fp32, with the page's factor and behind the last product.
// The larger scales stay fp32: the page's goes on the logits,
// the token's on the probability before it is rounded. (Values in bf16 with bf16 probabilities took five
// times the conversion's instructions, and their two roundings made the error 1.5 times the output's own.)
//
// bf16 pages: query and probabilities are bf16 because both operands of a product have one type, and are rounded
// once. Each of the two roundings is as large as the output's own: 2.5e-3 to 2.9e-3 in the 2-norm for 1.65e-3. A
// remainder of the query as a second operand would take half as much tensor work again and 64 KB of shared memory for
// one of them, a remainder of the probabilities as much again and a second conversion in the softmax.
//
// What it measures: 8192 tokens, 32 heads over 8 of 128, bf16, causal: 574 us, 958 TFLOP/s, 59 % of the
// measured bf16 peak: a token tile takes 3350 clocks where the products need 2050. 512 tokens behind 32768
// in fp8 pages, 32 heads over 4: 418 us, 661 TFLOP/s, 5400 clocks a tile: bound by the conversion, in the
// issue slots of the softmax warps, and the chain behind it. (Waits with one verdict a warp, and so without
// divergence behind them, were worth 10 of 427 us.)
// Tried and slower: steps of 64 tokens with two buffers of logits per row tile (N = 64 costs the tensor
// core as much as N = 128 when both operands come from shared memory: 748 us), four more converting warps
// (fewer registers for the softmax: 602 us for 477), a quarter or half of the exponentials as polynomials
// on the FMA pipe (613 and 640 us for 594), the conversion in batches of two or eight rows a thread (444 and
// 433 us for 427).
#pragma once

#include <cuda.h>

#include <type_traits>

#include "../clustered_page_decode/page_decode_kernel.cuh"
#include "../decode_quant_linear/w4a16_gemm_tile.cuh"
#include "paged_attention.cuh"

namespace fk_paged_kv {

namespace umma = fk_w4a16::umma;
namespace tile = fk_w4a16::tile;
using fk_w4a16::lds64;
using fk_w4a16::mbar_expect_tx;
using fk_w4a16::mbar_init;
using fk_w4a16::mbar_init_fence;
using fk_w4a16::mbar_wait_parked;
using fk_w4a16::proxy_fence_async;
using fk_w4a16::smem_addr;

constexpr int kTileRows = 128;
constexpr int kTileTokens = 128;
constexpr int kFactorRing = 4;  // token tiles whose scales are kept for the softmax warps
constexpr int kStatusWaitTimeout = 1;

template <int D, int KV>
struct TcLayout {
  static constexpr bool kQuant = KV != kKvBf16;
  static constexpr int kHalves = D / 64;
  static constexpr int kHalfBytes = kTileTokens * 128;             // 64 dimensions of 128 rows
  static constexpr int kOperandBytes = kHalves * kHalfBytes;       // a tile of queries, keys or values
  static constexpr int kSlots = D == 64 ? (kQuant ? 4 : 8) : (kQuant ? 3 : 5);
  static constexpr int kRawBytes = kTileTokens * D;                // a tile of 8-bit keys or values
  static constexpr int kRawScaleBytes = kTileTokens * (D / 64) * 4;
  static constexpr int kRawSlots = kQuant ? (D == 64 ? 6 : 3) : 0;
  static constexpr int kRawSlotBytes = kRawBytes + kRawScaleBytes;
  static constexpr int kThreads = kQuant ? 512 : 384;
  // A softmax thread holds a row of 128 logits. Two warpgroups of them and one or two of the others draw
  // on what the block was launched with: 2 x 208 + 88 = 3 x 168, 2 x 184 + 2 x 72 = 4 x 128.
  static constexpr int kSoftmaxRegisters = kQuant ? 184 : 208;
  static constexpr int kOtherRegisters = kQuant ? 72 : 88;
  // offsets from a 1024-byte aligned base
  static constexpr int kQueries = 0;
  static constexpr int kRing = kQueries + 2 * kOperandBytes;
  static constexpr int kRaw = kRing + kSlots * kOperandBytes;
  static constexpr int kKeyFactors = kRaw + kRawSlots * kRawSlotBytes;              // [ring][8 pages]
  static constexpr int kValueFactors = kKeyFactors + (kQuant ? kFactorRing * 32 : 0);  // [ring][128 tokens], then their log2
  static constexpr int kRawKeyScales = kValueFactors + (kQuant ? kFactorRing * 1024 : 0);  // [raw slot][8 pages][2]
  static constexpr int kRatios = kRawKeyScales + kRawSlots * 64;                    // [keys, values][128 tokens][2]
  static constexpr int kTileLogs = kRatios + (kQuant ? 2048 : 0);              // [ring][4 warps]
  static constexpr int kRowPower = kTileLogs + (kQuant ? kFactorRing * 16 : 0);     // [256]
  static constexpr int kTurns = kRowPower + (kQuant ? 1024 : 0);                    // [64]
  static constexpr int kBarriers = kTurns + 512;
  static constexpr int kBytes = kBarriers + 512 + 1024;            // and the alignment's slack
  // results are staged over the operands
  static_assert(2 * kTileRows * (D + 4) * 4 <= kRing + kSlots * kOperandBytes, "rows of results fit the operands' memory");
};

// Bounded wait. The plain test comes first: most waits of the issuer and the copies are over when they
// begin, and a test costs a few dozen clocks where try_wait takes some 150 even then.
__device__ __forceinline__ bool wait_for(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      "selp.u32 %0, 1, 0, p;\n"
      "}\n"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0 || mbar_wait_parked(bar, parity);
}
// The same by a whole warp: one verdict for all lanes. Each lane's limit runs out by its own clock, and lanes
// that went different ways would meet shuffles, tensor memory loads and barriers with members missing.
__device__ __forceinline__ bool wait_all(uint32_t bar, uint32_t parity) {
  return __all_sync(0xffffffffu, wait_for(bar, parity));
}

__device__ __forceinline__ void mma_f16_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
      "}\n" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
// Shared memory -> global, both 16-byte aligned, `bytes` a multiple of 16.
__device__ __forceinline__ void bulk_store(void* dst, uint32_t src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(src), "r"(bytes) : "memory");
}
// This thread's bulk stores are complete.
__device__ __forceinline__ void bulk_store_wait() {
  asm volatile("cp.async.bulk.commit_group;\ncp.async.bulk.wait_group 0;" ::: "memory");
}
// Operand descriptors: 128-byte swizzle (bits 61-63 = 2), version 1 (bit 46), offsets in 16-byte units.
// Rows are the M or N dimension (K contiguous): groups of 8 rows are 1024 bytes apart.
__device__ __forceinline__ uint64_t rows_desc(uint32_t address) {
  return static_cast<uint64_t>((address & 0x3FFFFu) >> 4) | (uint64_t{1} << 16) | (uint64_t{1024 >> 4} << 32) |
         (uint64_t{1} << 46) | (uint64_t{2} << 61);
}
// Rows are the K dimension (N contiguous): blocks of 64 columns are a half apart, groups of 8 rows 1024 bytes.
__device__ __forceinline__ uint64_t columns_desc(uint32_t address) {
  return static_cast<uint64_t>((address & 0x3FFFFu) >> 4) | (uint64_t{(kTileTokens * 128) >> 4} << 16) |
         (uint64_t{1024 >> 4} << 32) | (uint64_t{1} << 46) | (uint64_t{2} << 61);
}
// fp32 accumulate, M = 128; `columns_b`: B's N dimension is contiguous.
__host__ __device__ constexpr uint32_t instruction_desc(bool bf16, int n, bool columns_b) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((columns_b ? 1u : 0u) << 16) |
         (static_cast<uint32_t>(n / 8) << 17) | (static_cast<uint32_t>(kTileRows / 16) << 24);
}
// Element (row, 16-byte chunk of the row) of a swizzled operand.
__device__ __forceinline__ uint32_t operand_chunk(int row, int chunk) {
  return (chunk >> 3) * (kTileRows * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4);
}
__device__ __forceinline__ void sts128(uint32_t addr, uint4 v) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ void st32_tmem(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

using fk_page_decode::f32x2;
using fk_page_decode::fma2;
using fk_page_decode::mul2;
using fk_page_decode::pack2;
using fk_page_decode::unpack2;
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ f32x2 pair_of(const uint32_t* r) { return pack2(__uint_as_float(r[0]), __uint_as_float(r[1])); }
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// Largest of N values, as two chains.
template <int N>
__device__ __forceinline__ float largest_of(const uint32_t* r) {
  float a = __uint_as_float(r[0]), b = __uint_as_float(r[1]);
#pragma unroll
  for (int i = 2; i + 3 < N; i += 4) {
    a = max3(a, __uint_as_float(r[i]), __uint_as_float(r[i + 1]));
    b = max3(b, __uint_as_float(r[i + 2]), __uint_as_float(r[i + 3]));
  }
  return max3(a, b, max3(a, __uint_as_float(r[N - 2]), __uint_as_float(r[N - 1])));
}

// Two copies of mine / larger in fp16, times 2^7 (exactly that for the block that has the larger scale).
constexpr float kRatioPower = 128.0f;
constexpr float kRatioLog2 = 7.0f;
__device__ __forceinline__ uint32_t scale_ratio(float mine, float larger) {
  const __half2 ratio = __float2half2_rn(larger > 0.0f ? __fdividef(mine, larger) * kRatioPower : 0.0f);
  return *reinterpret_cast<const uint32_t*>(&ratio);
}
__device__ __forceinline__ uint32_t mul_half2(uint32_t a, uint32_t b) {
  const __half2 product = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&product);
}

template <int D, int KV>
__global__ void __launch_bounds__(TcLayout<D, KV>::kThreads, 1)
    paged_attention_tc_kernel(const __grid_constant__ AttentionParams p, const __grid_constant__ CUtensorMap key_map,
                              const __grid_constant__ CUtensorMap value_map) {
  using L = TcLayout<D, KV>;
  constexpr bool QUANT = L::kQuant;
  constexpr int kBlocks = D / 64;          // scale blocks, and halves of an operand
  constexpr int kChunks = D / 8;           // 16-byte chunks of a row
  // How far a row's largest probability (weight) may be above 1, as a power of two, before O is rescaled:
  // 8-bit pages, fp16 weights: below 2^16; bf16 has the range, and O should not lose it.
  constexpr float kGrowth = QUANT ? 15.0f : 8.0f;
  constexpr float kHeadroom = 7.0f;
  constexpr uint32_t kScoresDesc = instruction_desc(!QUANT, kTileTokens, false);
  constexpr uint32_t kValuesDesc = instruction_desc(!QUANT, D, true);
  extern __shared__ __align__(16) uint8_t raw_smem[];

  const int tid = static_cast<int>(threadIdx.x);
  const int lane = tid & 31;
  const int warp = tid >> 5;
  const uint32_t base = (smem_addr(raw_smem) + 1023u) & ~1023u;
  uint8_t* smem = raw_smem + (base - smem_addr(raw_smem));
  const uint32_t bars = base + L::kBarriers;
  const uint32_t q_ready = bars + 16;
  const uint32_t s_ready = bars + 24;             // [2] logits of a tile are there
  // [half][2] probabilities of a half tile are stored (and O is rescaled). A barrier each: with one for
  // both, a late issuer would find its phase overtaken by the next.
  const uint32_t p_ready = bars + 352;
  const uint32_t o_final = bars + 56;             // [2] the last product is done
  const uint32_t turn = bars + 384;               // [2] the tile's issuer may issue
  const uint32_t v_clear = bars + 72;
  const uint32_t drain = bars + 80;
  const uint32_t v_landed = bars + 88;
  const uint32_t full = bars + 96;                // [slots] operand tile is there
  const uint32_t empty = full + 8 * 8;            // [slots] MMAs are done with it
  const uint32_t raw_full = empty + 8 * 8;        // [raw slots]
  const uint32_t raw_empty = raw_full + 8 * 8;
  volatile uint32_t* fail_flag = reinterpret_cast<volatile uint32_t*>(smem + L::kBarriers + 8);
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(smem + L::kBarriers);
  volatile int* issued_slot = reinterpret_cast<volatile int*>(smem + L::kBarriers + 12);  // operand copies begun

  if (tid == 0) {
    *fail_flag = 0u;
    *issued_slot = 0;
    mbar_init(q_ready, 8);
    for (int x = 0; x < 2; ++x) {
      mbar_init(s_ready + 8 * x, 1);
      mbar_init(p_ready + 8 * x, 4);
      mbar_init(p_ready + 16 + 8 * x, 4);
      mbar_init(o_final + 8 * x, 1);
      mbar_init(turn + 8 * x, 1);
    }
    mbar_init(v_landed, 1);
    mbar_init(v_clear, 1);
    mbar_init(drain, 2);
    for (int s = 0; s < L::kSlots; ++s) {
      mbar_init(full + 8 * s, QUANT ? 4 : 1);
      mbar_init(empty + 8 * s, 2);
    }
    for (int s = 0; s < L::kRawSlots; ++s) {
      mbar_init(raw_full + 8 * s, 1);
      mbar_init(raw_empty + 8 * s, 4);
    }
    mbar_init_fence();
  }
  uint64_t* turns = reinterpret_cast<uint64_t*>(smem + L::kTurns);
  if (warp == 8) {
    umma::tmem_alloc(bars, 512);
    umma::tmem_relinquish();
  }
  if (tid < D / 2) {
    turns[tid] = p.rope.turns[tid];  // (a parameter indexed by the lane is read lane by lane: once is enough)
  }
  umma::fence_before_sync();
  __syncthreads();
  umma::fence_after_sync();
  const uint32_t tmem = *tmem_slot;

  // From here on memory is read; the next kernel of the stream may be scheduled, knowing that what was
  // launched before this one has completed.
  fk_w4a16::pdl_wait_for_prerequisites();
  fk_w4a16::pdl_launch_dependents();

  const Item item = load_item(p, blockIdx.x);
  const bool fits = item_fits(p, item);
  const int rows = item.vectors * p.group;
  // Tokens that the rows of tile x see, and how many tiles of them.
  auto limit_of = [&](int x, bool last) -> int {
    const int row = last ? min(rows, (x + 1) * kTileRows) - 1 : x * kTileRows;
    return item.causal != 0 ? min(item.end_token, p.vectors[item.first_vector + row / p.group].y + 1) : item.end_token;
  };
  int tiles[2] = {0, 0};
  int unmasked[2] = {0, 0};  // tokens that every row of the tile sees
  if (fits) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      if (x * kTileRows < rows) {
        const int seen = max(0, limit_of(x, true) - item.first_token);
        tiles[x] = (seen + kTileTokens - 1) / kTileTokens;
        // positions of an item's vectors need not ascend without `causal`; with it they do
        unmasked[x] = max(0, limit_of(x, false) - item.first_token);
      }
    }
  }
  const int count = max(tiles[0], tiles[1]);
  const int loaded = min(item.end_token - item.first_token, count * kTileTokens);  // tokens that are fetched
  const bool clear_needed = count > 0 && loaded < count * kTileTokens;

  auto give_up = [&]() {
    *fail_flag = 1u;
    atomicExch(p.status, kStatusWaitTimeout);
  };

  if (warp < 8) {
    tile::registers_up<L::kSoftmaxRegisters>();
    const int x = warp >> 2;
    const int row = (warp & 3) * 32 + lane;      // of the tile; also its tensor memory lane
    float* row_power = reinterpret_cast<float*>(smem + L::kRowPower);
    // ---- queries: turned, scaled, rounded, stored ----------------------------------------------
    if (count > 0) {
      // A thread takes 8 dimensions (four rotary pairs) of a vector: their cosines and sines serve all
      // the query heads that it walks. `slices` threads share a vector's heads where there are few vectors.
      const int columns = item.vectors * kChunks;
      const int slices = max(1, min(p.group, 256 / columns));
      const int tasks = columns * slices;
      const int round = (tasks + 31) / 32 * 32;
      const int heads_each = (p.group + slices - 1) / slices;
      constexpr int kBatch = 4;  // heads whose loads are in flight together
      // (with one slice no division by a number that only the item knows; with more, a thread has one task)
      auto vector_of = [&](int task) -> int {
        return task >= tasks ? 0 : slices == 1 ? task / kChunks : (task / kChunks) % item.vectors;
      };
      auto slice_of = [&](int task) -> int { return task >= tasks || slices == 1 ? 0 : task / columns; };
      auto descriptor = [&](int task) -> int4 { return __ldg(p.vectors + item.first_vector + vector_of(task)); };
      // Heads h0 .. h0 + 3 of a task, as they are.
      auto fetch = [&](int task, const int4& v, int h0, uint4 (&w)[kBatch]) {
        const bool readable = task < tasks && v.x >= 0 && v.x < p.num_rows;
        const int head0 = slice_of(task) * heads_each;
        const uint16_t* src = p.query + static_cast<long long>(readable ? v.x : 0) * p.query_row_stride +
                              static_cast<long long>(item.kv_head * p.group + head0) * p.query_head_stride + (task % kChunks) * 8;
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
          w[b] = make_uint4(0u, 0u, 0u, 0u);
          if (readable && h0 + b < heads_each && head0 + h0 + b < p.group) {
            w[b] = __ldg(reinterpret_cast<const uint4*>(src + static_cast<long long>(h0 + b) * p.query_head_stride));
          }
        }
      };
      int4 v = descriptor(tid), next_v = descriptor(tid + 256);
      uint4 w[kBatch], next_w[kBatch];
      fetch(tid, v, 0, w);
      for (int task = tid; task < round; task += 256) {
        const int4 after_v = descriptor(task + 512);
        fetch(task + 256, next_v, 0, next_w);
        const int chunk = task % kChunks;
        const int vector = vector_of(task);
        const int head0 = slice_of(task) * heads_each;
        float2 cs[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 turn = rope_cos_sin_quick(turns[chunk * 4 + i], v.y);
          cs[i] = make_float2(turn.x * p.scale_log2e, turn.y * p.scale_log2e);
        }
        for (int h0 = 0; h0 < heads_each; h0 += kBatch) {
          if (h0 > 0) {
            fetch(task, v, h0, w);
          }
          uint4 out[kBatch];
          int bits[kBatch];
#pragma unroll
          for (int b = 0; b < kBatch; ++b) {
            const uint32_t words[4] = {w[b].x, w[b].y, w[b].z, w[b].w};
            float q[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float even = bf16_low(words[i]), odd = bf16_high(words[i]);
              q[2 * i] = even * cs[i].x - odd * cs[i].y;
              q[2 * i + 1] = even * cs[i].y + odd * cs[i].x;
            }
            bits[b] = 0;
            if constexpr (QUANT) {
              // fp16 has the precision but not the range: the row is divided by the power of two of its
              // largest element, which goes back on in fp32
              float largest = 0.0f;
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                largest = fmaxf(largest, fabsf(q[i]));
              }
#pragma unroll
              for (int o = 1; o < kChunks; o <<= 1) {
                largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o));
              }
              bits[b] = fk_page_decode::exponent_bits(largest);
              const float shrink = fk_page_decode::inverse_power(bits[b]);
              out[b] = make_uint4(pack_half(q[0] * shrink, q[1] * shrink), pack_half(q[2] * shrink, q[3] * shrink),
                                  pack_half(q[4] * shrink, q[5] * shrink), pack_half(q[6] * shrink, q[7] * shrink));
            } else {
              out[b] = make_uint4(pack_bf16(q[0], q[1]), pack_bf16(q[2], q[3]), pack_bf16(q[4], q[5]), pack_bf16(q[6], q[7]));
            }
          }
#pragma unroll
          for (int b = 0; b < kBatch; ++b) {
            const int head = head0 + h0 + b;
            if (task < tasks && h0 + b < heads_each && head < p.group) {
              const int r = vector * p.group + head;
              if (QUANT && chunk == 0) {
                row_power[r] = __int_as_float(bits[b]);
              }
              sts128(base + L::kQueries + (r >> 7) * L::kOperandBytes + operand_chunk(r & 127, chunk), out[b]);
            }
          }
        }
        v = next_v;
        next_v = after_v;
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
          w[b] = next_w[b];
        }
      }
      for (int idx = tid; idx < (256 - rows) * kChunks; idx += 256) {  // rows without a vector
        const int r = rows + idx / kChunks;
        sts128(base + L::kQueries + (r >> 7) * L::kOperandBytes + operand_chunk(r & 127, idx % kChunks),
               make_uint4(0u, 0u, 0u, 0u));
        if (QUANT && idx % kChunks == 0) {
          row_power[r] = 0.0f;
        }
      }
      proxy_fence_async();
      __syncwarp();
      if (lane == 0) {
        umma::mbar_arrive(q_ready);
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");  // row_power is read by other warps than its writers
    }
    // ---- softmax --------------------------------------------------------------------------------
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t s_tmem = tmem + lanes + x * kTileTokens;
    const uint32_t o_tmem = tmem + lanes + 256 + x * D;
    const int r = x * kTileRows + row;
    const int my_vector = r < rows ? r / p.group : 0;
    const int my_head = item.kv_head * p.group + (r < rows ? r % p.group : 0);
    const int4 vec = fits ? p.vectors[item.first_vector + my_vector] : make_int4(0, 0, 0, 0);
    const int limit = (item.causal != 0 ? min(item.end_token, vec.y + 1) : item.end_token) - item.first_token;
    const float power = QUANT && count > 0 ? row_power[r] : 1.0f;
    // `m` is what probabilities are relative to, 2^(logit - m). bf16 pages: the largest logit (kept lazily).
    // 8-bit pages: the largest logit + log2 of the token's value scale, that is the heaviest weight
    // (probability times scale), which is what has to stay within fp16, less kHeadroom: the heaviest weight is 2^kHeadroom
    // to begin with and may grow to 2^kGrowth, so that one of 2^-21 of it still has all its bits.
    float m = -INFINITY, l = 0.0f;
    bool ok = true;
    for (int j = 0; j < tiles[x]; ++j) {
      ok = wait_all(s_ready + 8 * x, j & 1);
      if (!ok) {
        give_up();
        break;
      }
      umma::fence_after_sync();
      const bool masked = (j + 1) * kTileTokens > unmasked[x];
      const int seen = limit - j * kTileTokens;
      // QUANT: what 16 neighbouring logits are multiplied by, the page's key scale and the row's power of two: from
      // shared memory in the loops that are not unrolled, from registers for the exponentials
      const float4* value_factors = reinterpret_cast<const float4*>(smem + L::kValueFactors) + (j % kFactorRing) * 32;
      const float4* value_logs = value_factors + kFactorRing * 32;
      const float* factors = reinterpret_cast<const float*>(smem + L::kKeyFactors) + (j % kFactorRing) * 8;
      auto factor = [&](int g) -> float { return factors[p.page_size == 16 ? g : g >> 1] * power; };
      float kept[8];
      if constexpr (QUANT) {
#pragma unroll
        for (int g = 0; g < 8; ++g) {
          kept[g] = factor(g);
        }
      }
      uint32_t buffer[2][32];
      // Products of 32 tokens; with `masked` the logits, -inf where the row does not see the token.
      auto take = [&](int c, uint32_t(&s)[32], uint32_t(&next)[32], auto all_seen) {
        tile::wait_ld32(s);
        if (c + 1 < 4) {
          tile::ld32(s_tmem + 32 * (c + 1), next);
        }
        if (!decltype(all_seen)::value && masked) {
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float logit = QUANT ? __uint_as_float(s[i]) * factor(2 * c + i / 16) : __uint_as_float(s[i]);
            s[i] = c * 32 + i < seen ? __float_as_uint(logit) : 0xff800000u;
          }
        }
      };
      auto factor_of = [&](int g) -> float { return masked ? 1.0f : factor(g); };
      // ---- the tile's largest logit ----
      float top = -INFINITY;
      tile::ld32(s_tmem, buffer[0]);
#pragma unroll (QUANT ? 1 : 2)
      for (int c0 = 0; c0 < 4; c0 += 2)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int c = c0 + u;
        uint32_t(&s)[32] = buffer[u];
        take(c, s, buffer[u ^ 1], std::false_type{});
        if constexpr (QUANT) {  // (scales are not negative)
          top = max3(top, largest_of<16>(s) * factor_of(2 * c), largest_of<16>(s + 16) * factor_of(2 * c + 1));
        } else {
          top = fmaxf(top, largest_of<32>(s));
        }
      }
      if constexpr (QUANT) {
        const int index = 2 * j + 1;  // the value scales come with the tile's values
        ok = wait_all(full + 8 * (index % L::kSlots), (index / L::kSlots) & 1);
        if (!ok) {
          give_up();
          break;
        }
        const float4 logs = reinterpret_cast<const float4*>(smem + L::kTileLogs)[j % kFactorRing];
        const float bound = top + fmaxf(fmaxf(logs.x, logs.y), fmaxf(logs.z, logs.w));
        if (j == 0 || __any_sync(0xffffffffu, bound > m + kGrowth)) {
          // the heaviest weight itself: the bound may be far above it
          top = -INFINITY;
          tile::ld32(s_tmem, buffer[0]);
#pragma unroll 1
          for (int c0 = 0; c0 < 4; c0 += 2)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int c = c0 + u;
            uint32_t(&s)[32] = buffer[u];
            take(c, s, buffer[u ^ 1], std::false_type{});
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              const f32x2 f = pack2(factor_of(2 * c + i / 16), factor_of(2 * c + i / 16));
              const float4 v = value_logs[c * 8 + i / 4];
              float a, b, e, g;
              unpack2(fma2(pair_of(s + i), f, pack2(v.x, v.y)), a, b);
              unpack2(fma2(pair_of(s + i + 2), f, pack2(v.z, v.w)), e, g);
              top = max3(top, max3(a, b, e), g);
            }
          }
          top -= kHeadroom;
        } else {
          top = m;
        }
      }
      tile::ld32(s_tmem, buffer[0]);
      if (j == 0) {
        m = top;
      } else if (__any_sync(0xffffffffu, top > m + (QUANT ? 0.0f : kGrowth))) {
        const float m_new = fmaxf(m, top);
        const float carry = m == -INFINITY ? 0.0f : fk_page_decode::exp2_quick(m - m_new);
        m = m_new;
        l *= carry;
        uint32_t o[32];
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          tile::ld32(o_tmem + c, o);
          tile::wait_ld32(o);
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            o[i] = __float_as_uint(__uint_as_float(o[i]) * carry);
          }
          st32_tmem(o_tmem + c, o);
        }
      }
      // ---- probabilities, over the logits' own columns: a half of the tile at a time, so that the
      // ---- second product starts while the other half is still worked on
      const float ref = m == -INFINITY ? 0.0f : m;
      const f32x2 minus_ref = pack2(-ref, -ref);
      f32x2 sum[2] = {pack2(0.0f, 0.0f), pack2(0.0f, 0.0f)};
      auto probabilities = [&](auto all_seen) {  // in two instances: the compiler leaves the branch in otherwise
        [[maybe_unused]] constexpr bool kAllSeen = decltype(all_seen)::value;
#pragma unroll (QUANT || kAllSeen ? 2 : 1)
      for (int c0 = 0; c0 < 4; c0 += 2)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int c = c0 + u;
        uint32_t(&s)[32] = buffer[u];
        take(c, s, buffer[u ^ 1], all_seen);
        uint32_t packed[16];
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          f32x2 e;
          if constexpr (QUANT) {
            const float f = kAllSeen ? kept[2 * c + i / 16] : 1.0f;
            e = fma2(pair_of(s + i), pack2(f, f), minus_ref);
          } else {
            e = add2(pair_of(s + i), minus_ref);
          }
          float a, b;
          unpack2(e, a, b);
          s[i] = __float_as_uint(fk_page_decode::exp2_quick(a));
          s[i + 1] = __float_as_uint(fk_page_decode::exp2_quick(b));
        }
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          const f32x2 first = pair_of(s + i), second = pair_of(s + i + 2);
          sum[0] = add2(sum[0], first);
          sum[1] = add2(sum[1], second);
          float a, b;
          if constexpr (QUANT) {
            const float4 v = value_factors[c * 8 + i / 4];
            unpack2(mul2(first, pack2(v.x, v.y)), a, b);
            packed[i / 2] = pack_half(a, b);
            unpack2(mul2(second, pack2(v.z, v.w)), a, b);
            packed[i / 2 + 1] = pack_half(a, b);
          } else {
            unpack2(first, a, b);
            packed[i / 2] = pack_bf16(a, b);
            unpack2(second, a, b);
            packed[i / 2 + 1] = pack_bf16(a, b);
          }
        }
        umma::st16(s_tmem + 16 * c, packed);
        if (u == 1) {
          umma::wait_st();
          umma::fence_before_sync();
          __syncwarp();
          if (lane == 0) {
            umma::mbar_arrive(p_ready + 16 * (c >> 1) + 8 * x);
          }
        }
      }
      };
      if (masked) {
        probabilities(std::false_type{});
      } else {
        probabilities(std::true_type{});
      }
      {
        float a, b;
        unpack2(add2(sum[0], sum[1]), a, b);
        l += a + b;
      }
    }
    // ---- results --------------------------------------------------------------------------------
    // Every thread lays its row out in shared memory (once both row tiles are done with the operands there)
    // and a bulk copy takes it away: stores straight from a thread per row touch 32 lines an instruction,
    // 9000 clocks for 256 rows of partial results.
    if (tiles[x] > 0 && ok && !wait_all(o_final + 8 * x, 0)) {
      give_up();
      ok = false;
    }
    asm volatile("bar.sync 1, 256;" ::: "memory");
    if (ok && x * kTileRows < rows && fits && __all_sync(0xffffffffu, *fail_flag == 0u)) {
      umma::fence_after_sync();
      const bool direct = item.partial < 0;
      const bool write_row = r < rows && vec.x >= 0 && vec.x < p.num_rows &&
                             (direct || (item.partial < vec.w && vec.z >= 0 && vec.z + item.partial < p.num_partials));
      constexpr float kPower = QUANT && kBlocks == 2 ? kRatioPower : 1.0f;  // what the values were multiplied by
      constexpr float kPowerLog2 = QUANT && kBlocks == 2 ? kRatioLog2 : 0.0f;
      const float inv = l == 0.0f ? 0.0f : (1.0f / kPower) / l;
      constexpr uint32_t kRowBytes = (D + 4) * 4;  // 16 bytes off a multiple of 128: lanes take turns at the banks
      const uint32_t staged = base + r * kRowBytes;
#pragma unroll
      for (int c = 0; c < D; c += 32) {
        uint32_t o[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          o[i] = 0u;
        }
        if (tiles[x] > 0) {
          tile::ld32(o_tmem + c, o);
          tile::wait_ld32(o);
        }
        if (direct) {
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            uint4 w;
            w.x = pack_bf16(__uint_as_float(o[i]) * inv, __uint_as_float(o[i + 1]) * inv);
            w.y = pack_bf16(__uint_as_float(o[i + 2]) * inv, __uint_as_float(o[i + 3]) * inv);
            w.z = pack_bf16(__uint_as_float(o[i + 4]) * inv, __uint_as_float(o[i + 5]) * inv);
            w.w = pack_bf16(__uint_as_float(o[i + 6]) * inv, __uint_as_float(o[i + 7]) * inv);
            sts128(staged + (c + i) * 2, w);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            sts128(staged + (c + i) * 4, make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]));
          }
        }
      }
      if (!direct) {
        // (the values keep their power: denominator and maximum are brought to it)
        sts128(staged + D * 4, make_uint4(__float_as_uint(m - kPowerLog2), __float_as_uint(l * kPower), 0u, 0u));
      }
      proxy_fence_async();
      if (write_row) {
        if (direct) {
          bulk_store(p.output + (static_cast<size_t>(vec.x) * p.num_q_heads + my_head) * D, staged, D * 2);
        } else {
          bulk_store(p.partials + (static_cast<size_t>(vec.z + item.partial) * p.num_q_heads + my_head) * (D + 4), staged,
                     kRowBytes);
        }
      }
      bulk_store_wait();
    }
  } else {
    tile::registers_down<L::kOtherRegisters>();
    if ((warp == 8 || warp == 11) && lane == 0 && count > 0) {
      // ---- MMA issuers --------------------------------------------------------------------------
      // One per row tile, taking turns: while one issues O_X += P_X(j) V(j) and, behind it, S_X(j + 1) over
      // P_X(j)'s columns, the other goes through its waits and commits. (A single issuer left the tensor
      // core idle for 700 of 3450 clocks a token tile; without the turns the two row tiles' products run,
      // and end, at the same time, and so do the exponentials that wait for them: 707 us for 628.)
      const int x = warp == 8 ? 0 : 1;
      const int mine = tiles[x];
      auto slot_of = [&](int index) -> uint32_t { return index % L::kSlots; };  // keys 2 j, values 2 j + 1
      auto landed = [&](int index) -> bool { return wait_for(full + 8 * slot_of(index), (index / L::kSlots) & 1); };
      auto release = [&](int index, bool used) {
        if (used) {
          umma::commit(empty + 8 * slot_of(index));
        } else {
          umma::mbar_arrive(empty + 8 * slot_of(index));
        }
      };
      // Row tile 0 begins; a turn's end is an arrival at the other's barrier.
      auto wait_turn = [&](int n) -> bool { return wait_for(turn + 8 * x, (n & 1) ^ (x == 0 ? 1 : 0)); };
      auto end_turn = [&]() { umma::mbar_arrive(turn + 8 * (1 - x)); };
      const uint64_t queries = rows_desc(base + L::kQueries + x * L::kOperandBytes);
      auto scores = [&](int j) {
        const uint64_t b = rows_desc(base + L::kRing + slot_of(2 * j) * L::kOperandBytes);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint64_t step = static_cast<uint64_t>((k / 4) * (L::kHalfBytes >> 4) + (k % 4) * 2);
          mma_f16_ss(tmem + x * kTileTokens, queries + step, b + step, kScoresDesc, k == 0 ? 0u : 1u);
        }
        umma::commit(s_ready + 8 * x);
      };
      bool ok = wait_for(q_ready, 0) && landed(0) && wait_turn(0);
      if (ok) {
        if (mine > 0) {
          umma::fence_after_sync();
          scores(0);
        }
        end_turn();
        release(0, mine > 0);
      }
      for (int j = 0; ok && j < count; ++j) {
        const bool more = j + 1 < count;
        ok = landed(2 * j + 1);
        if (ok && !QUANT && clear_needed && !more) {
          if (x == 0) {
            umma::mbar_arrive(v_landed);
          }
          ok = wait_for(v_clear, 0);
        }
        ok = ok && (!more || landed(2 * j + 2));
        if (ok && j < mine) {
          ok = wait_for(p_ready + 8 * x, j & 1);
        }
        ok = ok && wait_turn(j + 1);
        if (!ok) {
          break;
        }
        if (j < mine) {
          const uint64_t b = columns_desc(base + L::kRing + slot_of(2 * j + 1) * L::kOperandBytes);
          auto values = [&](int half) {
            umma::fence_after_sync();
#pragma unroll
            for (int k = 4 * half; k < 4 * half + 4; ++k) {
              umma::mma_f16_ts(tmem + 256 + x * D, tmem + x * kTileTokens + 8 * k, b + k * (2048 >> 4), kValuesDesc,
                               j == 0 && k == 0 ? 0u : 1u);
            }
          };
          values(0);
          ok = wait_for(p_ready + 16 + 8 * x, j & 1);
          if (!ok) {
            break;
          }
          values(1);
          if (j + 1 < mine) {
            scores(j + 1);
          } else {
            umma::commit(o_final + 8 * x);
          }
        }
        end_turn();
        release(2 * j + 1, j < mine);
        if (more) {
          release(2 * j + 2, j + 1 < mine);
        }
      }
      if (!ok) {
        give_up();
      }
    } else if (warp == 9 && count > 0) {
      // ---- copies -------------------------------------------------------------------------------
      // Lane i < pages_per_tile fetches page i of a tile; its ids are read one tile ahead (and, for
      // 8-bit pages, the keys' scales).
      const int pages_per_tile = kTileTokens / p.page_size;
      const int entry = item.entry + item.first_token / p.page_size;
      const int pages = (loaded + p.page_size - 1) / p.page_size;
      const uint32_t bars_full = QUANT ? raw_full : full;
      const uint32_t bars_empty = QUANT ? raw_empty : empty;
      constexpr int kSlotCount = QUANT ? L::kRawSlots : L::kSlots;
      auto page_of = [&](int j) -> int {
        const int i = j * pages_per_tile + lane;
        if (lane >= pages_per_tile || i >= pages) {
          return -1;
        }
        const int page = __ldg(p.page_ids + entry + i);
        return min(max(page, 0), p.num_pages - 1);
      };
      auto scales_of = [&](int page) -> float2 {
        float2 v = make_float2(0.0f, 0.0f);
        if (QUANT && page >= 0) {
          const float* src = p.key_scales + (static_cast<size_t>(page) * p.num_kv_heads + item.kv_head) * kBlocks;
          v = kBlocks == 2 ? __ldg(reinterpret_cast<const float2*>(src)) : make_float2(__ldg(src), 0.0f);
        }
        return v;
      };
      int slot = 0;
      uint32_t uses = 0;  // how often the ring has gone round
      int issued = 0;
      bool ok = true;
      int page = page_of(0);
      float2 key_scale = scales_of(page);
      int next_page = count > 1 ? page_of(1) : -1;
      for (int j = 0; ok && j < count; ++j) {
        const float2 next_scale = scales_of(next_page);
        const int after_page = j + 2 < count ? page_of(j + 2) : -1;
        const int here = min(pages_per_tile, pages - j * pages_per_tile);  // pages of this tile
        for (int which = 0; which < 2; ++which) {  // keys, then values
          if (uses > 0) {
            ok = wait_all(bars_empty + 8 * slot, (uses - 1) & 1);
            if (!ok) {
              break;
            }
          }
          const uint32_t bar = bars_full + 8 * slot;
          if constexpr (QUANT) {
            const uint32_t page_bytes = p.page_size * D;
            const uint32_t scale_bytes = which == 1 ? p.page_size * kBlocks * 4 : 0;
            if (which == 0 && lane < here) {
              *reinterpret_cast<float2*>(smem + L::kRawKeyScales + slot * 64 + lane * 8) = key_scale;
            }
            proxy_fence_async();  // the slot was read through the generic proxy
            __syncwarp();
            if (lane == 0) {
              mbar_expect_tx(bar, here * (page_bytes + scale_bytes));
            }
            __syncwarp();
            if (lane < here) {
              const size_t page_head = static_cast<size_t>(page) * p.num_kv_heads + item.kv_head;
              const uint32_t dst = base + L::kRaw + slot * L::kRawSlotBytes;
              fk_page_decode::bulk_copy_plain(dst + lane * page_bytes,
                                              (which == 0 ? p.key_pages : p.value_pages) + page_head * page_bytes,
                                              page_bytes, bar);
              if (which == 1) {
                fk_page_decode::bulk_copy_plain(dst + L::kRawBytes + lane * scale_bytes,
                                                p.value_scales + page_head * (p.page_size * kBlocks), scale_bytes, bar);
              }
            }
          } else {
            if (lane == 0) {
              mbar_expect_tx(bar, here * p.page_size * (D * 2));
            }
            __syncwarp();
            if (lane < here) {
              const int y = (page * p.num_kv_heads + item.kv_head) * p.page_size;
              const uint32_t dst = base + L::kRing + slot * L::kOperandBytes + lane * p.page_size * 128;
#pragma unroll
              for (int h = 0; h < kBlocks; ++h) {
                tma_load_2d(dst + h * L::kHalfBytes, which == 0 ? &key_map : &value_map, 64 * h, y, bar);
              }
            }
          }
          ++issued;
          if (++slot == kSlotCount) {
            slot = 0;
            ++uses;
          }
        }
        page = next_page;
        key_scale = next_scale;
        next_page = after_page;
      }
      if (lane == 0) {
        *issued_slot = issued;
      }
      if (!ok) {
        give_up();
      }
    } else if (!QUANT && warp == 10 && clear_needed) {
      // ---- value rows behind the end ------------------------------------------------------------
      // The issuer says when they have landed: it follows the ring's phases one by one, and a wait for
      // a later phase's parity would be over at once.
      const int slot = (2 * count - 1) % L::kSlots;  // the last tile's values, in the order of the copies
      if (wait_all(v_landed, 0)) {
        const int valid = loaded - (count - 1) * kTileTokens;
        const uint32_t v_base = base + L::kRing + slot * L::kOperandBytes;
        for (int idx = lane; idx < (kTileTokens - valid) * kChunks; idx += 32) {
          sts128(v_base + operand_chunk(valid + idx / kChunks, idx % kChunks), make_uint4(0u, 0u, 0u, 0u));
        }
        proxy_fence_async();
        __syncwarp();
        if (lane == 0) {
          umma::mbar_arrive(v_clear);
        }
      } else {
        give_up();
      }
    } else if (QUANT && warp >= 12 && count > 0) {
      // ---- 8-bit tiles to 16 bits ---------------------------------------------------------------
      constexpr int kRowsPerPass = 128 / kChunks;  // 128 threads, 8 elements each
      constexpr int kPasses = kTileTokens / kRowsPerPass;
      // A thread's rows are first + pass * kRowsPerPass, a batch at a time: all loads, all arithmetic, all
      // stores. (The loads and stores are volatile: in the order of one row after the other every row
      // waits for the one before, 230 clocks each.)
      constexpr int kBatch = 4;
      constexpr int kRawSlots = QUANT ? L::kRawSlots : 1;
      const int t = tid - 384;
      const int page_shift = p.page_size == 16 ? 4 : 5;
      const int chunk = t % kChunks;
      const int block = chunk / 8;
      const int first = t / kChunks;
      // A warp that gives up goes on through the loop, as far as the barrier that it shares with the others.
      bool ok = true;
      for (int i = 0; i < 2 * count; ++i) {
        const int raw_slot = i % kRawSlots;
        const int slot = i % L::kSlots;
        const int raw_use = i / kRawSlots;
        const int use = i / L::kSlots;
        const int j = i >> 1;
        const bool keys = (i & 1) == 0;
        ok = ok && (use == 0 || wait_all(empty + 8 * slot, (use - 1) & 1)) && wait_all(raw_full + 8 * raw_slot, raw_use & 1);
        const uint32_t from = base + L::kRaw + raw_slot * L::kRawSlotBytes;
        const uint32_t to = base + L::kRing + slot * L::kOperandBytes;
        const int valid = min(kTileTokens, loaded - j * kTileTokens);
        // [128 rows][2 blocks], keys' and values' apart: the next operand's are written while this one's are read. (A
        // table of the keys' pages instead took four instructions more for every eight elements.)
        uint2* ratios = reinterpret_cast<uint2*>(smem + L::kRatios) + (i & 1) * kTileTokens;
        if (ok && keys) {
          const int page = t >> page_shift;
          const float2 s = *reinterpret_cast<const float2*>(smem + L::kRawKeyScales + raw_slot * 64 + page * 8);
          const float larger = fmaxf(s.x, s.y);
          if ((t & (p.page_size - 1)) == 0) {
            reinterpret_cast<float*>(smem + L::kKeyFactors)[(j % kFactorRing) * 8 + page] = kBlocks == 2 ? larger * (1.0f / kRatioPower) : larger;
          }
          if constexpr (kBlocks == 2) {
            ratios[t] = make_uint2(scale_ratio(s.x, larger), scale_ratio(s.y, larger));
          }
        } else if (ok) {
          // row t's larger scale, and what softmax adds to the logit to know the heaviest weight
          const float* scales = reinterpret_cast<const float*>(smem + L::kRaw + raw_slot * L::kRawSlotBytes + L::kRawBytes) + t * kBlocks;
          float larger = scales[0];
          if constexpr (kBlocks == 2) {
            larger = fmaxf(larger, scales[1]);
            ratios[t] = make_uint2(scale_ratio(scales[0], larger), scale_ratio(scales[1], larger));
          }
          float* factors = reinterpret_cast<float*>(smem + L::kValueFactors) + (j % kFactorRing) * kTileTokens + t;
          factors[0] = t < valid ? larger : 0.0f;
          // (a scale of 0 must not leave a tile without a finite heaviest weight, nor one near it make the sum of
          // probabilities, 2^(kGrowth - log) each at most, overflow; scales from 5e-31 on have all their weights' bits)
          const float log = t < valid ? __log2f(fmaxf(larger, 1e-24f)) : -INFINITY;
          factors[kFactorRing * kTileTokens] = log;
          float most = log;
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) {
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
          }
          if (lane == 0) {
            reinterpret_cast<float*>(smem + L::kTileLogs)[(j % kFactorRing) * 4 + (warp & 3)] = most;
          }
        }
        if constexpr (kBlocks == 2) {
          asm volatile("bar.sync 2, 128;" ::: "memory");  // the ratios, by the rows' other threads
        }
        if (!ok) {
          continue;
        }
        const uint32_t* my_ratios = reinterpret_cast<const uint32_t*>(ratios + first) + block;
        const uint32_t source = from + t * 8;
        const uint32_t target = to + operand_chunk(first, chunk);  // (rows of a pass are a multiple of 8 further on)
#pragma unroll 1
        for (int pass0 = 0; pass0 < kPasses; pass0 += kBatch) {
          uint2 w[kBatch];
          uint32_t ratio[kBatch];
#pragma unroll
          for (int b = 0; b < kBatch; ++b) {
            w[b] = lds64(source + (pass0 + b) * kRowsPerPass * D);
            ratio[b] = kBlocks == 2 ? my_ratios[(pass0 + b) * kRowsPerPass * 2] : 0u;
          }
#pragma unroll
          for (int b = 0; b < kBatch; ++b) {
            uint4 out;
            fk_page_decode::bytes_to_half2<KV, false>(w[b].x, out.x, out.y);
            fk_page_decode::bytes_to_half2<KV, false>(w[b].y, out.z, out.w);
            if constexpr (kBlocks == 2) {
              out.x = mul_half2(out.x, ratio[b]);
              out.y = mul_half2(out.y, ratio[b]);
              out.z = mul_half2(out.z, ratio[b]);
              out.w = mul_half2(out.w, ratio[b]);
            }
            sts128(target + (pass0 + b) * kRowsPerPass * 128, out);
          }
        }
        if (valid < kTileTokens) {
          // a row behind the end has weight 0, but what its page holds there times 0 need not be 0
          for (int row = first; row < kTileTokens; row += kRowsPerPass) {
            if (row >= valid) {
              sts128(to + operand_chunk(row, chunk), make_uint4(0u, 0u, 0u, 0u));
            }
          }
        }
        proxy_fence_async();
        __syncwarp();
        if (lane == 0) {
          umma::mbar_arrive(full + 8 * slot);
          umma::mbar_arrive(raw_empty + 8 * raw_slot);
        }
      }
      if (!ok) {
        give_up();
      }
    }
  }

  __syncwarp();
  umma::fence_before_sync();
  __syncthreads();
  umma::fence_after_sync();
  if (*fail_flag != 0u) {
    // whatever is in flight still is let land before the memory is handed on: products, copies
    if ((warp == 8 || warp == 11) && lane == 0) {
      umma::commit(drain);
    }
    __syncwarp();
    if (warp == 8) {
      (void)wait_all(drain, 0);
    } else if (warp == 9) {
      constexpr int kSlotCount = QUANT ? L::kRawSlots : L::kSlots;
      const int issued = *issued_slot;
      for (int i = max(0, issued - kSlotCount); i < issued; ++i) {
        (void)wait_all((QUANT ? raw_full : full) + 8 * (i % kSlotCount), (i / kSlotCount) & 1);
      }
    }
  }
  if (warp == 8) {
    umma::tmem_dealloc(tmem, 512);
  }
}

}  // namespace fk_paged_kv
