// Products with 4-bit weights for few rows, and for f32 activations of any number of rows (w4.cuh has the layout):
//   y = x W^T + bias,  or  y = act(x W^T) * (x up^T) with both products, the activation and the multiplication in this one kernel.
//
// Bound by the weights' way from HBM: 0.53 bytes a weight. Weights are the M operand of mma.sync (16 rows of 16 k), tokens its N. A code less its zero
// point is a whole number of at most 15, exact in bf16; so the products are exact, a group is summed in f32, and the scale multiplies that sum in f32:
// nothing is rounded but sums. Dequantisation is one AND and one fused multiply-add per PAIR of weights (plus a shift per eight): the masked pair, read
// as bf16, is code * 2^-133 or code * 2^-129 (subnormal numbers are multiples of 2^-133, and so are those of the first binade above them), and
// fma(pair, 2^120 or 2^116, -zero * 2^-13) = (code - zero) * 2^-13, exactly.
//
// f32 activations go through the same instructions as three bf16 terms of eight bits each: hi + mid + lo = x exactly down to the smallest bf16 number, 2^-133, so
// that values of 2^-109 and more have all of their 24 bits, and f32 results f32 accuracy.
// The warps that share a slab of tokens make its terms together (211 rows of k 2048 to 5504 outputs: 98 us with each warp making its own, 90 together). More than
// 16 rows are bound by these instructions, so two CTAs share an SM there too (512 rows of k 4096 to 14336: 734 us with one of up to 210 registers a thread,
// 562 with two of 128, which spill some registers; 211 rows as above 90 and 79. With small results kept, below, 569 and 81).
//
// A CTA of eight warps, two CTAs to an SM: WR warps side by side over weight rows, 8 / WR groups of them over k. Few tokens: WR = 4, and the tokens' slab of a
// k group serves 128 rows; more tokens: all eight warps share it, so that L2 delivers it less often. Each k group has a ring of slabs of 128 or 256 k, weights,
// tokens and scales, filled by cp.async (no waits on barriers). A CTA has one tile: CTAs that went from tile to tile, the rings running ahead, left more of
// the device idle at the end (8 rows of k 4096 to 128256 outputs: 68 us against 62). Sums of k groups meet in shared memory, and where the rows of weights
// give too few CTAs the k of a tile is dealt to the CTAs of a cluster, whose sums meet over distributed shared memory: in both places in a fixed order, so
// results do not vary from run to run, and no workspace is needed.
//
// Measured: 8 rows of k 4096 to 128256 outputs 64 to 67 us, 4.2 to 4.4 TB/s (0.64 to 0.67 of a copy's rate), 1 row of k 4096 with a gate to 14336 16.7 us,
// 3.6 TB/s. Instructions are issued in 54 % of all cycles (k 4096 to 32768: 17 for the eight weights of a lane, nine of which are the dequantisation), from
// 16 warps to an SM that also wait for each other's slabs: neither bound is reached alone. Of many f32 rows mma.sync is the bound, three terms a product.
#include "kernels.h"
#include "mma.cuh"
#include "w4.cuh"

#include <algorithm>

namespace orion {
namespace {

constexpr uint32_t kThreads = 256, kWarps = 8;
constexpr float kUnit = 8192.f;        // dequantised codes are multiples of 1 / kUnit: a group's sum stays finite for any tokens that are

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void sts128_zero(uint32_t addr) { asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(addr), "r"(0u) : "memory"); }
__device__ __forceinline__ void sts128(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void sts32(uint32_t addr, uint32_t v) { asm volatile("st.shared.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }
__device__ __forceinline__ void sts16(uint32_t addr, uint32_t v) { asm volatile("st.shared.u16 [%0], %1;" ::"r"(addr), "h"((uint16_t)v) : "memory"); }
__device__ __forceinline__ void sts8(uint32_t addr, uint32_t v) { asm volatile("st.shared.u8 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }
__device__ __forceinline__ void cp_async4(uint32_t dst, const void *src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
template <uint32_t N>
__device__ __forceinline__ void lds_words(uint32_t addr, uint32_t (&w)[N]) {
  if constexpr (N == 1) w[0] = lds32(addr);
  if constexpr (N == 2) asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr) : "memory");
  if constexpr (N == 4) asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t lds16(uint32_t addr) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t lds8(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr, uint32_t rank) {
  uint32_t remote;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(addr), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t fma_bf16x2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
// Tiles of 16 rows x 8 k of codes as fragments: pairs (0,1), (2,3), (4,5), (6,7) of a word, less the zero point, times 2^-13.
__device__ __forceinline__ void dequant(uint32_t word, uint32_t minus_zero, uint32_t (&pair)[4]) {
  constexpr uint32_t kLow = 0x7b807b80u, kHigh = 0x79807980u;  // 2^120, 2^116
  const uint32_t rest = word >> 8;
  pair[0] = fma_bf16x2(word & 0x000f000fu, kLow, minus_zero);
  pair[1] = fma_bf16x2(word & 0x00f000f0u, kHigh, minus_zero);
  pair[2] = fma_bf16x2(rest & 0x000f000fu, kLow, minus_zero);
  pair[3] = fma_bf16x2(rest & 0x00f000f0u, kHigh, minus_zero);
}
// d = a b (+ c)
__device__ __forceinline__ void mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
// What is left of x beyond its first eight bits; nothing of an infinity.
__device__ __forceinline__ float beyond(float x, float first) { return x == first ? 0.f : x - first; }
__device__ __forceinline__ float first_bits(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }
__device__ __forceinline__ uint32_t upper_halves(float a, float b) { return __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632); }

template <typename T, bool GATED, bool ZEROS, uint32_t GROUP, uint32_t RT, uint32_t NT, uint32_t WR>
struct FewConfig {
  static_assert(RT % (GATED ? 2 : 1) == 0, "with a gate half of a warp's tiles are the gate's");
  static constexpr uint32_t kKGroups = kWarps / WR;
  static constexpr uint32_t kTileRows = 16 * RT * WR;                       // rows of weights per CTA, gate and up together
  static constexpr uint32_t kMatrices = GATED ? 2 : 1;
  static constexpr uint32_t kOutputs = kTileRows / kMatrices;               // columns of y
  static constexpr uint32_t kTokens = 8 * NT;
  static constexpr uint32_t kSlab = NT == 1 && sizeof(T) == 2 ? 256 : 128, kWRow = kSlab / 2;  // k of a slab, bytes of a weight row in it
  static constexpr uint32_t kXRow = kSlab * sizeof(T);
  static constexpr uint32_t kWStage = kTileRows * kWRow;
  static constexpr uint32_t kPerSlab = kSlab / GROUP;                       // groups in a slab
  static constexpr uint32_t kScaleRow = kOutputs * 2, kZeroRow = kOutputs;  // scales, and zero points, of a group and matrix
  static constexpr uint32_t kSStage = kMatrices * kPerSlab * (kScaleRow + (ZEROS ? kZeroRow : 0));
  static constexpr uint32_t kSums = kKGroups * kTokens * kTileRows * 4;     // bytes of the sums that meet in shared memory, over the rings
  // Slabs in the ring: what leaves room for two CTAs in an SM.
  static constexpr uint32_t kStages = kSlab == 256 || (sizeof(T) == 4 && NT == 4 && RT == 2) ? 2 : NT <= 2 || sizeof(T) == 4 ? 3 : 4;
  static constexpr uint32_t kStage = kWStage + kTokens * kXRow + kSStage, kRings = kKGroups * kStages * kStage;
  // f32 tokens of the slab at hand, in bf16 terms: [term][token][k]
  static constexpr uint32_t kTermRow = kSlab * 2, kTerms = sizeof(T) == 4 ? 3 * kTokens * kTermRow : 0, kAll = kRings + kKGroups * kTerms;
  static constexpr uint32_t kSmem = kAll > kSums ? kAll : kSums;
  static_assert(kSmem <= 113 * 1024, "rings of two CTAs exceed the shared memory of an SM");
};

template <typename T, bool GATED, bool ZEROS, uint32_t GROUP, uint32_t RT, uint32_t NT, uint32_t WR>
__global__ void __launch_bounds__(kThreads, 2)
w4_few_kernel(const W4Call c, const uint32_t tiles_m) {
  using Cfg = FewConfig<T, GATED, ZEROS, GROUP, RT, NT, WR>;
  constexpr bool kF32 = sizeof(T) == 4;
  constexpr uint32_t kPerSlab = Cfg::kPerSlab, kStages = Cfg::kStages, kStageBytes = Cfg::kStage, kSlab = Cfg::kSlab, kWRow = Cfg::kWRow;
  extern __shared__ __align__(128) uint8_t smem[];
  pdl_trigger();

  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t kg = warp / WR, wr = warp % WR, in_kg = wr * 32 + lane;
  const uint32_t ranks = gridDim.z, rank = blockIdx.z;
  const uint32_t slabs = (c.k + kSlab - 1) / kSlab, units = Cfg::kKGroups * ranks, unit = rank * Cfg::kKGroups + kg;
  const uint32_t mine = unit < slabs ? (slabs - unit + units - 1) / units : 0;  // slabs of a tile that this k group takes
  const uint32_t groups = c.k / GROUP;
  const uint32_t ring = smem_u32(smem) + kg * kStages * kStageBytes, terms = smem_u32(smem) + Cfg::kRings + kg * Cfg::kTerms;
  auto sync_k_group = [&] {
    if constexpr (WR == kWarps) __syncthreads();
    else asm volatile("bar.sync %0, %1;" ::"r"(kg + 1), "n"(WR * 32) : "memory");
  };
  const uint32_t n0 = blockIdx.x / tiles_m * Cfg::kOutputs, m0 = blockIdx.x % tiles_m * Cfg::kTokens, tokens = min(Cfg::kTokens, c.rows - m0);

  // First output of a tile of 16 rows within the CTA's; with a gate the first half of a warp's tiles are the gate's.
  constexpr uint32_t kTilesPerMatrix = RT / Cfg::kMatrices;
  auto col_of = [&](uint32_t rt) { return (wr * kTilesPerMatrix + rt % kTilesPerMatrix) * 16; };
  auto matrix_of = [&](uint32_t rt) { return rt / kTilesPerMatrix; };
  pdl_wait();

  // Scales and zero points of a slab. Where the outputs are whole words (n a multiple of 4) they come by cp.async like the rest, zeros in place of groups
  // beyond the last. Else they pass through registers: asked for with the slab's loads, stored after the products of
  // the slab before, ahead of the barrier that lets the warps at them.
  constexpr uint32_t kScaleWords = Cfg::kOutputs / 2, kZeroWords = Cfg::kOutputs / 4, kRowsOfParams = Cfg::kMatrices * kPerSlab;
  constexpr uint32_t kParamTurns = (kRowsOfParams * Cfg::kOutputs + WR * 32 - 1) / (WR * 32);
  const bool words = (c.n & 3) == 0;
  uint32_t held_s[kParamTurns], held_z[kParamTurns], held_at = 0;  // as loaded, and where they go
  auto store_held = [&] {
    if (words || !held_at) return;
#pragma unroll
    for (uint32_t j = 0; j < kParamTurns; ++j) {
      const uint32_t i = in_kg + j * WR * 32, row = i / Cfg::kOutputs, col = i % Cfg::kOutputs;
      if (row < kRowsOfParams) {
        sts16(held_at + row * Cfg::kScaleRow + col * 2, held_s[j]);
        if (ZEROS) sts8(held_at + kRowsOfParams * Cfg::kScaleRow + row * Cfg::kZeroRow + col, held_z[j]);
      }
    }
    held_at = 0;
  };
  constexpr uint32_t kScaleTurns = (kRowsOfParams * kScaleWords + WR * 32 - 1) / (WR * 32), kZeroTurns = (kRowsOfParams * kZeroWords + WR * 32 - 1) / (WR * 32);
  const uint64_t slab_step = (uint64_t)units * kPerSlab * c.n;  // scales from one slab to the next
  const bf16 *load_s[kScaleTurns];
  const uint8_t *load_z[kZeroTurns];
#pragma unroll
  for (uint32_t j = 0; j < kScaleTurns; ++j) {
    const uint32_t i = in_kg + j * WR * 32, row = i / kScaleWords;
    load_s[j] = (row >= kPerSlab ? c.up.scales : c.w.scales) + (uint64_t)(unit * kPerSlab + row % kPerSlab) * c.n + n0 + i % kScaleWords * 2;
  }
#pragma unroll
  for (uint32_t j = 0; ZEROS && j < kZeroTurns; ++j) {
    const uint32_t i = in_kg + j * WR * 32, row = i / kZeroWords;
    const uint8_t *p = row >= kPerSlab ? c.up.zeros : c.w.zeros;
    load_z[j] = p ? p + (uint64_t)(unit * kPerSlab + row % kPerSlab) * c.n + n0 + i % kZeroWords * 4 : nullptr;
  }
  auto load_params = [&](uint32_t s_at, uint32_t slab, bool whole) {
    if (words) {
#pragma unroll
      for (uint32_t j = 0; j < kScaleTurns; ++j) {
        const uint32_t i = in_kg + j * WR * 32, row = i / kScaleWords, col = i % kScaleWords * 2;
        if (row < kRowsOfParams) {
          if (whole || (slab * kPerSlab + row % kPerSlab < groups && n0 + col < c.n)) cp_async4(s_at + row * Cfg::kScaleRow + col * 2, load_s[j]);
          else sts32(s_at + row * Cfg::kScaleRow + col * 2, 0);
        }
        load_s[j] += slab_step;
      }
#pragma unroll
      for (uint32_t j = 0; ZEROS && j < kZeroTurns; ++j) {
        const uint32_t i = in_kg + j * WR * 32, row = i / kZeroWords, col = i % kZeroWords * 4, at = s_at + kRowsOfParams * Cfg::kScaleRow + row * Cfg::kZeroRow + col;
        if (row < kRowsOfParams) {
          if (load_z[j] && (whole || (slab * kPerSlab + row % kPerSlab < groups && n0 + col < c.n))) cp_async4(at, load_z[j]);
          else sts32(at, 0x08080808u);
        }
        if (load_z[j]) load_z[j] += slab_step;
      }
    } else {
      held_at = s_at;
#pragma unroll
      for (uint32_t j = 0; j < kParamTurns; ++j) {
        const uint32_t i = in_kg + j * WR * 32, row = i / Cfg::kOutputs, col = i % Cfg::kOutputs, group = slab * kPerSlab + row % kPerSlab;
        held_s[j] = 0, held_z[j] = 8;
        if (row < kRowsOfParams && group < groups && n0 + col < c.n) {
          const W4View &w = row >= kPerSlab ? c.up : c.w;
          const uint64_t at = (uint64_t)group * c.n + n0 + col;
          held_s[j] = __ldg(reinterpret_cast<const uint16_t *>(w.scales) + at);
          if (ZEROS && w.zeros) held_z[j] = __ldg(w.zeros + at);
        }
      }
    }
  };

  // Weight rows of 64 or 128 bytes, their 16-byte pieces permuted so that the eight rows of a fragment lie in different banks; a lane copies one piece of
  // every fourth or eighth row of its warp's tiles. Rows beyond the last are left as they are: nothing of them is stored. Token rows: every other one with its
  // halves of 64 bytes exchanged, zeros beyond the last k.
  constexpr uint32_t kPieces = Cfg::kXRow / 16, kPer = 16 / sizeof(T), kXTurns = (Cfg::kTokens * kPieces + WR * 32 - 1) / (WR * 32);
  constexpr uint32_t kXStep = WR * 32 / kPieces;  // token rows from one turn to the next, an even number
  static_assert(kXStep % 2 == 0, "rows of a lane's turns are permuted alike");
  constexpr uint32_t kWPieces = kSlab / 32, kWStep = 32 / kWPieces, kWTurns = kTilesPerMatrix * 16 / kWStep;  // rows from one turn to the next, turns per matrix
  const uint32_t w_row = lane / kWPieces, w_piece = lane % kWPieces;
  // Where a piece goes within its row, so that the rows that are read together lie in different banks: eight of them 4 bytes a lane (groups of 32), four 8
  // bytes (64), two 16 bytes (128). Of rows of 128 bytes every other turn has row & 4 set.
  constexpr uint32_t kWide = GROUP / 32, kBlock = 32 * kWide;  // words of a row that a lane takes together, k of the four lanes of a row
  auto w_place = [](uint32_t piece, uint32_t row) {
    if (kWPieces == 8) return piece ^ (kWide == 1 ? row & 7 : kWide == 2 ? (row & 3) << 1 : (row & 1) << 2);
    return piece ^ (kWide == 1 ? (row >> 1) & 3 : kWide == 2 ? row & 2 : 0);
  };
  const uint32_t w_to = wr * RT * 16 * kWRow + w_row * kWRow;
  const uint32_t w_to_places[2] = {w_to + w_place(w_piece, w_row) * 16, w_to + w_place(w_piece, w_row + kWStep) * 16};
  auto x_place = [](uint32_t piece, uint32_t row) {  // likewise: lanes read pieces kWide apart, of two rows together
    return piece ^ (kWide == 1 ? (row & 1) << 2 : row & 1) ^ (kWide == 4 ? (piece >> 3 & 1) << 1 : 0);
  };
  const uint32_t x_row = in_kg / kPieces, x_piece = in_kg % kPieces, x_to = Cfg::kWStage + x_row * Cfg::kXRow + (kF32 ? x_piece ^ (x_row & 1) << 2 : x_place(x_piece, x_row)) * 16;
  const uint64_t w_step = (uint64_t)c.k / 2 * kWStep, x_step = kXStep * c.ldx * sizeof(T);  // bytes
  const uint32_t first_row = n0 + wr * kTilesPerMatrix * 16 + w_row, rows_there = first_row < c.n ? (c.n - first_row + kWStep - 1) / kWStep : 0;  // per matrix
  const uint64_t first_at = ((uint64_t)first_row * (c.k / 8) + unit * (kSlab / 8) + w_piece * 4) * 4;
  const uint8_t *load_w[Cfg::kMatrices];
  load_w[0] = reinterpret_cast<const uint8_t *>(c.w.packed) + first_at;
  if (GATED) load_w[Cfg::kMatrices - 1] = reinterpret_cast<const uint8_t *>(c.up.packed) + first_at;
  const uint8_t *load_x = static_cast<const uint8_t *>(c.x) + ((uint64_t)(m0 + x_row) * c.ldx + unit * kSlab + x_piece * kPer) * sizeof(T);
  const bool whole_rows = n0 + Cfg::kOutputs <= c.n;
  uint32_t load_index = 0, load_slot = 0;
  auto load = [&] {  // the next slab of this k group
    store_held();
    if (load_index < mine) {
      const uint32_t slab = unit + load_index * units, k0 = slab * kSlab, base = ring + load_slot * kStageBytes;
      const uint32_t to[2] = {base + w_to_places[0], base + w_to_places[1]};
      const bool whole = whole_rows && k0 + kSlab <= c.k;
      if (whole) {
#pragma unroll
        for (uint32_t i = 0; i < Cfg::kMatrices * kWTurns; ++i) cp_async16(to[i % 2] + i * kWStep * kWRow, load_w[i / kWTurns] + i % kWTurns * w_step);
      } else {
        const uint32_t rows = k0 + w_piece * 32 < c.k ? rows_there : 0;
#pragma unroll
        for (uint32_t i = 0; i < Cfg::kMatrices * kWTurns; ++i)
          if (i % kWTurns < rows) cp_async16(to[i % 2] + i * kWStep * kWRow, load_w[i / kWTurns] + i % kWTurns * w_step);
      }
#pragma unroll
      for (uint32_t m = 0; m < Cfg::kMatrices; ++m) load_w[m] += units * kWRow;
      const bool x_inside = k0 + x_piece * kPer < c.k;
#pragma unroll
      for (uint32_t j = 0; j < kXTurns; ++j) {
        const uint32_t row = x_row + j * kXStep;
        if (row < tokens && x_inside) cp_async16(base + x_to + j * kXStep * Cfg::kXRow, load_x + j * x_step);
        else if (row < tokens) sts128_zero(base + x_to + j * kXStep * Cfg::kXRow);
      }
      load_x += (uint64_t)units * kSlab * sizeof(T);
      load_params(base + Cfg::kWStage + Cfg::kTokens * Cfg::kXRow, slab, whole);
      ++load_index;
      load_slot = load_slot + 1 == kStages ? 0 : load_slot + 1;
    }
    cp_async_commit();
  };
  // token rows that nothing is loaded to
  for (uint32_t s = 0; s < kStages; ++s)
    for (uint32_t i = tokens * kPieces + in_kg; i < Cfg::kTokens * kPieces; i += WR * 32) sts128_zero(ring + s * kStageBytes + Cfg::kWStage + i * 16);
#pragma unroll
  for (uint32_t s = 0; s + 1 < kStages; ++s) load();
  store_held();

  // Offsets in a stage of this lane's words of a block of its weight rows
  uint32_t w_from[kSlab / kBlock];
#pragma unroll
  for (uint32_t i = 0; i < kSlab / kBlock; ++i)
    w_from[i] = (wr * RT * 16 + g) * kWRow + w_place(i * kWide + t * kWide / 4, g) * 16 + t * kWide % 4 * 4;

  float sum[RT][NT][4];
#pragma unroll
  for (uint32_t rt = 0; rt < RT; ++rt)
#pragma unroll
    for (uint32_t nt = 0; nt < NT; ++nt)
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) sum[rt][nt][i] = 0.f;

  uint32_t slot = 0;
  for (uint32_t index = 0; index < mine; ++index) {
    cp_async_wait<kStages - 2>();
    sync_k_group();
    load();

    const uint32_t base = ring + slot * kStageBytes, s_at = base + Cfg::kWStage + Cfg::kTokens * Cfg::kXRow;
    const uint32_t z_at = s_at + kRowsOfParams * Cfg::kScaleRow;
    if constexpr (kF32) {  // the terms of the slab's values, once for all warps of the k group
      for (uint32_t i = in_kg; i < Cfg::kTokens * (kSlab / 8); i += WR * 32) {
        const uint32_t row = i / (kSlab / 8), piece = i % (kSlab / 8), at = base + Cfg::kWStage + row * Cfg::kXRow + (2 * piece ^ (row & 1) << 2) * 16;
        const uint4 lo = lds128(at), hi = lds128(at + 16);
        float v[8] = {__uint_as_float(lo.x), __uint_as_float(lo.y), __uint_as_float(lo.z), __uint_as_float(lo.w),
                      __uint_as_float(hi.x), __uint_as_float(hi.y), __uint_as_float(hi.z), __uint_as_float(hi.w)};
#pragma unroll
        for (uint32_t term = 0; term < 3; ++term) {
          sts128(terms + (term * Cfg::kTokens + row) * Cfg::kTermRow + x_place(piece, row) * 16, upper_halves(v[0], v[1]), upper_halves(v[2], v[3]),
                 upper_halves(v[4], v[5]), upper_halves(v[6], v[7]));
#pragma unroll
          for (uint32_t j = 0; j < 8; ++j) v[j] = beyond(v[j], first_bits(v[j]));
        }
      }
      sync_k_group();
    }
    slot = slot + 1 == kStages ? 0 : slot + 1;
    float part[RT][NT][4];
    uint32_t minus_zero[RT][2], words[RT][2][kWide];
#pragma unroll
    for (uint32_t q = 0; q < kSlab / 32; ++q) {  // a word of the lane's, 32 k of the four lanes of a row
      const bool begins = q * 32 % GROUP == 0, ends = (q + 1) * 32 % GROUP == 0;
      if (begins) {
#pragma unroll
        for (uint32_t rt = 0; rt < RT; ++rt)
#pragma unroll
          for (uint32_t h = 0; h < 2; ++h) {
            minus_zero[rt][h] = 0xba80ba80u;  // -8 / kUnit
            if (ZEROS) {
              const uint32_t row = matrix_of(rt) * kPerSlab + q * 32 / GROUP;
              // as the codes: at most eight bits, so exact
              minus_zero[rt][h] = fma_bf16x2(lds8(z_at + row * Cfg::kZeroRow + col_of(rt) + h * 8 + g) * 0x10001u, 0xfb80fb80u, 0x80008000u);
            }
          }
      }
      if (q % kWide == 0) {
#pragma unroll
        for (uint32_t rt = 0; rt < RT; ++rt)
#pragma unroll
          for (uint32_t h = 0; h < 2; ++h) lds_words<kWide>(base + w_from[q / kWide] + (rt * 16 + h * 8) * kWRow, words[rt][h]);
      }
      uint32_t a[RT][2][4];  // [rows 0-7 / 8-15][pair]
#pragma unroll
      for (uint32_t rt = 0; rt < RT; ++rt)
#pragma unroll
        for (uint32_t h = 0; h < 2; ++h) dequant(words[rt][h][q % kWide], minus_zero[rt][h], a[rt][h]);
#pragma unroll
      for (uint32_t nt = 0; nt < NT; ++nt) {
        auto multiply = [&](const uint32_t (&b)[4], bool first) {
#pragma unroll
          for (uint32_t rt = 0; rt < RT; ++rt)
#pragma unroll
            for (uint32_t half = 0; half < 2; ++half) {
              const uint32_t frag[4] = {a[rt][0][2 * half], a[rt][1][2 * half], a[rt][0][2 * half + 1], a[rt][1][2 * half + 1]};
              if (first && half == 0) mma_first(part[rt][nt], frag, b[2 * half], b[2 * half + 1]);
              else mma_bf16_16816(part[rt][nt], frag, b[2 * half], b[2 * half + 1]);
            }
        };
        const uint32_t x_piece_at = q / kWide * (kBlock / 8) + t * kWide + q % kWide;  // the 8 k of the word
        if constexpr (kF32) {
#pragma unroll
          for (uint32_t term = 0; term < 3; ++term) {
            const uint4 r = lds128(terms + (term * Cfg::kTokens + nt * 8 + g) * Cfg::kTermRow + x_place(x_piece_at, g) * 16);
            const uint32_t b[4] = {r.x, r.y, r.z, r.w};
            multiply(b, begins && term == 0);
          }
        } else {
          const uint4 r = lds128(base + Cfg::kWStage + (nt * 8 + g) * Cfg::kXRow + x_place(x_piece_at, g) * 16);
          const uint32_t b[4] = {r.x, r.y, r.z, r.w};
          multiply(b, begins);
        }
      }
      if (ends) {
#pragma unroll
        for (uint32_t rt = 0; rt < RT; ++rt)
#pragma unroll
          for (uint32_t h = 0; h < 2; ++h) {
            const uint32_t row = matrix_of(rt) * kPerSlab + q * 32 / GROUP;
            const float scale = __uint_as_float(lds16(s_at + row * Cfg::kScaleRow + (col_of(rt) + h * 8 + g) * 2) << 16);
            // Sums of f32 are held as they are: in kUnit they would lose bits below 2^-113, where those of bf16 have bits to spare. So kUnit goes to the scale, or
            // to the group's sums where the scale times kUnit would not be finite. (One test for all of a lane's scales is no faster: 211 rows of k 2048 to 5504
            // outputs 78.9 us without, 81.4 so, 82.5 with one.)
            const bool large = kF32 && fabsf(scale) >= 0x1p114f;
            const float per_unit = kF32 && !large ? scale * kUnit : scale;
            if (large) {
#pragma unroll
              for (uint32_t nt = 0; nt < NT; ++nt) part[rt][nt][2 * h] *= kUnit, part[rt][nt][2 * h + 1] *= kUnit;
            }
#pragma unroll
            for (uint32_t nt = 0; nt < NT; ++nt)
#pragma unroll
              for (uint32_t i = 2 * h; i < 2 * h + 2; ++i) sum[rt][nt][i] = fmaf(part[rt][nt][i], per_unit, sum[rt][nt][i]);
          }
      }
    }
    store_held();
  }

  // The k groups' sums, [k group][token][row], over the rings
  cp_async_wait<0>();
  __syncthreads();
  float *const sums = reinterpret_cast<float *>(smem);
#pragma unroll
  for (uint32_t rt = 0; rt < RT; ++rt)
#pragma unroll
    for (uint32_t nt = 0; nt < NT; ++nt)
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) {
        const uint32_t token = nt * 8 + t * 2 + (i & 1);
        if (token < tokens) sums[(kg * Cfg::kTokens + token) * Cfg::kTileRows + (wr * RT + rt) * 16 + (i >> 1) * 8 + g] = kF32 ? sum[rt][nt][i] : sum[rt][nt][i] * kUnit;
      }
  if (ranks > 1) cluster_barrier();
  else __syncthreads();
  auto total = [&](uint32_t token, uint32_t row) {
    float v = 0.f;
    for (uint32_t r = 0; r < ranks; ++r) {
#pragma unroll
      for (uint32_t j = 0; j < Cfg::kKGroups; ++j) {
        const float *p = sums + (j * Cfg::kTokens + token) * Cfg::kTileRows + row;
        v += ranks == 1 ? *p : ld_cluster_f32(smem_u32(p), r);
      }
    }
    return v;
  };
  for (uint32_t i = rank * kThreads + threadIdx.x; i < tokens * Cfg::kOutputs; i += ranks * kThreads) {
    const uint32_t token = i / Cfg::kOutputs, col = i % Cfg::kOutputs;
    if (n0 + col >= c.n) continue;
    float y;
    if constexpr (GATED) {
      constexpr uint32_t kHalf = kTilesPerMatrix * 16;
      const uint32_t at = col / kHalf * (2 * kHalf) + col % kHalf;
      y = gated<T>(GatedAct{c.act, 0.f}, total(token, at), total(token, at + kHalf));
    } else {
      y = total(token, col) + (c.bias ? c.bias[n0 + col] : 0.f);
    }
    static_cast<T *>(c.out)[(uint64_t)(m0 + token) * c.ldo + n0 + col] = from_f32<T>(y);
  }
  if (ranks > 1) cluster_barrier();  // nobody leaves while its sums are being read
}

template <typename Cfg>
uint32_t tiles_m_of(const W4Call &c) { return (c.rows + Cfg::kTokens - 1) / Cfg::kTokens; }
template <typename Cfg>
uint64_t tiles_of(const W4Call &c) { return (uint64_t)((c.n + Cfg::kOutputs - 1) / Cfg::kOutputs) * tiles_m_of<Cfg>(c); }

// CTAs that share the k of a tile, a cluster of up to eight where there are few tiles: as many as are at work together, two to an SM, less those that would
// not shorten the most slabs a k group has. A cluster starts when it has room for all of its CTAs, so one too many costs a second turn: 64 rows of k 3584 to
// 4608 outputs (36 tiles) take 40, 33, 29, 21, 20, 18, 17 and 21 us with one to eight, 1 row of k 4096 to 28672 (224 tiles) 18, 30 with two and 45 with four.
template <typename Cfg>
uint32_t ranks_of(const W4Call &c) {
  const uint64_t tiles = tiles_of<Cfg>(c);
  const uint32_t slabs = (c.k + Cfg::kSlab - 1) / Cfg::kSlab;
  auto steps = [&](uint32_t ranks) { return (slabs + Cfg::kKGroups * ranks - 1) / (Cfg::kKGroups * ranks); };
  uint32_t ranks = 1;
  for (uint32_t r = 2; r <= 8 && tiles * r <= 256; ++r)
    if (steps(r) < steps(ranks)) ranks = r;
  return ranks;
}
template <typename Cfg>
uint64_t ctas_of(const W4Call &c) { return tiles_of<Cfg>(c) * ranks_of<Cfg>(c); }

template <typename T, bool GATED, bool ZEROS, uint32_t GROUP, uint32_t RT, uint32_t NT, uint32_t WR>
int launch_config(const W4Call &c, cudaStream_t stream) {
  using Cfg = FewConfig<T, GATED, ZEROS, GROUP, RT, NT, WR>;
  static bool done[kMaxDeviceOrdinals] = {};
  const auto kernel = w4_few_kernel<T, GATED, ZEROS, GROUP, RT, NT, WR>;
  ORION_CUDA_CHECK("4-bit product", ensure_dynamic_smem(kernel, (int)Cfg::kSmem, done));
  const uint32_t tiles_m = tiles_m_of<Cfg>(c), ranks = ranks_of<Cfg>(c);
  const uint64_t tiles = tiles_of<Cfg>(c);
  if (tiles > 0x7fffffffull) return set_error(ORION_ERR_INVALID_REQUEST, "4-bit product: %u rows x %u outputs are too many for one call", c.rows, c.n);
  if (ranks == 1)
    ORION_CUDA_CHECK("4-bit product", launch_pdl(kernel, dim3((uint32_t)tiles), dim3(kThreads), Cfg::kSmem, stream, c, tiles_m));
  else
    ORION_CUDA_CHECK("4-bit product", launch_pdl_cluster(kernel, dim3((uint32_t)tiles, 1, ranks), dim3(kThreads), dim3(1, 1, ranks), Cfg::kSmem, stream, c, tiles_m));
  count_launch();
  return ORION_OK;
}

// Eight warps side by side: tiles of 256 rows, or of 128 where the CTAs of the wide ones would not fill the device (f32, 24 rows of k 4096 to 4096: 17 us, 26
// with wide ones; 12 rows of k 4096 to 14336: 32 and 27). A gate needs two tiles a warp.
template <typename T, bool GATED, bool ZEROS, uint32_t GROUP, uint32_t NT>
int launch_wide(const W4Call &c, cudaStream_t stream) {
  if constexpr (!GATED) {
    if (ctas_of<FewConfig<T, GATED, ZEROS, GROUP, 2, NT, 8>>(c) < 224) return launch_config<T, GATED, ZEROS, GROUP, 1, NT, 8>(c, stream);
  }
  return launch_config<T, GATED, ZEROS, GROUP, 2, NT, 8>(c, stream);
}

template <typename T, bool GATED, bool ZEROS, uint32_t GROUP>
int launch_shape(const W4Call &c, cudaStream_t stream) {
  if (c.rows <= 8) return launch_config<T, GATED, ZEROS, GROUP, 2, 1, 4>(c, stream);
  if constexpr (sizeof(T) == 2) {
    if (c.rows <= 16) return launch_config<T, GATED, ZEROS, GROUP, 2, 2, 4>(c, stream);
    if constexpr (!GATED) {
      // 64 tokens a tile unless 32 give more CTAs and the device is not full
      using Long = FewConfig<T, GATED, ZEROS, GROUP, 1, 8, 8>;
      if (c.rows > 32 && ctas_of<Long>(c) >= std::min<uint64_t>(148, ctas_of<FewConfig<T, GATED, ZEROS, GROUP, 1, 4, 8>>(c))) return launch_config<T, GATED, ZEROS, GROUP, 1, 8, 8>(c, stream);
    }
  } else {
    if (c.rows <= 16) return launch_wide<T, GATED, ZEROS, GROUP, 2>(c, stream);
  }
  return launch_wide<T, GATED, ZEROS, GROUP, 4>(c, stream);
}

template <typename T, bool GATED, bool ZEROS>
int launch_group(const W4Call &c, cudaStream_t stream) {
  switch (c.group) {
    case 32: return launch_shape<T, GATED, ZEROS, 32>(c, stream);
    case 64: return launch_shape<T, GATED, ZEROS, 64>(c, stream);
    default: return launch_shape<T, GATED, ZEROS, 128>(c, stream);
  }
}

}  // namespace

template <typename T>
int launch_w4_few(const W4Call &c, cudaStream_t stream) {
  const bool zeros = c.w.zeros || c.up.zeros;
  if (c.up.packed) return zeros ? launch_group<T, true, true>(c, stream) : launch_group<T, true, false>(c, stream);
  return zeros ? launch_group<T, false, true>(c, stream) : launch_group<T, false, false>(c, stream);
}
template int launch_w4_few<float>(const W4Call &, cudaStream_t);
template int launch_w4_few<bf16>(const W4Call &, cudaStream_t);

}  // namespace orion
