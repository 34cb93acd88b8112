// Products with 4-bit weights for few rows, and for f32 activations of any number of rows (w4.cuh has the layout):
//   y = x W^T + bias,  or  y = act(x W^T) * (x up^T) with both products, the activation and the multiplication in this one kernel.
//
// Bound by the weights' way from HBM: 0.53 bytes a weight. Weights are the M operand of mma.sync (16 rows of 16 k), tokens its N. A code less its zero
// point is a whole number of at most 15, exact in bf16; so the products are exact, a group is summed in f32, and the scale multiplies that sum in f32:
// nothing is rounded but sums. Dequantisation is one AND and one fused multiply-add per PAIR of weights (plus a shift per eight): the masked pair, read
// as bf16, is code * 2^-133 or code * 2^-129 (subnormal numbers are multiples of 2^-133, and so are those of the first binade above them), and
// fma(pair, 2^120 or 2^116, -zero * 2^-13) = (code - zero) * 2^-13, exactly.
//
// f32 activations go through the same instructions as three bf16 terms of eight bits each (hi + mid + lo = x exactly), so f32 results have f32 accuracy.
//
// A CTA of eight warps: WR of them side by side over weight rows, 8 / WR groups of them over k. Few tokens: WR = 1, every warp streams k slabs of its own
// and only reads the tokens' values it needs; more tokens: warps share the tokens' slab, so that L2 delivers it less often. Each k group has a ring of
// slabs of 128 k, weights, tokens and scales, filled by cp.async (no waits on barriers). CTAs stay and go from tile to tile, with the ring running ahead
// across tiles. Sums of k groups meet in shared memory, and where the rows of weights give too few CTAs the k of a tile is dealt to the CTAs of a cluster, whose sums meet over
// distributed shared memory: in both places in a fixed order, so results do not vary from run to run, and no workspace is needed.
#include "kernels.h"
#include "mma.cuh"
#include "w4.cuh"

#include <algorithm>

namespace orion {
namespace {

constexpr uint32_t kThreads = 256, kWarps = 8, kSlab = 128;
constexpr uint32_t kWRow = kSlab / 2;  // bytes of a weight row in a slab
constexpr float kUnit = 8192.f;        // dequantised codes are multiples of 1 / kUnit

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool some) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(some ? 16u : 0u) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void *src, uint32_t bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
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
// What is left of x beyond its first eight bits; nothing of an infinity.
__device__ __forceinline__ float beyond(float x, float first) { return x == first ? 0.f : x - first; }
__device__ __forceinline__ float first_bits(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }
__device__ __forceinline__ uint32_t upper_halves(float a, float b) { return __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632); }

template <typename T, bool GATED, uint32_t GROUP, uint32_t RT, uint32_t NT, uint32_t WR>
struct FewConfig {
  static constexpr uint32_t kKGroups = kWarps / WR;
  static constexpr uint32_t kTileRows = 16 * RT * WR;                       // rows of weights per CTA, gate and up together
  static constexpr uint32_t kMatrices = GATED ? 2 : 1;
  static constexpr uint32_t kOutputs = kTileRows / kMatrices;               // columns of y
  static constexpr uint32_t kTokens = 8 * NT;
  static constexpr uint32_t kXRow = kSlab * sizeof(T);
  static constexpr uint32_t kWStage = kTileRows * kWRow;
  static constexpr uint32_t kPerSlab = kSlab / GROUP;                       // groups in a slab
  // scales, and zero points, of a group and matrix: the outputs' and what stands before them in their first word
  static constexpr uint32_t kScaleRow = kOutputs * 2 + 4, kZeroRow = kOutputs + 4;
  static constexpr uint32_t kSStage = kMatrices * kPerSlab * (kScaleRow + kZeroRow);
  static constexpr uint32_t kSums = kKGroups * kTokens * kTileRows;         // floats of the sums that meet in shared memory
  // Slabs in the ring, and sets of sums: with few tokens two CTAs share an SM, with many one takes what there is.
  static constexpr uint32_t kStages = NT == 1 || (sizeof(T) == 4) ? 3 : 4, kSets = NT <= 2 ? 2 : 1;
  static uint32_t stage(uint32_t tokens) { return (kWStage + tokens * kXRow + kSStage + 15) / 16 * 16; }
  static uint32_t smem(uint32_t tokens) { return kKGroups * kStages * stage(tokens) + kSets * kSums * 4; }
};

template <typename T, bool GATED, uint32_t GROUP, uint32_t RT, uint32_t NT, uint32_t WR>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 2 : 1)
w4_few_kernel(const W4Call c, const uint32_t tiles, const uint32_t tiles_m, const uint32_t stored_tokens, const uint32_t stage_bytes) {
  using Cfg = FewConfig<T, GATED, GROUP, RT, NT, WR>;
  constexpr bool kF32 = sizeof(T) == 4;
  constexpr uint32_t kPerSlab = Cfg::kPerSlab, kStages = Cfg::kStages;
  extern __shared__ __align__(128) uint8_t smem[];
  pdl_trigger();

  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t kg = warp / WR, wr = warp % WR, in_kg = wr * 32 + lane;
  const uint32_t ranks = gridDim.z, rank = blockIdx.z;
  const uint32_t slabs = (c.k + kSlab - 1) / kSlab, units = Cfg::kKGroups * ranks, unit = rank * Cfg::kKGroups + kg;
  const uint32_t mine = unit < slabs ? (slabs - unit + units - 1) / units : 0;  // slabs of a tile that this k group takes
  const uint32_t groups = c.k / GROUP;
  const uint32_t ring = smem_u32(smem) + kg * kStages * stage_bytes;
  float *const sums = reinterpret_cast<float *>(smem + Cfg::kKGroups * kStages * stage_bytes);

  // First output of a tile of 16 rows within the CTA's; with a gate the first half of a warp's tiles are the gate's.
  constexpr uint32_t kTilesPerMatrix = RT / Cfg::kMatrices;
  auto col_of = [&](uint32_t rt) { return (wr * kTilesPerMatrix + rt % kTilesPerMatrix) * 16; };
  auto matrix_of = [&](uint32_t rt) { return rt / kTilesPerMatrix; };
  pdl_wait();

  // What is loaded next: a slab of a tile. The loads run ahead of the products across tiles, so that the ring never drains.
  uint32_t load_tile = blockIdx.x, load_index = 0, load_slot = 0;
  auto load = [&] {
    if (load_tile < tiles && mine > 0) {
      const uint32_t n0 = load_tile / tiles_m * Cfg::kOutputs, m0 = load_tile % tiles_m * Cfg::kTokens, tokens = min(Cfg::kTokens, c.rows - m0);
      const uint32_t slab = unit + load_index * units, k0 = slab * kSlab, base = ring + load_slot * stage_bytes;
      // Weight rows of 64 bytes, 16-byte pieces permuted by (row / 2) & 3 so that the eight rows of a fragment lie in different banks; eight of a
      // tile's 16 rows at a time
#pragma unroll
      for (uint32_t i = 0; i < 2 * RT; ++i) {
        const uint32_t rt = i >> 1, r = (i & 1) * 8 + g, row = n0 + col_of(rt) + r, at = (wr * RT + rt) * 16 + r;
        const bool some = row < c.n && k0 + t * 32 < c.k;
        const uint32_t *from = matrix_of(rt) ? c.up.packed : c.w.packed;
        cp_async16(base + at * kWRow + (t ^ ((at >> 1) & 3)) * 16, some ? from + (uint64_t)row * (c.k / 8) + k0 / 8 + t * 4 : from, some);
      }
      // token rows, every other one with its halves of 64 bytes exchanged
      constexpr uint32_t kPieces = Cfg::kXRow / 16, kPer = 16 / sizeof(T);
      const T *x = static_cast<const T *>(c.x);
      for (uint32_t i = in_kg; i < stored_tokens * kPieces; i += WR * 32) {
        const uint32_t row = i / kPieces, piece = i % kPieces;
        const bool some = row < tokens && k0 + piece * kPer < c.k;
        cp_async16(base + Cfg::kWStage + row * Cfg::kXRow + (piece ^ ((row & 1) << 2)) * 16, some ? x + (uint64_t)(m0 + row) * c.ldx + k0 + piece * kPer : x, some);
      }
      // scales and zero points, in words: an odd number of outputs leaves them at any place within theirs
      const uint32_t s_at = base + Cfg::kWStage + stored_tokens * Cfg::kXRow;
      constexpr uint32_t kWords = Cfg::kScaleRow / 4, kZeroWords = Cfg::kZeroRow / 4;
#pragma unroll
      for (uint32_t j = 0; j < Cfg::kMatrices * kPerSlab; ++j) {
        const W4View &w = j >= kPerSlab ? c.up : c.w;
        const uint32_t group = slab * kPerSlab + j % kPerSlab;
        const uint64_t first = (uint64_t)group * c.n + n0, scales = (uint64_t)groups * c.n;
        for (uint32_t i = in_kg; i < kWords; i += WR * 32) {
          const uint64_t at = (first & ~1ull) + 2 * i;
          const uint32_t left = group < groups && at < scales ? (uint32_t)min(scales - at, (uint64_t)2) * 2 : 0;
          cp_async4(s_at + j * Cfg::kScaleRow + i * 4, left ? w.scales + at : w.scales, left);
        }
        if (w.zeros) {
          for (uint32_t i = in_kg; i < kZeroWords; i += WR * 32) {
            const uint64_t at = (first & ~3ull) + 4 * i;
            const uint32_t left = group < groups && at < scales ? (uint32_t)min(scales - at, (uint64_t)4) : 0;
            cp_async4(s_at + Cfg::kMatrices * kPerSlab * Cfg::kScaleRow + j * Cfg::kZeroRow + i * 4, left ? w.zeros + at : w.zeros, left);
          }
        }
      }
      if (++load_index == mine) load_index = 0, load_tile += gridDim.x;
      load_slot = load_slot + 1 == kStages ? 0 : load_slot + 1;
    }
    cp_async_commit();
  };
#pragma unroll
  for (uint32_t s = 0; s + 1 < kStages; ++s) load();

  uint32_t slot = 0, turn = 0;
  for (uint32_t tile = blockIdx.x; tile < tiles; tile += gridDim.x, turn ^= Cfg::kSets - 1) {
    const uint32_t n0 = tile / tiles_m * Cfg::kOutputs, m0 = tile % tiles_m * Cfg::kTokens, tokens = min(Cfg::kTokens, c.rows - m0);
    float sum[RT][NT][4];
#pragma unroll
    for (uint32_t rt = 0; rt < RT; ++rt)
#pragma unroll
      for (uint32_t nt = 0; nt < NT; ++nt)
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) sum[rt][nt][i] = 0.f;

    for (uint32_t index = 0; index < mine; ++index) {
      cp_async_wait<kStages - 2>();
      if constexpr (WR == 1) __syncwarp();
      else if constexpr (WR == kWarps) __syncthreads();
      else asm volatile("bar.sync %0, %1;" ::"r"(kg + 1), "n"(WR * 32) : "memory");
      load();

      const uint32_t w_at = ring + slot * stage_bytes, x_at = w_at + Cfg::kWStage, s_at = x_at + stored_tokens * Cfg::kXRow;
      const uint32_t z_at = s_at + Cfg::kMatrices * kPerSlab * Cfg::kScaleRow;
      slot = slot + 1 == kStages ? 0 : slot + 1;
      float part[RT][NT][4];
      uint32_t minus_zero[RT][2];
      float scale[RT][2];
#pragma unroll
      for (uint32_t q = 0; q < kSlab / 32; ++q) {  // 32 k: one 16-byte piece of a weight row
        if (q * 32 % GROUP == 0) {  // a group begins
          const uint32_t first = ((unit + index * units) * kPerSlab + q * 32 / GROUP) * c.n + n0;  // its place within words: the low bits
#pragma unroll
          for (uint32_t rt = 0; rt < RT; ++rt) {
            const uint32_t j = matrix_of(rt) * kPerSlab + q * 32 / GROUP;
            const bool zeros = (matrix_of(rt) ? c.up : c.w).zeros != nullptr;
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h) {
              const uint32_t at = col_of(rt) + h * 8 + g;
              scale[rt][h] = __uint_as_float(lds16(s_at + j * Cfg::kScaleRow + ((first & 1) + at) * 2) << 16) * kUnit;
              float z = -8.f / kUnit;
              if (zeros) z = -(float)lds8(z_at + j * Cfg::kZeroRow + (first & 3) + at) / kUnit;  // eight bits at most: exact in bf16
              minus_zero[rt][h] = upper_halves(z, z);
            }
#pragma unroll
            for (uint32_t nt = 0; nt < NT; ++nt)
#pragma unroll
              for (uint32_t i = 0; i < 4; ++i) part[rt][nt][i] = 0.f;
          }
        }
        uint32_t a[RT][2][4];  // [rows 0-7 / 8-15][pair]
#pragma unroll
        for (uint32_t rt = 0; rt < RT; ++rt)
#pragma unroll
          for (uint32_t h = 0; h < 2; ++h) {
            const uint32_t at = (wr * RT + rt) * 16 + h * 8 + g;
            dequant(lds32(w_at + at * kWRow + (q ^ ((at >> 1) & 3)) * 16 + t * 4), minus_zero[rt][h], a[rt][h]);
          }
#pragma unroll
        for (uint32_t nt = 0; nt < NT; ++nt) {
          const uint32_t row = nt * 8 + g;
          auto multiply = [&](const uint32_t (&b)[4]) {
#pragma unroll
            for (uint32_t rt = 0; rt < RT; ++rt)
#pragma unroll
              for (uint32_t half = 0; half < 2; ++half) {
                const uint32_t frag[4] = {a[rt][0][2 * half], a[rt][1][2 * half], a[rt][0][2 * half + 1], a[rt][1][2 * half + 1]};
                mma_bf16_16816(part[rt][nt], frag, b[2 * half], b[2 * half + 1]);
              }
          };
          if constexpr (kF32) {
            float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (row < stored_tokens) {
#pragma unroll
              for (uint32_t i = 0; i < 2; ++i) {
                const uint4 r = lds128(x_at + row * Cfg::kXRow + ((q * 8 + t * 2 + i) ^ ((row & 1) << 2)) * 16);
                v[4 * i] = __uint_as_float(r.x), v[4 * i + 1] = __uint_as_float(r.y), v[4 * i + 2] = __uint_as_float(r.z), v[4 * i + 3] = __uint_as_float(r.w);
              }
            }
#pragma unroll
            for (uint32_t term = 0; term < 3; ++term) {
              uint32_t b[4];
#pragma unroll
              for (uint32_t i = 0; i < 4; ++i) {
                b[i] = upper_halves(v[2 * i], v[2 * i + 1]);
                v[2 * i] = beyond(v[2 * i], first_bits(v[2 * i]));
                v[2 * i + 1] = beyond(v[2 * i + 1], first_bits(v[2 * i + 1]));
              }
              multiply(b);
            }
          } else {
            uint4 r = make_uint4(0, 0, 0, 0);
            if (row < stored_tokens) r = lds128(x_at + row * Cfg::kXRow + ((q * 4 + t) ^ ((row & 1) << 2)) * 16);
            const uint32_t b[4] = {r.x, r.y, r.z, r.w};
            multiply(b);
          }
        }
        if ((q + 1) * 32 % GROUP == 0) {  // a group ends
#pragma unroll
          for (uint32_t rt = 0; rt < RT; ++rt)
#pragma unroll
            for (uint32_t nt = 0; nt < NT; ++nt)
#pragma unroll
              for (uint32_t i = 0; i < 4; ++i) sum[rt][nt][i] = fmaf(part[rt][nt][i], scale[rt][i >> 1], sum[rt][nt][i]);
        }
      }
    }

    // The k groups' sums, [k group][token][row]. Where two sets take turns one barrier a tile is enough.
    if (Cfg::kSets == 1 && tile != blockIdx.x) {
      if (ranks > 1) cluster_barrier();
      else __syncthreads();
    }
    float *const mine_at = sums + turn * Cfg::kSums;
#pragma unroll
    for (uint32_t rt = 0; rt < RT; ++rt)
#pragma unroll
      for (uint32_t nt = 0; nt < NT; ++nt)
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
          const uint32_t token = nt * 8 + t * 2 + (i & 1);
          if (token < stored_tokens) mine_at[(kg * Cfg::kTokens + token) * Cfg::kTileRows + (wr * RT + rt) * 16 + (i >> 1) * 8 + g] = sum[rt][nt][i];
        }
    if (ranks > 1) cluster_barrier();
    else __syncthreads();
    auto total = [&](uint32_t token, uint32_t row) {
      float v = 0.f;
      for (uint32_t r = 0; r < ranks; ++r) {
#pragma unroll
        for (uint32_t j = 0; j < Cfg::kKGroups; ++j) {
          const float *p = mine_at + (j * Cfg::kTokens + token) * Cfg::kTileRows + row;
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
  }
  cp_async_wait<0>();
  if (ranks > 1) cluster_barrier();  // nobody leaves while its sums are being read
}

template <typename T, bool GATED, uint32_t GROUP, uint32_t RT, uint32_t NT, uint32_t WR>
int launch_config(const W4Call &c, cudaStream_t stream) {
  using Cfg = FewConfig<T, GATED, GROUP, RT, NT, WR>;
  static bool done[kMaxDeviceOrdinals] = {};
  const auto kernel = w4_few_kernel<T, GATED, GROUP, RT, NT, WR>;
  ORION_CUDA_CHECK("4-bit product", ensure_dynamic_smem(kernel, (int)Cfg::smem(Cfg::kTokens), done));
  const uint32_t tiles_n = (c.n + Cfg::kOutputs - 1) / Cfg::kOutputs, tiles_m = (c.rows + Cfg::kTokens - 1) / Cfg::kTokens;
  const uint32_t stored = std::min(c.rows, Cfg::kTokens), smem = Cfg::smem(stored);
  const uint64_t tiles = (uint64_t)tiles_n * tiles_m;
  if (tiles > 0x7fffffffull) return set_error(ORION_ERR_INVALID_REQUEST, "4-bit product: %u rows x %u outputs are too many for one call", c.rows, c.n);
  // k over a cluster while the tiles leave SMs without work and every k group keeps two slabs
  const uint32_t resident = 148 * (NT == 1 && smem + 1024 <= 114 * 1024 ? 2 : 1), slabs = (c.k + kSlab - 1) / kSlab;
  uint32_t ranks = 1;
  while (ranks < 8 && tiles * ranks * 2 <= resident && slabs >= Cfg::kKGroups * ranks * 4) ranks *= 2;
  const uint32_t ctas = (uint32_t)std::min<uint64_t>(tiles, resident);
  ORION_CUDA_CHECK("4-bit product", launch_pdl_cluster(kernel, dim3(ctas, 1, ranks), dim3(kThreads), dim3(1, 1, ranks), smem, stream, c, (uint32_t)tiles, tiles_m,
                                                       stored, Cfg::stage(stored)));
  count_launch();
  return ORION_OK;
}

template <typename T, bool GATED, uint32_t GROUP>
int launch_shape(const W4Call &c, cudaStream_t stream) {
  if (c.rows <= 8) return launch_config<T, GATED, GROUP, 2, 1, 2>(c, stream);
  if (c.rows <= 16) return launch_config<T, GATED, GROUP, 2, 2, 2>(c, stream);
  if constexpr (sizeof(T) == 2) {
    if (c.rows > 32) return launch_config<T, GATED, GROUP, 2, 8, 8>(c, stream);
  }
  return launch_config<T, GATED, GROUP, 2, 4, 4>(c, stream);
}

template <typename T, bool GATED>
int launch_group(const W4Call &c, cudaStream_t stream) {
  switch (c.group) {
    case 32: return launch_shape<T, GATED, 32>(c, stream);
    case 64: return launch_shape<T, GATED, 64>(c, stream);
    default: return launch_shape<T, GATED, 128>(c, stream);
  }
}

}  // namespace

template <typename T>
int launch_w4_few(const W4Call &c, cudaStream_t stream) {
  return c.up.packed ? launch_group<T, true>(c, stream) : launch_group<T, false>(c, stream);
}
template int launch_w4_few<float>(const W4Call &, cudaStream_t);
template int launch_w4_few<bf16>(const W4Call &, cudaStream_t);

}  // namespace orion
