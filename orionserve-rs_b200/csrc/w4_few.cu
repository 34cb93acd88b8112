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
// slabs of 128 k filled by cp.async (no waits on barriers); scales are loaded as many slabs ahead into registers and come to their lanes by shuffles. Sums of k
// groups meet in shared memory, and where the rows of weights give too few CTAs the k of a tile is dealt to the CTAs of a cluster, whose sums meet over
// distributed shared memory: in both places in a fixed order, so results do not vary from run to run, and no workspace is needed.
#include "kernels.h"
#include "mma.cuh"
#include "w4.cuh"

#include <algorithm>

namespace orion {
namespace {

constexpr uint32_t kThreads = 256, kWarps = 8, kSlab = 128, kStages = 4;
constexpr uint32_t kWRow = kSlab / 2;  // bytes of a weight row in a slab
constexpr float kUnit = 8192.f;        // dequantised codes are multiples of 1 / kUnit

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool some) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(some ? 16u : 0u) : "memory");
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
  static constexpr uint32_t kOutputs = GATED ? kTileRows / 2 : kTileRows;   // columns of y
  static constexpr uint32_t kTokens = 8 * NT;
  static constexpr uint32_t kXRow = kSlab * sizeof(T);
  static constexpr uint32_t kWStage = kTileRows * kWRow;
  static constexpr uint32_t kSums = kKGroups * kTokens * kTileRows * 4;     // bytes of the sums that meet in shared memory
  static uint32_t smem(uint32_t tokens) { return std::max(kKGroups * kStages * (kWStage + tokens * kXRow), kSums); }
};

template <typename T, bool GATED, uint32_t GROUP, uint32_t RT, uint32_t NT, uint32_t WR>
__global__ void __launch_bounds__(kThreads)
w4_few_kernel(const W4Call c, const uint32_t tiles_m, const uint32_t stored_tokens) {
  using Cfg = FewConfig<T, GATED, GROUP, RT, NT, WR>;
  constexpr bool kF32 = sizeof(T) == 4;
  constexpr uint32_t kPerSlab = kSlab / GROUP;                    // groups in a slab
  constexpr uint32_t kScales = RT * kPerSlab, kScaleRegs = (kScales + 1) / 2;  // sets of 16 scales per slab; two sets fill a register of a warp
  extern __shared__ __align__(128) uint8_t smem[];
  pdl_trigger();

  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t kg = warp / WR, wr = warp % WR, in_kg = wr * 32 + lane;
  const uint32_t n0 = blockIdx.x / tiles_m * Cfg::kOutputs, m0 = blockIdx.x % tiles_m * Cfg::kTokens;
  const uint32_t tokens = min(Cfg::kTokens, c.rows - m0);
  const uint32_t slabs = (c.k + kSlab - 1) / kSlab, units = Cfg::kKGroups * gridDim.z, unit = blockIdx.z * Cfg::kKGroups + kg;
  const uint32_t mine = unit < slabs ? (slabs - unit + units - 1) / units : 0;
  const uint32_t groups = c.k / GROUP;

  // First row of a tile of 16 in its matrix; with a gate the first half of a warp's tiles are the gate's.
  auto row_of = [&](uint32_t rt) {
    return GATED ? n0 + (wr * (RT / 2) + rt % (RT / 2 ? RT / 2 : 1)) * 16 : n0 + (wr * RT + rt) * 16;
  };
  auto is_up = [&](uint32_t rt) { return GATED && rt >= RT / 2; };

  const uint32_t stage_bytes = Cfg::kWStage + stored_tokens * Cfg::kXRow;
  const uint32_t ring = smem_u32(smem) + kg * kStages * stage_bytes;
  pdl_wait();

  // A slab of this k group, by its WR warps: weight rows of 64 bytes, 16-byte pieces permuted by (row / 2) & 3 so that the eight rows of a fragment lie in
  // different banks; token rows likewise, neighbouring rows half a line apart.
  auto load = [&](uint32_t stage, uint32_t index) {
    if (index < mine) {
      const uint32_t k0 = (unit + index * units) * kSlab, base = ring + stage * stage_bytes;
#pragma unroll
      for (uint32_t i = 0; i < 2 * RT; ++i) {  // eight of a tile's 16 rows at a time; the warp that reads them loads them
        const uint32_t rt = i >> 1, r = (i & 1) * 8 + g, piece = t, row = row_of(rt) + r;
        const uint32_t at = (wr * RT + rt) * 16 + r;
        const bool some = row < c.n && k0 + piece * 32 < c.k;
        const uint32_t *from = is_up(rt) ? c.up.packed : c.w.packed;
        cp_async16(base + at * kWRow + (piece ^ ((at >> 1) & 3)) * 16, some ? from + (uint64_t)row * (c.k / 8) + k0 / 8 + piece * 4 : from, some);
      }
      constexpr uint32_t kPieces = Cfg::kXRow / 16, kPer = 16 / sizeof(T);
      for (uint32_t i = in_kg; i < stored_tokens * kPieces; i += WR * 32) {
        const uint32_t row = i / kPieces, piece = i % kPieces;
        const bool some = row < tokens && k0 + piece * kPer < c.k;
        const T *x = static_cast<const T *>(c.x);
        cp_async16(base + Cfg::kWStage + row * Cfg::kXRow + (piece ^ ((row & 1) << 2)) * 16, some ? x + (uint64_t)(m0 + row) * c.ldx + k0 + piece * kPer : x, some);
      }
    }
    cp_async_commit();
  };
  // scale (lower half) and zero point (upper half) of set 2 j + lane / 16, row lane % 16 of its tile
  auto load_scales = [&](uint32_t index, uint32_t (&s)[kScaleRegs]) {
#pragma unroll
    for (uint32_t j = 0; j < kScaleRegs; ++j) {
      const uint32_t set = 2 * j + (lane >> 4), rt = set / kPerSlab;
      const uint32_t group = (unit + index * units) * kPerSlab + set % kPerSlab, row = row_of(rt) + (lane & 15);
      uint32_t v = 8u << 16;
      if (index < mine && set < kScales && group < groups && row < c.n) {
        const W4View &w = is_up(rt) ? c.up : c.w;
        const uint64_t at = (uint64_t)group * c.n + row;
        const uint32_t scale = __ldg(reinterpret_cast<const uint16_t *>(w.scales) + at);
        v = w.zeros ? scale | (uint32_t)__ldg(w.zeros + at) << 16 : scale | v;
      }
      s[j] = v;
    }
  };

  float sum[RT][NT][4];
#pragma unroll
  for (uint32_t rt = 0; rt < RT; ++rt)
#pragma unroll
    for (uint32_t nt = 0; nt < NT; ++nt)
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) sum[rt][nt][i] = 0.f;

  uint32_t scales[kStages][kScaleRegs];
#pragma unroll
  for (uint32_t s = 0; s + 1 < kStages; ++s) {
    load(s, s);
    load_scales(s, scales[s]);
  }
  for (uint32_t i0 = 0; i0 < mine; i0 += kStages) {
#pragma unroll
    for (uint32_t s = 0; s < kStages; ++s) {
      const uint32_t index = i0 + s;
      if (index >= mine) break;
      cp_async_wait<kStages - 2>();
      if constexpr (WR == 1) __syncwarp();
      else asm volatile("bar.sync %0, %1;" ::"r"(kg + 1), "r"(WR * 32) : "memory");
      load((s + kStages - 1) % kStages, index + kStages - 1);
      load_scales(index + kStages - 1, scales[(s + kStages - 1) % kStages]);

      const uint32_t w_at = ring + s * stage_bytes, x_at = w_at + Cfg::kWStage;
      float part[RT][NT][4];
      uint32_t minus_zero[RT][2];
      float scale[RT][2];
#pragma unroll
      for (uint32_t q = 0; q < kSlab / 32; ++q) {  // 32 k: one 16-byte piece of a weight row
        if (q * 32 % GROUP == 0) {  // a group begins
#pragma unroll
          for (uint32_t rt = 0; rt < RT; ++rt) {
            const uint32_t set = rt * kPerSlab + q * 32 / GROUP;
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h) {
              const uint32_t v = __shfl_sync(0xffffffffu, scales[s][set >> 1], (set & 1) * 16 + h * 8 + g);
              scale[rt][h] = __uint_as_float(v << 16) * kUnit;
              const float z = -(float)(v >> 16) / kUnit;  // at most four bits: exact in bf16
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
  }

  // The k groups' sums, [k group][token][row], over the rings
  cp_async_wait<0>();
  __syncthreads();
  float *sums = reinterpret_cast<float *>(smem);
#pragma unroll
  for (uint32_t rt = 0; rt < RT; ++rt)
#pragma unroll
    for (uint32_t nt = 0; nt < NT; ++nt)
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i)
        sums[(kg * Cfg::kTokens + nt * 8 + t * 2 + (i & 1)) * Cfg::kTileRows + (wr * RT + rt) * 16 + (i >> 1) * 8 + g] = sum[rt][nt][i];
  const uint32_t ranks = gridDim.z, rank = blockIdx.z;
  if (ranks > 1) {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  } else {
    __syncthreads();
  }
  auto total = [&](uint32_t token, uint32_t row) {
    float v = 0.f;
    for (uint32_t r = 0; r < ranks; ++r) {
#pragma unroll
      for (uint32_t j = 0; j < Cfg::kKGroups; ++j) {
        const float *p = sums + (j * Cfg::kTokens + token) * Cfg::kTileRows + row;
        if (ranks == 1) {
          v += *p;
        } else {
          uint32_t remote;
          float f;
          asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(p)), "r"(r));
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f) : "r"(remote) : "memory");
          v += f;
        }
      }
    }
    return v;
  };
  for (uint32_t i = rank * kThreads + threadIdx.x; i < tokens * Cfg::kOutputs; i += ranks * kThreads) {
    const uint32_t token = i / Cfg::kOutputs, col = i % Cfg::kOutputs;
    if (n0 + col >= c.n) continue;
    float y;
    if constexpr (GATED) {
      constexpr uint32_t kHalf = RT / 2 * 16;
      const uint32_t at = col / kHalf * (2 * kHalf) + col % kHalf;
      y = gated<T>(GatedAct{c.act, 0.f}, total(token, at), total(token, at + kHalf));
    } else {
      y = total(token, col) + (c.bias ? c.bias[n0 + col] : 0.f);
    }
    static_cast<T *>(c.out)[(uint64_t)(m0 + token) * c.ldo + n0 + col] = from_f32<T>(y);
  }
  if (ranks > 1) {  // nobody leaves while its sums are being read
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
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
  // k over a cluster while that gives an SM more CTAs than it holds now and every k group keeps two slabs
  const uint32_t per_sm = std::max(1u, std::min(4u, 227u * 1024u / (smem + 1024u)));
  const uint32_t slabs = (c.k + kSlab - 1) / kSlab;
  uint32_t ranks = 1;
  while (ranks < 8 && tiles * ranks * 2 <= 148ull * per_sm && slabs >= Cfg::kKGroups * ranks * 4) ranks *= 2;
  ORION_CUDA_CHECK("4-bit product", launch_pdl_cluster(kernel, dim3((uint32_t)tiles, 1, ranks), dim3(kThreads), dim3(1, 1, ranks), smem, stream, c, tiles_m, stored));
  count_launch();
  return ORION_OK;
}

template <typename T, bool GATED, uint32_t GROUP>
int launch_shape(const W4Call &c, cudaStream_t stream) {
  if (c.rows <= 8) return launch_config<T, GATED, GROUP, 2, 1, 1>(c, stream);
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
