// Products with 4-bit weights for many rows of bf16 activations (w4.cuh has the layout): persistent CTA pairs on tcgen05, weights dequantised on their way
// into shared memory.
//
// From some 20 rows on the tensor cores of mma.sync are the bound, from some 100 those of tcgen05: 4096 rows of k 4096 with a gate to 14336 take 751 us, 1.3
// PFLOP/s (0.92 of a library product's rate at the power limit); 64 rows of k 3584 with a gate to 18944 35 us, of which the weights' way from HBM is 12 and the first
// kernel, which is not hidden, some 7. A pair of CTAs works as one MMA unit on 256 weight rows x
// up to 256 tokens, as for 16-bit weights (gemm_pair.cuh), but its weights come as codes: teams of warps read them into
// registers, a round of stages ahead, and write the operand tiles of a CTA's 128 rows into the 128-byte-swizzled ring, so HBM delivers half a byte a weight.
//
// The operands are f16, not bf16. (code - zero) * scale has at most 11 significant bits with a zero of 8 and 12 with any other, f16 holds 11: products are
// exact, or off by 2^-12 of a weight, where bf16 would round every weight by 2^-9. For f16's range both sides are scaled by powers of two, every row of
// weights by the exponent of its largest scale and every token by that of its largest value: weights keep their bits where their scale is above 2^-21 of the
// row's largest, tokens down to 2^-30 of the largest value; what is smaller is off by at most 2^-29 of that scale, 2^-38 of that value. A first kernel
// finds these exponents and converts the tokens; the epilogue scales back. Dequantisation costs a lane 13 instructions for eight weights: the masked pairs, read as f16, are code * 2^-24
// or code * 2^-20 (subnormal numbers and the first binade count in steps of 2^-24), one fused multiply-add subtracts the zero point, which is exact, and one
// multiplication applies the scale.
//
// Where tiles are too few for the device, k is cut as well: the parts are summed in order, of single CTAs over the distributed shared memory of a cluster, of
// pairs by a third kernel, so results do not vary.
//
// Warp 0 loads tokens, 1 of the leader issues the MMAs, then come the dequantising warps, eight of the epilogue, which works under the next tile's main loop.
// Every wait is bounded; one that runs out sets the projections' error word.
#include "gemm_pair.cuh"
#include "w4.cuh"

#include <cuda_fp16.h>

#include <algorithm>

namespace orion {
namespace {

using Pair = PairConfig;
constexpr uint32_t kDequantWarps = 4, kFirstDequant = 2;             // warps that make a stage's weights; as many such teams as the rings have stages

// CTAS: 1 or 2 that work as an MMA unit on 128 weight rows each; TOKENS: rows of x in a stage of a CTA (a pair's CTAs hold half of a tile's each).
//
// Where the accumulators leave room (single CTAs), the weights of a stage go to tensor memory, 64 columns of it: through shared memory they would cost it 64
// KiB of traffic a stage, 512 cycles, where HBM brings the codes in some 360. Shared memory then holds codes instead, two stages for each team.
template <uint32_t CTAS, uint32_t TOKENS, uint32_t STAGE_K, uint32_t STAGES>
struct Form {
  static constexpr uint32_t kCtas = CTAS, kStages = STAGES, kTeams = STAGES, kStageK = STAGE_K, kTileRows = CTAS * Pair::kRows, kAccCols = CTAS * TOKENS;
  static constexpr bool kWeightsInTmem = CTAS == 1;
  static constexpr uint32_t kTmemStage = STAGE_K / 2, kTmemWeights = 2 * kAccCols;  // columns
  static constexpr uint32_t kCodeStages = kWeightsInTmem ? 2 * STAGES : 1, kCodeRow = STAGE_K / 2, kCodeBytes = kWeightsInTmem ? Pair::kRows * kCodeRow : 0;
  static constexpr uint32_t kSlabs = STAGE_K / Pair::kSlabK, kXSlab = TOKENS * Pair::kSlabK * 2, kXBytes = kSlabs * kXSlab, kXRing = kWeightsInTmem ? 0 : STAGES * Pair::kWBytes;
  static constexpr uint32_t kCodeRing = kXRing + STAGES * kXBytes, kBarriers = kCodeRing + kCodeStages * kCodeBytes;
  static constexpr int kSmemBytes = kBarriers + 1024 /*align*/ + 512 /*barriers*/;
  static constexpr uint32_t kFirstEpilogue = kFirstDequant + STAGES * kDequantWarps, kCodesWarp = kFirstEpilogue + Pair::kEpilogueWarps;
  static constexpr uint32_t kWarps = kCodesWarp + (kWeightsInTmem ? 1 : 0);
  static_assert(kTeams <= STAGES, "a team could wait for a barrier that is two phases behind, and two phases are one to a wait");
  static_assert(STAGE_K == 128 || kWeightsInTmem, "the pairs' stages of weights");
  static_assert(kSmemBytes <= 232448, "rings exceed the shared memory of an SM");
  static_assert(kTmemWeights + (kWeightsInTmem ? STAGES * kTmemStage : 0) <= Pair::kTmemCols, "weights and accumulators exceed tensor memory");
};
// Up to 64 tokens a stage's MMAs take a quarter of what its hand-overs do, and it holds 256 k (64 rows of k 14336 to 18944 outputs: 53 us with 128 k).
using Single64 = Form<1, 64, 256, 3>;
using Single128 = Form<1, 128, 128, 4>;
using Paired = Form<2, 128, 128, 3>;
constexpr uint32_t kWordBytes = 4;       // by which a pair's second CTA tells of its weights
constexpr uint32_t kSms = 2 * kPairs;
constexpr int kTop = 14;                 // exponent that the largest scale of a row, and the largest value of a token, are brought to, or one less

// What the first kernel leaves for the second, and the parts of k that the third one sums.
struct Workspace {
  __half *x = nullptr;        // [rows][k], scaled
  // Square roots of what the epilogue multiplies a sum by: it does so with (row's x token's), twice. Both are at most 1 or both at least 1, so what is infinite
  // or loses bits on the way would in the end; in other orders a scale of 2^124 and tokens of 2^-110 passed through infinities, and 2^-120 and 2^118 through
  // subnormal numbers. So these powers of two are squares of others: rows and tokens are brought to within a factor of four instead of two.
  float *x_unit = nullptr;    // [rows, rounded up to 32] of what a token was divided by, but for 2^kTop
  // Weight rows as tiles hold them: with a gate its rows and the other matrix's in turn. Rounded up to whole tiles.
  float *w_unit = nullptr;    // [weight rows] likewise, with the powers that scales (2^14), codes (2^-9) and tokens (2^14) are brought to
  uint32_t *params = nullptr; // [k / group][weight rows] scale, in f16 and with the largest at 2^(kTop - 1) .. 2^(kTop + 1), | zero << 16
  float *parts = nullptr;     // [splits][rows][weight rows]
};

struct Plan {
  uint32_t tokens = 256, splits = 1, tiles_w = 0, tiles_x = 0, stages = 0;
  uint32_t ctas = 2;  // of an MMA unit
};

// Up to 128 tokens single CTAs, beyond them pairs. Tiles and parts of k so that the rounds of the units, times what a round takes, are least, in cycles: a
// stage takes the tensor cores four cycles a token column and the dequantising warps some 450, a tile's end some 3000. Parts of k: of single CTAs they meet in a
// cluster, all parts of a launch at once; of pairs they are written and read again.
Plan make_plan(uint32_t rows, uint32_t weight_rows, uint32_t k) {
  // CTAs of one to an SM that are at work together in clusters of so many, with the SMs of a GPC that are left over (36 clusters of four took two turns, 22 us
  // instead of 12 for 32 of them; 16 of seven 31, 16 of six 20)
  constexpr uint32_t kClustered[9] = {0, 148, 144, 132, 128, 120, 126, 105, 112};
  Plan best;
  double cost = 1e300;
  const uint32_t ctas = rows <= Single128::kAccCols ? 1 : 2, units = kSms / ctas;
  const uint32_t stage_k = rows <= Single64::kAccCols ? Single64::kStageK : ctas == 1 ? Single128::kStageK : Paired::kStageK;
  const uint32_t stages = (k + stage_k - 1) / stage_k, tiles_w = (weight_rows + ctas * Pair::kRows - 1) / (ctas * Pair::kRows);
  const uint32_t most = std::min(256u, (rows + 31) / 32 * 32);
  for (uint32_t tokens = most; tokens >= std::min(most, 128u); tokens -= 32) {
    const uint32_t tiles_x = (rows + tokens - 1) / tokens;
    for (uint32_t splits = 1; splits <= 8 && splits <= stages; ++splits) {
      const uint64_t tiles = (uint64_t)tiles_w * tiles_x;
      if (splits > 1 && (ctas == 1 ? tiles * splits > kClustered[splits] : tiles > 8 * units)) continue;
      const uint64_t jobs = (uint64_t)tiles_w * tiles_x * splits, rounds = (jobs + units - 1) / units;
      double c = (double)rounds * ((stages + splits - 1) / splits * std::max(4.0 * tokens, 450.0) * (stage_k / 128) + 3000.0);
      if (splits > 1) c += ctas == 1 ? 2000.0 : 4000.0 + (double)splits * rows * weight_rows * 8.0 / 2500.0;
      if (c < cost) cost = c, best = {tokens, splits, tiles_w, tiles_x, stages, ctas};
    }
  }
  return best;
}

constexpr uint32_t kParamRows = 2 * Pair::kRows;
uint64_t padded_rows(uint32_t weight_rows) { return ((uint64_t)weight_rows + kParamRows - 1) / kParamRows * kParamRows; }
uint64_t place(uint64_t *at, uint64_t bytes) {
  const uint64_t here = *at;
  *at += (bytes + 255) / 256 * 256;
  return here;
}
Workspace workspace_at(uint8_t *base, uint32_t rows, uint32_t weight_rows, uint32_t k, uint32_t group, const Plan &plan, uint64_t *bytes) {
  uint64_t at = 0;
  Workspace w;
  w.x = reinterpret_cast<__half *>(base + place(&at, (uint64_t)rows * k * 2));
  w.x_unit = reinterpret_cast<float *>(base + place(&at, ((uint64_t)rows + 31) / 32 * 32 * 4));
  w.w_unit = reinterpret_cast<float *>(base + place(&at, padded_rows(weight_rows) * 4));
  w.params = reinterpret_cast<uint32_t *>(base + place(&at, padded_rows(weight_rows) * (k / group) * 4));
  w.parts = reinterpret_cast<float *>(base + place(&at, plan.ctas == 2 && plan.splits > 1 ? (uint64_t)plan.splits * rows * weight_rows * 4 : 0));
  *bytes = at;
  return w;
}

// ---- first kernel: tokens to f16, exponents of tokens and of weight rows ------------------------

constexpr uint32_t kPrepThreads = 256, kPrepWarps = kPrepThreads / 32;

__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -126 <= e <= 127

// 32 weight rows, their groups dealt to eight warps; eight groups of a thread's are on their way together.
__device__ __forceinline__ void prepare_weights(const W4Call &c, const Workspace &ws, uint32_t matrices, uint32_t param_rows, uint32_t block) {
  constexpr uint32_t kAtOnce = 8;
  __shared__ uint32_t tops[kPrepWarps][32];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = block * 32 + lane, row = r / matrices, groups = c.k / c.group;
  const W4View &w = r % matrices ? c.up : c.w;
  const bool there = row < c.n, zeros = there && w.zeros;
  uint32_t scale[kAtOnce], zero[kAtOnce], top = 0;
  auto load = [&](uint32_t first) {
#pragma unroll
    for (uint32_t j = 0; j < kAtOnce; ++j) {
      const uint32_t g = first + j * kPrepWarps;
      const uint64_t at = (uint64_t)g * c.n + row;
      scale[j] = there && g < groups ? (uint32_t)__ldg(reinterpret_cast<const uint16_t *>(w.scales) + at) : 0u;
      zero[j] = 8;
      if (zeros && g < groups) zero[j] = __ldg(w.zeros + at);
    }
  };
  for (uint32_t first = warp; first < groups; first += kAtOnce * kPrepWarps) {
    load(first);
#pragma unroll
    for (uint32_t j = 0; j < kAtOnce; ++j) {
      const uint32_t e = scale[j] >> 7 & 255u;
      top = max(top, e == 255u ? 0u : e);
    }
  }
  tops[warp][lane] = top;
  __syncthreads();
#pragma unroll
  for (uint32_t i = 0; i < kPrepWarps; ++i) top = max(top, tops[i][lane]);
  top += top & 1;  // an odd power of two (its field in a float, 127 more, is even): with the 2^19 that the epilogue takes off too, a square
  const int32_t raise = top ? kTop + 127 - (int32_t)top : 0;
  for (uint32_t first = warp; first < groups; first += kAtOnce * kPrepWarps) {
    if (groups > kAtOnce * kPrepWarps) load(first);  // else they are still there
#pragma unroll
    for (uint32_t j = 0; j < kAtOnce; ++j) {
      const uint32_t g = first + j * kPrepWarps, p = scale[j], e = p >> 7 & 255u;
      // infinities and NaN stay; 0 (whose exponent field would count as a power of two where the row's largest scale is small) and what is far below the row's
      // largest scale vanish
      const uint32_t f = e == 255u ? p << 16 : e == 0u || (int32_t)e + raise <= 127 - 30 ? 0u : (p << 16) + ((uint32_t)raise << 23);
      if (g < groups) ws.params[(uint64_t)g * param_rows + r] = (uint32_t)__half_as_ushort(__float2half_rn(__uint_as_float(f))) | zero[j] << 16;
    }
  }
  if (warp == 0) ws.w_unit[r] = top ? power_of_two(((int)top - 127 - 19) / 2) : 1.f;
}

// A token, by THREADS threads (a block or a warp), HELD pieces of eight values each in registers.
template <uint32_t THREADS, uint32_t HELD>
__device__ __forceinline__ void prepare_token(const W4Call &c, const Workspace &ws, uint32_t m) {
  const uint32_t thread = threadIdx.x % THREADS, pieces = c.k / 8;
  const uint4 *x = reinterpret_cast<const uint4 *>(static_cast<const bf16 *>(c.x) + (uint64_t)m * c.ldx);
  uint4 held[HELD];
  uint32_t top = 0;  // the largest finite magnitude's bits
  auto load = [&](uint32_t first) {
#pragma unroll
    for (uint32_t j = 0; j < HELD; ++j) held[j] = first + j * THREADS < pieces ? __ldg(x + first + j * THREADS) : make_uint4(0, 0, 0, 0);
  };
  for (uint32_t first = thread; first < pieces; first += HELD * THREADS) {
    load(first);
#pragma unroll
    for (uint32_t j = 0; j < HELD; ++j) {
      const uint32_t u[4] = {held[j].x, held[j].y, held[j].z, held[j].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t lo = u[i] & 0x7fffu, hi = u[i] >> 16 & 0x7fffu;
        top = max(top, max(lo < 0x7f80u ? lo : 0u, hi < 0x7f80u ? hi : 0u));
      }
    }
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if constexpr (THREADS > 32) {
    __shared__ uint32_t tops[kPrepWarps];
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < kPrepWarps; ++i) top = max(top, tops[i]);
  }
  int e = top == 0 ? 0 : top >= 0x80u ? (int)(top >> 7) - 127 : 31 - __clz((int)top) - 133;
  e += e & 1;
  const int up = kTop - e, half = up / 2;
  // two factors: one alone would not be finite where the token's values are the smallest there are
  const float f0 = power_of_two(half), f1 = power_of_two(up - half);
  uint4 *out = reinterpret_cast<uint4 *>(ws.x + (uint64_t)m * c.k);
  for (uint32_t first = thread; first < pieces; first += HELD * THREADS) {
    if (pieces > HELD * THREADS) load(first);
#pragma unroll
    for (uint32_t j = 0; j < HELD; ++j) {
      const uint32_t u[4] = {held[j].x, held[j].y, held[j].z, held[j].w};
      uint32_t r[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __half2 h = __floats2half2_rn(__uint_as_float(u[i] << 16) * f0 * f1, __uint_as_float(u[i] & 0xffff0000u) * f0 * f1);
        r[i] = *reinterpret_cast<const uint32_t *>(&h);
      }
      if (first + j * THREADS < pieces) out[first + j * THREADS] = make_uint4(r[0], r[1], r[2], r[3]);
    }
  }
  if (thread == 0) ws.x_unit[m] = power_of_two(e / 2);
}

// Blocks 0 .. token_blocks - 1 make tokens, one each or, of many tokens, one a warp: a block to a row is there sooner, a warp to a row needs no barrier so that more
// of them are at work (2048 x 4096 with the weights of 4096 outputs: 14 us with blocks). The others make weight rows.
__global__ void __launch_bounds__(kPrepThreads, 4)
w4_prepare_kernel(const W4Call c, const Workspace ws, uint32_t matrices, uint32_t param_rows, uint32_t token_blocks) {
  pdl_wait();
  pdl_trigger();  // after the wait: what the next kernel reads ahead of its own wait was complete before this one began
  if (blockIdx.x >= token_blocks) {
    prepare_weights(c, ws, matrices, param_rows, blockIdx.x - token_blocks);
  } else if (token_blocks == c.rows) {
    prepare_token<kPrepThreads, 8>(c, ws, blockIdx.x);
  } else {
    const uint32_t m = blockIdx.x * kPrepWarps + threadIdx.x / 32;
    if (m < c.rows) prepare_token<32, 8>(c, ws, m);
  }
}

// ---- second kernel: the products ------------------------------------------------------------------

__device__ __forceinline__ bool mbar_try_wait_cluster(uint64_t *bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
// As mbar_wait, but the clock is not read before the sixty-fourth poll: a stage has several hand-overs, and reading it takes longer than one. REMOTE: for
// barriers that threads of the other CTA arrive at.
template <bool REMOTE>
__device__ __forceinline__ bool wait_for(uint64_t *bar, uint32_t parity) {
  uint64_t start = 0;
  for (uint32_t i = 0; i < (1u << 30); ++i) {
    if (REMOTE ? mbar_try_wait_cluster(bar, parity) : mbar_try_wait(bar, parity)) return true;
    if ((i & 63u) == 63u) {
      const uint64_t now = global_timer_ns();
      if (start == 0) start = now;
      else if (now - start > 2000000000ull) return false;
    }
  }
  return false;
}
// Four bytes to the other CTA's shared memory, counted on its barrier.
__device__ __forceinline__ void st_async(uint32_t cluster_addr, uint32_t v, uint32_t bar_cluster_addr) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.u32 [%0], %1, [%2];" ::"r"(cluster_addr), "r"(v), "r"(bar_cluster_addr) : "memory");
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
// A from tensor memory (128 rows, 16 k in eight columns), B from shared memory
__device__ __forceinline__ void umma_tmem_a(uint32_t tmem_d, uint32_t tmem_a, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// 32 codes of a row, all of one group, as sixteen pairs in f16: (code - zero) * 2^-9 * scale. The difference first, which is exact: one fused multiply-add
// of codes, scale and -8 * scale would save an instruction a pair where zeros are 8, but leaves a weight in steps of 2^-24, which are coarser than its last
// bits where its scale is below 2^-7 of the row's largest; these are exact down to 2^-21 of it.
__device__ __forceinline__ void dequant_piece(uint4 codes, uint32_t param, uint32_t *v) {
  constexpr uint32_t kLow = 0x78007800u, kHigh = 0x68006800u;  // 2^15, 2^11: of pairs in bits 0-3, and in bits 4-7
  const uint32_t scale = __byte_perm(param, 0, 0x1010), minus_zero = hmul2(__byte_perm(param, 0, 0x3232), 0xf800f800u);
  const uint32_t words[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
  for (uint32_t j = 0; j < 4; ++j) {
    const uint32_t rest = words[j] >> 8;
    v[4 * j] = hmul2(hfma2(words[j] & 0x000f000fu, kLow, minus_zero), scale);
    v[4 * j + 1] = hmul2(hfma2(words[j] & 0x00f000f0u, kHigh, minus_zero), scale);
    v[4 * j + 2] = hmul2(hfma2(rest & 0x000f000fu, kLow, minus_zero), scale);
    v[4 * j + 3] = hmul2(hfma2(rest & 0x00f000f0u, kHigh, minus_zero), scale);
  }
}
__device__ __forceinline__ uint4 ld_codes(const uint8_t *p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint32_t ld_params(const uint32_t *p) {  // in program order, so that a later load does not wait for the stage's arithmetic
  uint32_t v;
  asm volatile("ld.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void sts128(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// f32 accumulation, f16 x f16
__device__ __forceinline__ constexpr uint32_t idesc_f16(uint32_t m, uint32_t n) { return (1u << 4) | ((n >> 3) << 17) | ((m >> 4) << 24); }

template <typename F, bool GATED>
__global__ void __launch_bounds__(F::kWarps * 32, 1)
w4_tile_kernel(const W4Call c, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
               const __grid_constant__ CUtensorMap map_up, const Workspace ws, const Plan plan, const uint32_t param_rows, uint32_t *error) {
  constexpr uint32_t kStages = F::kStages, kMatrices = GATED ? 2 : 1;
  constexpr bool kPair = F::kCtas == 2;
  extern __shared__ uint8_t raw_smem[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~uintptr_t(1023));
  uint8_t *w_ring = smem, *x_ring = smem + F::kXRing;
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + F::kBarriers);
  uint64_t *empty = full + kStages, *acc_full = empty + kStages, *acc_empty = acc_full + 2, *code_full = acc_empty + 2, *code_empty = code_full + F::kCodeStages;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(code_empty + F::kCodeStages), *word = tmem_slot + 1;  // word: of a pair's leader, one a stage

  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = blockIdx.x % F::kCtas, unit = blockIdx.x / F::kCtas, units = gridDim.x / F::kCtas;
  const bool leader = rank == 0;
  const uint32_t total = plan.tiles_w * plan.tiles_x * plan.splits, weight_rows = kMatrices * c.n;

  if (threadIdx.x == 0) {
    for (uint32_t s = 0; s < kStages; ++s) {
      // leader: its own weights, the announcement of bytes (both CTAs' tokens, word of the peer's weights); peer: its weights
      mbar_init(&full[s], !leader ? kDequantWarps : 1 + kDequantWarps);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], F::kCtas * Pair::kEpilogueWarps);  // both CTAs' epilogues (used in the leader)
    }
    for (uint32_t s = 0; s < F::kCodeStages; ++s) {
      mbar_init(&code_full[s], 1);
      mbar_init(&code_empty[s], kDequantWarps);
    }
    mbar_fence_init();
  }
  if (warp == 1) {
    if constexpr (kPair) {
      tmem_alloc_pair(tmem_slot, Pair::kTmemCols);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_slot, Pair::kTmemCols);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (kPair) {
    cluster_arrive_release();  // the peer's barriers exist before anything of this CTA signals them
    cluster_wait_acquire();
  }
  tc_fence_after();
  pdl_trigger();
  const uint32_t tmem_base = *tmem_slot;
  bool ok = true;
  auto wait = [](uint64_t *bar, uint32_t parity) {  // one answer for a warp
    return (bool)__all_sync(0xffffffffu, wait_for<kPair>(bar, parity));
  };
  auto commit = [](uint64_t *bar) {  // on this barrier in all CTAs of the unit, once the MMAs issued so far have ended
    if constexpr (kPair) umma_commit_both(bar);
    else umma_commit(bar);
  };

  // A job: weight rows w_row .. + 255 against tokens x_row .. + cols - 1, stages kb .. end - 1 of k. Splits of a tile are neighbours: they share tokens and
  // weights of L2.
  struct Job {
    uint32_t w_row, x_row, cols, kb, end, split;
  };
  auto job = [&](uint32_t id) {
    const TileXy t = raster(id / plan.splits, plan.tiles_w, plan.tiles_x);
    const uint32_t split = id % plan.splits, x_row = t.y * plan.tokens;
    return Job{t.x * F::kTileRows, x_row, min(plan.tokens, (c.rows - x_row + 31) / 32 * 32), split * plan.stages / plan.splits, (split + 1) * plan.stages / plan.splits, split};
  };

  if (warp == 0) {
    // Tokens: this CTA's half of a tile's; the bytes of both CTAs are counted on the leader's barrier. Nothing is there beyond the last token and k: zeros.
    const bool elected = elect_one();
    const uint32_t box = plan.tokens / F::kCtas;
    uint32_t it = 0;
    pdl_wait();
    for (uint32_t t = unit; ok && t < total; t += units) {
      const Job j = job(t);
      for (uint32_t kb = j.kb; kb < j.end; ++kb, ++it) {
        const uint32_t s = it % kStages;
        if (it >= kStages && !wait(&empty[s], ((it / kStages) & 1) ^ 1)) { ok = false; break; }
        if (elected) {
          if (leader) mbar_arrive_expect_tx(&full[s], F::kCtas * F::kSlabs * box * Pair::kSlabK * 2 + (kPair ? kWordBytes : 0));
#pragma unroll
          for (uint32_t h = 0; h < F::kSlabs; ++h) {
            uint8_t *to = x_ring + s * F::kXBytes + h * F::kXSlab;
            const int k = (int)(kb * F::kStageK + h * Pair::kSlabK), row = (int)(j.x_row + rank * (j.cols / F::kCtas));
            if constexpr (kPair) tma_load_2d_pair(to, &map_x, k, row, mapa_u32(smem_u32(&full[s]), 0));
            else tma_load_2d(to, &map_x, k, row, &full[s]);
          }
        }
        __syncwarp();
      }
    }
    // the slots that are still being read: nobody signals a barrier of a CTA that is gone
    for (uint32_t i = it > kStages ? it - kStages : 0; ok && i < it; ++i) ok = wait(&empty[i % kStages], (i / kStages) & 1);
  } else if (warp == 1) {
    if (leader) {  // issues for both CTAs
      const uint64_t w_desc = desc_k_sw128(smem_u32(w_ring)), x_desc = desc_k_sw128(smem_u32(x_ring));
      const bool elected = elect_one();
      uint32_t it = 0, turn = 0;
      for (uint32_t t = unit; ok && t < total; t += units, ++turn) {
        const Job j = job(t);
        const uint32_t id = idesc_f16(F::kTileRows, j.cols), buf = turn & 1, acc = tmem_base + buf * F::kAccCols;
        if (!wait(&acc_empty[buf], ((turn >> 1) & 1) ^ 1)) { ok = false; break; }
        tc_fence_after();
        for (uint32_t kb = j.kb; kb < j.end; ++kb, ++it) {
          const uint32_t s = it % kStages;
          if (!wait(&full[s], (it / kStages) & 1)) { ok = false; break; }
          tc_fence_after();
          if (elected) {
            const uint64_t a = w_desc + s * (Pair::kWBytes >> 4), b = x_desc + s * (F::kXBytes >> 4);
#pragma unroll
            for (uint32_t h = 0; h < F::kSlabs; ++h)
#pragma unroll
              for (uint32_t k = 0; k < Pair::kSlabK / 16; ++k) {
                const uint64_t a_at = a + ((h * Pair::kWSlab + k * 32) >> 4), b_at = b + ((h * F::kXSlab + k * 32) >> 4);
                const uint32_t more = kb > j.kb || h > 0 || k > 0 ? 1u : 0u;
                if constexpr (kPair) umma_bf16_pair(acc, a_at, b_at, id, more);
                else umma_tmem_a(acc, tmem_base + F::kTmemWeights + s * F::kTmemStage + (h * (Pair::kSlabK / 16) + k) * 8, b_at, id, more);
              }
            commit(&empty[s]);
          }
          __syncwarp();
        }
        if (ok && elected) commit(&acc_full[buf]);
      }
    } else {
      // Hands word of this CTA's weights on to the leader, whose MMA reads them: an asynchronous store, whose completion on the leader's barrier is a release at
      // cluster scope that follows its issue here, behind the wait for the weights. (An arrival released to the cluster waits some hundred cycles at every stage:
      // 2048 x 4096 to 4096 in 109 us against 67.7, gated 4096 x 4096 to 14336 in 763 against 656. One at CTA scope, 67.0 and 651, orders nothing between the two.)
      uint32_t it = 0;
      for (uint32_t t = unit; ok && t < total; t += units) {
        const Job j = job(t);
        for (uint32_t kb = j.kb; kb < j.end; ++kb, ++it) {
          if (!wait(&full[it % kStages], (it / kStages) & 1)) { ok = false; break; }
          if (lane == 0) st_async(mapa_u32(smem_u32(&word[it % kStages]), 0), it, mapa_u32(smem_u32(&full[it % kStages]), 0));
          __syncwarp();
        }
      }
    }
  } else if (F::kWeightsInTmem && warp == F::kCodesWarp) {
    // Codes, ahead of everything else: the weights were complete before the first kernel began, whose beginning this one's launch waited for. With a gate the
    // 64 rows of the gate's come first, then those of the other matrix.
    if constexpr (F::kWeightsInTmem) {
      const bool elected = elect_one();
      uint32_t it = 0;
      for (uint32_t t = unit; ok && t < total; t += units) {
        const Job j = job(t);
        for (uint32_t kb = j.kb; kb < j.end; ++kb, ++it) {
          const uint32_t s = it % F::kCodeStages;
          if (it >= F::kCodeStages && !wait(&code_empty[s], ((it / F::kCodeStages) & 1) ^ 1)) { ok = false; break; }
          if (elected) {
            uint8_t *to = smem + F::kCodeRing + s * F::kCodeBytes;
            mbar_arrive_expect_tx(&code_full[s], F::kCodeBytes);
            tma_load_2d(to, &map_w, (int)(kb * F::kCodeRow), (int)(j.w_row / kMatrices), &code_full[s]);
            if (GATED) tma_load_2d(to + F::kCodeBytes / 2, &map_up, (int)(kb * F::kCodeRow), (int)(j.w_row / kMatrices), &code_full[s]);
          }
          __syncwarp();
        }
      }
    }
  } else if (F::kWeightsInTmem && warp < F::kFirstEpilogue) {
    // Weights to tensor memory: a lane is a row of the tile, a warp the 32 rows whose lanes of tensor memory it may write; it makes the k of a stage for
    // each, 64 at a time. With a gate every other row of a tile is the gate's and the next the other matrix's, so that a pair of lanes of the epilogue holds
    // both. What a stage costs a warp besides its weights counts less with few warps to a stage: teams of four take turns.
    constexpr uint32_t kPieces = F::kStageK / 32;
    const uint32_t team = (warp - kFirstDequant) / kDequantWarps, in_tile = (warp & 3) * 32 + lane;
    const uint32_t code_row = GATED ? (in_tile & 1) * 64 + (in_tile >> 1) : in_tile, code_turn = F::kCodeRow == 128 ? code_row & 7 : (code_row >> 1) & 3;  // how TMA permutes rows of 128 and of 64 bytes
    const uint32_t code_from = smem_u32(smem + F::kCodeRing) + code_row * F::kCodeRow;
    const uint32_t to = tmem_base + (((warp & 3) * 32u) << 16) + F::kTmemWeights;
    const uint32_t group_bits = 31 - __clz((int)c.group), groups = c.k / c.group;
    pdl_wait();

    // Jobs and stages. The scales and zero points of the team's next stage are on their way while this one is made; they stay as loaded, since anything done
    // to them ahead of time would wait for them.
    uint32_t load_t = unit, load_kb = 0, load_end = 0, load_row = 0, next[kPieces];
    auto aim = [&] {
      if (load_t >= total) return;
      const Job j = job(load_t);
      load_kb = j.kb, load_end = j.end, load_row = j.w_row + in_tile;
    };
    auto advance = [&] {
      if (load_t < total && ++load_kb == load_end) load_t += units, aim();
    };
    auto load = [&] {
      if (load_t >= total) return;
      // beyond the last k weights are zeros, as the tokens there
#pragma unroll
      for (uint32_t i = 0; i < kPieces; ++i)
        if (i % 4 == 0 || group_bits < 7 - (i & 1 ? 1 : 0)) {  // one, two or four groups in 128 k
          const uint32_t group = (load_kb * F::kStageK + i * 32) >> group_bits;
          next[i] = group < groups ? ld_params(ws.params + (uint64_t)group * param_rows + load_row) : 0u;
        }
    };
    aim();
    for (uint32_t i = 0; i < team; ++i) advance();
    load();
    for (uint32_t round = 0; ok && load_t < total; ++round) {
      uint32_t param[kPieces];
#pragma unroll
      for (uint32_t i = 0; i < kPieces; i += 4) {
        param[i] = next[i], param[i + 2] = group_bits < 7 ? next[i + 2] : param[i];
        param[i + 1] = group_bits < 6 ? next[i + 1] : param[i], param[i + 3] = group_bits < 6 ? next[i + 3] : param[i + 2];
      }
#pragma unroll
      for (uint32_t i = 0; i < F::kTeams; ++i) advance();
      const uint32_t it = team + round * F::kTeams, s = it % kStages, cs = it % F::kCodeStages;
      if (!wait(&code_full[cs], (it / F::kCodeStages) & 1)) { ok = false; break; }
      load();
      if (it >= kStages && !wait(&empty[s], ((it / kStages) & 1) ^ 1)) { ok = false; break; }
      tc_fence_after();
#pragma unroll
      for (uint32_t i0 = 0; i0 < kPieces; i0 += 4) {
        uint4 codes[4];
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) codes[i] = lds128(code_from + cs * F::kCodeBytes + (((i0 + i) ^ code_turn) * 16));
#pragma unroll
        for (uint32_t half = 0; half < 2; ++half) {
          uint32_t v[32];
#pragma unroll
          for (uint32_t i = 0; i < 2; ++i) dequant_piece(codes[half * 2 + i], param[i0 + half * 2 + i], &v[i * 16]);
          tmem_st32(to + s * F::kTmemStage + (i0 + half * 2) * 16, v);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&code_empty[cs]);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&full[s]);
    }
  } else if (!F::kWeightsInTmem && warp < F::kFirstEpilogue) {
    // Weights to shared memory: 32 rows of the CTA's 128 a warp, as four sets of eight; a lane has 32 k (piece) of a row of each. Rows and teams as above.
    const uint32_t piece = lane & 3, q8 = lane >> 2, team = (warp - kFirstDequant) / kDequantWarps;
    const uint32_t in_tile = (warp - kFirstDequant) % kDequantWarps * 32 + (GATED ? 2 * (q8 & 3) + (q8 >> 2) : q8);
    // chunks of 16 bytes are permuted by row & 7; lanes of the upper 64 k take theirs in another order, so that eight lanes meet eight different banks
    constexpr uint32_t kTurn = GATED ? 1 : 2;
    const bool turned = piece >= 2;
    const uint32_t to = smem_u32(w_ring) + (piece >> 1) * Pair::kWSlab + in_tile * 128, chunk = (((piece & 1) * 4) ^ (turned ? kTurn : 0) ^ (in_tile & 7)) * 16;
    const uint32_t group_bits = 31 - __clz((int)c.group), groups = c.k / c.group;
    const uint8_t *packed = reinterpret_cast<const uint8_t *>(GATED && (in_tile & 1) ? c.up.packed : c.w.packed);
    const uint64_t set_step = (uint64_t)c.k / 2 * (8 / kMatrices);

    // Jobs and stages. The next stage of the team's, codes, scales and zero points, is on its way while this one is made; it stays as loaded, since anything
    // done to it ahead of time would wait for it.
    uint32_t load_t = unit, load_kb = 0, load_end = 0, load_row = 0, next[4];
    uint4 next_codes[4];
    auto aim = [&] {
      if (load_t >= total) return;
      const Job j = job(load_t);
      load_kb = j.kb, load_end = j.end, load_row = j.w_row + rank * Pair::kRows + in_tile;
    };
    auto load_codes = [&] {
      if (load_t >= total) return;
      // beyond the last k scales and tokens are zeros: any codes do
      const uint32_t row = load_row / kMatrices, at = min(load_kb * (Pair::kStageK / 2) + piece * 16, c.k / 2 - 16);
      const uint8_t *p = packed + (uint64_t)row * (c.k / 2) + at;
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) next_codes[i] = row + i * (8 / kMatrices) < c.n ? ld_codes(p + i * set_step) : make_uint4(0, 0, 0, 0);
    };
    auto advance = [&] {
      if (load_t < total && ++load_kb == load_end) load_t += units, aim();
    };
    auto load = [&] {
      if (load_t >= total) return;
      const uint32_t group = (load_kb * Pair::kStageK + piece * 32) >> group_bits;
      const uint32_t *p = ws.params + (uint64_t)group * param_rows + load_row;
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) next[i] = group < groups ? ld_params(p + i * 8) : 0u;
    };
    aim();
    for (uint32_t i = 0; i < team; ++i) advance();
    load_codes();  // ahead of everything else: the weights were complete before the first kernel began, whose beginning this one's launch waited for
    pdl_wait();
    load();
    for (uint32_t round = 0; ok && load_t < total; ++round) {
      uint32_t param[4];
      uint4 codes[4];
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) param[i] = next[i], codes[i] = next_codes[i];
#pragma unroll
      for (uint32_t i = 0; i < F::kTeams; ++i) advance();
      load_codes();
      load();
      const uint32_t it = team + round * F::kTeams, s = it % kStages;
      if (it >= kStages && !wait(&empty[s], ((it / kStages) & 1) ^ 1)) { ok = false; break; }
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) {
        uint32_t v[16];
        const uint4 w = codes[i];
        dequant_piece(!turned ? w : kTurn == 1 ? make_uint4(w.y, w.x, w.w, w.z) : make_uint4(w.z, w.w, w.x, w.y), param[i], v);
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) sts128(to + s * Pair::kWBytes + i * 8 * 128 + (chunk ^ (j * 16)), v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&full[s]);
    }
  } else {
    // Epilogue: warp w reads tensor-memory lanes 32 * (w % 4) .. + 31 (lane = weight row, column = token); the two warps of the same lanes take turns, 16
    // columns each.
    pdl_wait();
    uint32_t turn = 0;
    for (uint32_t t = unit; ok && t < total; t += units, ++turn) {
      const Job j = job(t);
      const uint32_t buf = turn & 1, acc = tmem_base + (((warp & 3) * 32u) << 16) + buf * F::kAccCols;
      const uint32_t r = j.w_row + rank * Pair::kRows + (warp & 3) * 32 + lane, row = GATED ? r >> 1 : r;
      const bool inside = row < c.n;
      const float row_unit = ws.w_unit[r];
      const float bias = !GATED && inside && c.bias && plan.splits == 1 ? c.bias[row] : 0.f;
      if (!wait(&acc_full[buf], (turn >> 1) & 1)) { ok = false; break; }
      tc_fence_after();
      constexpr uint32_t kStep = 16 * (Pair::kEpilogueWarps / 4);
      uint32_t mb = 16 * ((warp - F::kFirstEpilogue) / 4);
      auto release = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane != 0) return;
        if constexpr (kPair) mbar_arrive_cluster(mapa_u32(smem_u32(&acc_empty[buf]), 0));
        else mbar_arrive(&acc_empty[buf]);
      };
      if (mb >= j.cols) release();
#pragma unroll 1
      for (; mb < j.cols; mb += kStep) {
        uint32_t rr[16];
        tmem_ld16(acc + mb, rr);
        tmem_ld_wait();
        if (mb + kStep >= j.cols) release();
        const uint32_t token = j.x_row + mb;
        float v[16];
#pragma unroll
        for (uint32_t q = 0; q < 4; ++q) {
          const float4 f = *reinterpret_cast<const float4 *>(ws.x_unit + token + 4 * q);
          const float unit[4] = {row_unit * f.x, row_unit * f.y, row_unit * f.z, row_unit * f.w};
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i) v[4 * q + i] = __uint_as_float(rr[4 * q + i]) * unit[i] * unit[i];
        }
        // a lane's column of values, `count` of them there, `step` elements apart
        auto store = [&](auto *p, uint64_t step, uint32_t count, uint32_t most, auto value) {
          if (count >= most) {
#pragma unroll
            for (uint32_t q = 0; q < 16; ++q, p += step)
              if (q < most) *p = value(q);
          } else {
#pragma unroll
            for (uint32_t q = 0; q < 16; ++q, p += step)
              if (q < count) *p = value(q);
          }
        };
        const uint32_t there = inside && token < c.rows ? c.rows - token : 0;
        if (!kPair && plan.splits > 1) {  // over the tokens, which nothing reads any more
          store(reinterpret_cast<float *>(smem) + mb * Pair::kRows + (warp & 3) * 32 + lane, Pair::kRows, 16, 16, [&](uint32_t q) { return v[q]; });
        } else if (plan.splits > 1) {
          store(ws.parts + ((uint64_t)j.split * c.rows + token) * weight_rows + r, weight_rows, there, 16, [&](uint32_t q) { return v[q]; });
        } else if (GATED) {
          const bool odd = lane & 1;
          float other[8];
#pragma unroll
          for (uint32_t q = 0; q < 8; ++q) other[q] = __shfl_xor_sync(0xffffffffu, odd ? v[q] : v[8 + q], 1);
          const uint32_t mine = odd ? there > 8 ? there - 8 : 0 : there;
          store(static_cast<bf16 *>(c.out) + (uint64_t)(token + (odd ? 8 : 0)) * c.ldo + row, c.ldo, mine, 8, [&](uint32_t q) {
            return __float2bfloat16_rn(gated<bf16>(GatedAct{c.act, 0.f}, odd ? other[q & 7] : v[q & 7], odd ? v[8 + (q & 7)] : other[q & 7]));
          });
        } else {
          store(static_cast<bf16 *>(c.out) + (uint64_t)token * c.ldo + row, c.ldo, there, 16, [&](uint32_t q) { return __float2bfloat16_rn(v[q] + bias); });
        }
      }
    }
  }
  if (!ok) {  // copies that are on their way land in a few microseconds: they find this CTA's memory still there
    atomicOr(error, 1u);
    const uint64_t start = global_timer_ns();
    for (uint32_t i = 0; i < (1u << 20) && global_timer_ns() - start < 200000u; ++i) {
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (!kPair) {
    if (plan.splits > 1) {
      // The parts of a tile's k, in the CTAs of a cluster, each of which sums every splits-th token, in the order of k.
      cluster_arrive_release();
      cluster_wait_acquire();
      const Job j = job(unit);
      const uint32_t part = smem_u32(smem), tokens = min(j.cols, c.rows - j.x_row), outputs = Pair::kRows / kMatrices;
      for (uint32_t i = threadIdx.x; i < (tokens + plan.splits - 1) / plan.splits * outputs; i += F::kWarps * 32) {
        const uint32_t token = i / outputs * plan.splits + j.split, col = i % outputs, row = j.w_row / kMatrices + col;
        if (token >= tokens || row >= c.n) continue;
        float y[kMatrices];
#pragma unroll
        for (uint32_t m = 0; m < kMatrices; ++m) {
          y[m] = 0.f;
          for (uint32_t s = 0; s < plan.splits; ++s) y[m] += ld_cluster_f32(mapa_u32(part + (token * Pair::kRows + col * kMatrices + m) * 4, s));
        }
        const float out = GATED ? gated<bf16>(GatedAct{c.act, 0.f}, y[0], y[kMatrices - 1]) : y[0] + (c.bias ? c.bias[row] : 0.f);
        static_cast<bf16 *>(c.out)[(uint64_t)(j.x_row + token) * c.ldo + row] = __float2bfloat16_rn(out);
      }
      cluster_arrive_release();  // nobody leaves while its parts are being read
      cluster_wait_acquire();
    }
  }
  // Neither CTA leaves, nor frees the tensor memory the pair allocated together, while the other may still be read by an MMA or be reading its accumulator.
  if constexpr (kPair) {
    cluster_arrive_release();
    cluster_wait_acquire();
  }
  if (warp == 1) {
    if constexpr (kPair) tmem_dealloc_pair(tmem_base, Pair::kTmemCols);
    else tmem_dealloc(tmem_base, Pair::kTmemCols);
  }
}

// ---- third kernel: the parts of k, in order --------------------------------------------------------

template <bool GATED>
__global__ void __launch_bounds__(256) w4_sum_kernel(const W4Call c, const float *__restrict__ parts, uint32_t splits, uint32_t blocks_n) {
  pdl_wait();
  pdl_trigger();
  const uint32_t m = blockIdx.x / blocks_n, n = blockIdx.x % blocks_n * 256 + threadIdx.x;
  if (n >= c.n) return;
  constexpr uint32_t kMatrices = GATED ? 2 : 1;
  const uint64_t slab = (uint64_t)c.rows * kMatrices * c.n;
  const float *p = parts + ((uint64_t)m * c.n + n) * kMatrices;
  float y;
  if constexpr (GATED) {
    float g = 0.f, u = 0.f;
    for (uint32_t s = 0; s < splits; ++s) {
      const float2 v = *reinterpret_cast<const float2 *>(p + s * slab);
      g += v.x, u += v.y;
    }
    y = gated<bf16>(GatedAct{c.act, 0.f}, g, u);
  } else {
    y = 0.f;
    for (uint32_t s = 0; s < splits; ++s) y += p[s * slab];
    if (c.bias) y += c.bias[n];
  }
  static_cast<bf16 *>(c.out)[(uint64_t)m * c.ldo + n] = __float2bfloat16_rn(y);
}

// [rows][cols] matrix of f16 values or of bytes, without gaps; boxes of box_cols x box_rows.
int matrix_map(CUtensorMap *map, bool bytes, CUtensorMapSwizzle swizzle, const void *base, uint64_t rows, uint64_t cols, uint32_t box_cols, uint32_t box_rows) {
  EncodeFn fn = encode_fn();
  if (!fn) return set_error(ORION_ERR_BACKEND, "backend cuda failed at tensor map: driver entry point missing");
  const cuuint64_t dims[2] = {cols, rows}, strides[1] = {cols * (bytes ? 1 : 2)};
  const cuuint32_t box[2] = {box_cols, box_rows}, one[2] = {1, 1};
  const CUresult r = fn(map, bytes ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void *>(base), dims, strides, box, one,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return set_error(ORION_ERR_BACKEND, "backend cuda failed at tensor map: encode returned %d (%llu x %llu)", (int)r, (unsigned long long)rows, (unsigned long long)cols);
  return ORION_OK;
}

template <typename F, bool GATED>
int launch_form(const W4Call &c, const Workspace &ws, const Plan &plan, uint32_t *error, cudaStream_t stream) {
  static bool done[kMaxDeviceOrdinals] = {};
  ORION_CUDA_CHECK("4-bit product", ensure_dynamic_smem(w4_tile_kernel<F, GATED>, F::kSmemBytes, done));
  const uint32_t matrices = GATED ? 2 : 1;
  CUtensorMap map_x, map_w, map_up;
  ORION_TRY(matrix_map(&map_x, false, CU_TENSOR_MAP_SWIZZLE_128B, ws.x, c.rows, c.k, Pair::kSlabK, plan.tokens / F::kCtas));
  map_w = map_up = map_x;
  constexpr CUtensorMapSwizzle code_swizzle = F::kCodeRow == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
  if (F::kWeightsInTmem) {
    ORION_TRY(matrix_map(&map_w, true, code_swizzle, c.w.packed, c.n, c.k / 2, F::kCodeRow, Pair::kRows / matrices));
    if (GATED) ORION_TRY(matrix_map(&map_up, true, code_swizzle, c.up.packed, c.n, c.k / 2, F::kCodeRow, Pair::kRows / 2));
  }
  const uint32_t jobs = plan.tiles_w * plan.tiles_x * plan.splits;
  const uint32_t param_rows = (uint32_t)padded_rows(c.n * matrices), token_blocks = c.rows > 512 ? (c.rows + kPrepWarps - 1) / kPrepWarps : c.rows;
  ORION_CUDA_CHECK("4-bit product", launch_pdl(w4_prepare_kernel, dim3(token_blocks + param_rows / 32), dim3(kPrepThreads), 0, stream, c, ws, matrices, param_rows, token_blocks));
  ORION_CUDA_CHECK("4-bit product", launch_pdl_cluster(w4_tile_kernel<F, GATED>, dim3(F::kCtas * std::min(jobs, kSms / F::kCtas)), dim3(F::kWarps * 32),
                                                       dim3(F::kCtas == 1 ? plan.splits : F::kCtas, 1, 1), F::kSmemBytes, stream, c, map_x, map_w, map_up, ws, plan, param_rows, error));
  count_launch();
  count_launch();
  if (F::kCtas == 2 && plan.splits > 1) {
    ORION_CUDA_CHECK("4-bit product", launch_pdl(w4_sum_kernel<GATED>, dim3((c.n + 255) / 256 * c.rows), dim3(256), 0, stream, c, (const float *)ws.parts, plan.splits,
                                                 (c.n + 255) / 256));
    count_launch();
  }
  return ORION_OK;
}

template <bool GATED>
int launch_kind(const W4Call &c, const Workspace &ws, const Plan &plan, uint32_t *error, cudaStream_t stream) {
  if (plan.ctas == 2) return launch_form<Paired, GATED>(c, ws, plan, error, stream);
  if (plan.tokens > Single64::kAccCols) return launch_form<Single128, GATED>(c, ws, plan, error, stream);
  return launch_form<Single64, GATED>(c, ws, plan, error, stream);
}

}  // namespace

uint64_t w4_tiles_workspace(uint32_t rows, uint32_t weight_rows, uint32_t k, uint32_t group) {
  uint64_t bytes = 0;
  workspace_at(nullptr, rows, weight_rows, k, group, make_plan(rows, weight_rows, k), &bytes);
  return bytes;
}

int launch_w4_tiles(const W4Call &c, void *workspace, uint32_t *error, cudaStream_t stream) {
  const uint32_t weight_rows = c.up.packed ? 2 * c.n : c.n;
  const Plan plan = make_plan(c.rows, weight_rows, c.k);
  if ((uint64_t)plan.tiles_w * plan.tiles_x * plan.splits > 0x7fffffffull || c.rows > 0x3fffffffu)
    return set_error(ORION_ERR_INVALID_REQUEST, "4-bit product: %u rows x %u outputs are too many for one call", c.rows, c.n);
  uint64_t bytes = 0;
  const Workspace ws = workspace_at(static_cast<uint8_t *>(workspace), c.rows, weight_rows, c.k, c.group, plan, &bytes);
  return c.up.packed ? launch_kind<true>(c, ws, plan, error, stream) : launch_kind<false>(c, ws, plan, error, stream);
}

}  // namespace orion
