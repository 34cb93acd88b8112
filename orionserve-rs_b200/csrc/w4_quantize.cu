// 4-bit codes, scales and zero points of a matrix (w4.cuh has the layout).
//
//   symmetric: scale = max|w| / 7, code = 8 + round(w / scale)
//   with zero points: lo = min(w, 0), hi = max(w, 0), scale = (hi - lo) / 15, zero = round(-lo / scale), code = round(w / scale) + zero in 0 .. 15
//
// Scales are rounded to bf16 (once, to the nearest, ties to even) before anything is divided by them, and a scale below the smallest normal number is 0,
// with every code the zero point's. A group that holds an infinity or a NaN gets a NaN for its scale, so that no product hides it. Quotients are rounded
// to the NEAREST whole number, ties to even: w * (1 / scale) in f32 is off by a few units of 2^-22, so a quotient that comes closer than that to a border
// between two codes is decided by the remainder w - code * scale, which is exact in f32 (a code has four bits, a scale eight, and the difference no more
// than w). One quotient in some 10^5 takes that path.
//
// Bound by HBM, with the instructions close behind: nine a weight where the rate of HBM leaves eleven (14336 x 4096 of f32 in 60 us, 4.5 TB/s, among other work;
// 45 us alone, instructions issued in 72 % of all cycles). So quotients are rounded by adding 1.5 * 2^23,
// codes are packed as sums of multiples of 16 in f32, which are exact, and a lane has sixteen bf16 weights of a row (eight f32 ones), so that what is done once
// for a group's scale is shared. The lanes of a group share its extremes by shuffles; a CTA of 32 rows gathers its scales in shared memory, since neighbours in
// memory are neighbours in n.
#include "kernels.h"
#include "w4.cuh"

namespace orion {
namespace {

constexpr uint32_t kRowsPerWarp = 4, kWarps = 8, kTileRows = kRowsPerWarp * kWarps;
template <typename T>
constexpr uint32_t kPerLane = sizeof(T) == 2 ? 16 : 8;
template <typename T>
constexpr uint32_t kTileK = 32 * kPerLane<T>;

__device__ __forceinline__ float max_or_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// (d + e) / divisor rounded to bf16 in one rounding, d >= 0, inv the f32 number next to 1 / divisor: the quotient in f32, corrected once, is moved to the
// neighbour with an odd last bit where it is not exact (rounding to odd), after which rounding to 8 bits gives what a single rounding would. The correction
// by a remainder that a fused multiply-add makes exact is Markstein's (Computation of elementary functions on the IBM RISC System/6000, 1990), rounding to odd ahead
// of a second rounding Boldo and Melquiond's (Emulation of a FMA and correctly rounded sums, 2008).
__device__ __forceinline__ float scale_of(float d, float e, float divisor, float inv) {
  const float guess = d * inv, q = fmaf(fmaf(-guess, divisor, d), inv, guess);
  const float rest = fmaf(-q, divisor, d) + e;
  uint32_t bits = __float_as_uint(q);
  if (rest != 0.f && (bits & 1u) == 0 && q > 0.f) bits += rest > 0.f ? 1u : 0xffffffffu;
  const float s = __bfloat162float(__float2bfloat16_rn(__uint_as_float(bits)));
  return s < 1.17549435e-38f ? 0.f : s;  // NaN stays
}

// 1 / s to a unit of 2^-23, s > 0; divided where the quotient is no normal number.
__device__ __forceinline__ float reciprocal(float s) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
  return s > 1e37f ? 1.f / s : r;
}

// w / s to the nearest whole number, ties to even, s > 0 finite and |w / s| below 2^20; `guess` is at most one off.
__device__ __forceinline__ float nearest(float w, float s, float guess) {
  const float rest = fmaf(-guess, s, w), twice = 2.f * fabsf(rest);
  const bool odd = (int)guess & 1;
  return twice > s || (twice == s && odd) ? guess + copysignf(1.f, rest) : guess;
}

// Values 8 i .. 8 i + 7 of a lane's sixteen bytes times two.
__device__ __forceinline__ void values_of(const uint4 (&raw)[2], uint32_t i, bf16, float (&v)[8]) {
  const uint32_t u[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
  for (int j = 0; j < 4; ++j) v[2 * j] = __uint_as_float(u[j] << 16), v[2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
}
__device__ __forceinline__ void values_of(const uint4 (&raw)[2], uint32_t, float, float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    v[4 * j] = __uint_as_float(raw[j].x), v[4 * j + 1] = __uint_as_float(raw[j].y);
    v[4 * j + 2] = __uint_as_float(raw[j].z), v[4 * j + 3] = __uint_as_float(raw[j].w);
  }
}

template <typename T, uint32_t GROUP, bool ZEROS>
__global__ void __launch_bounds__(kWarps * 32)
w4_quantize_kernel(const T *__restrict__ w, uint64_t ldw, uint32_t n, uint32_t k, uint32_t tiles_k, uint32_t *__restrict__ packed,
                   bf16 *__restrict__ scales, uint8_t *__restrict__ zeros) {
  constexpr uint32_t kPer = kPerLane<T>, kLanes = GROUP / kPer, kGroups = kTileK<T> / GROUP;
  __shared__ bf16 tile_s[kGroups][kTileRows];
  __shared__ uint8_t tile_z[kGroups][kTileRows];
  pdl_wait();
  pdl_trigger();
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t row0 = blockIdx.x / tiles_k * kTileRows, k0 = blockIdx.x % tiles_k * kTileK<T>, kk = k0 + lane * kPer;
  const bool inside = kk < k;  // whole groups: all lanes of a group agree
  uint4 raw[kRowsPerWarp][2];
#pragma unroll
  for (uint32_t r = 0; r < kRowsPerWarp; ++r) {
    const uint32_t row = row0 + warp * kRowsPerWarp + r;
    raw[r][0] = raw[r][1] = make_uint4(0, 0, 0, 0);
    if (inside && row < n) {
      const uint4 *p = reinterpret_cast<const uint4 *>(w + (uint64_t)row * ldw + kk);
      raw[r][0] = __ldg(p), raw[r][1] = __ldg(p + 1);
    }
  }
#pragma unroll
  for (uint32_t r = 0; r < kRowsPerWarp; ++r) {
    float hi = 0.f, lo = 0.f;
#pragma unroll
    for (uint32_t i = 0; i < kPer / 8; ++i) {
      float v[8];
      values_of(raw[r], i, T{}, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (ZEROS) lo = -max_or_nan(-lo, -v[j]), hi = max_or_nan(hi, v[j]);
        else hi = max_or_nan(hi, fabsf(v[j]));
      }
    }
#pragma unroll
    for (uint32_t o = kLanes / 2; o > 0; o >>= 1) {
      hi = max_or_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      if (ZEROS) lo = -max_or_nan(-lo, -__shfl_xor_sync(0xffffffffu, lo, o));
    }
    const bool finite = hi <= 3.4028234663852886e38f && (!ZEROS || lo >= -3.4028234663852886e38f);  // false for NaN
    float s, zero = 8.f;
    if (ZEROS) {
      // what the subtraction rounds off goes along (two-sum); halves where the span of f32 weights would not be finite
      const float shrink = hi > 1.7e38f || lo < -1.7e38f ? 0.5f : 1.f;
      const float a = shrink * hi, b = -shrink * lo, span = a + b, bb = span - a, off = (a - (span - bb)) + (b - bb);
      s = scale_of(span, off, 15.f, 1.f / 15.f) / shrink;
    } else {
      s = scale_of(hi, 0.f, 7.f, 1.f / 7.f);
    }
    const bool some = finite && s > 0.f;  // else every code is the zero point
    const float inv = some ? reciprocal(s) : 0.f;
    if (ZEROS) zero = some ? fminf(nearest(-lo, s, rintf(-lo * inv)), 15.f) : 0.f;
    constexpr float kMagic = 12582912.f;  // 1.5 * 2^23: the last bits of a sum with it are the whole number next to the other summand
    uint32_t words[kPer / 8];
#pragma unroll
    for (uint32_t i = 0; i < kPer / 8; ++i) {
      float v[8], code[8], near = 0.f;
      values_of(raw[r], i, T{}, v);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        code[j] = fmaf(v[j], inv, kMagic) - kMagic;
        near = fmaxf(near, fabsf(fmaf(v[j], inv, -code[j])));
      }
      if (near > 0.49999f && some) {
#pragma unroll
        for (int j = 0; j < 8; ++j) code[j] = nearest(v[j], s, code[j]);
      }
      if (ZEROS) {  // symmetric codes stay within 1 .. 15 by themselves: max|w| / scale is at most 7 (1 + 2^-8)
#pragma unroll
        for (int j = 0; j < 8; ++j) code[j] = fminf(fmaxf(code[j], -zero), 15.f - zero);
      }
      const float half0 = fmaf(fmaf(fmaf(code[6], 16.f, code[4]), 16.f, code[2]), 16.f, code[0]);
      const float half1 = fmaf(fmaf(fmaf(code[7], 16.f, code[5]), 16.f, code[3]), 16.f, code[1]);
      const float all = fmaf(zero, 4369.f, kMagic);  // the zero point in each of four places
      words[i] = __byte_perm(__float_as_uint(half0 + all), __float_as_uint(half1 + all), 0x5410);
      if (!some) words[i] = ZEROS ? 0u : 0x88888888u;
    }
    if (!finite) s = __uint_as_float(0x7fc00000u);
    const uint32_t row = row0 + warp * kRowsPerWarp + r;
    if (inside && row < n) {
      uint32_t *p = packed + (uint64_t)row * (k / 8) + kk / 8;
      if constexpr (kPer == 16) *reinterpret_cast<uint2 *>(p) = make_uint2(words[0], words[kPer / 8 - 1]);
      else *p = words[0];
    }
    if (lane % kLanes == 0) {
      tile_s[lane / kLanes][warp * kRowsPerWarp + r] = __float2bfloat16_rn(s);
      tile_z[lane / kLanes][warp * kRowsPerWarp + r] = (uint8_t)zero;
    }
  }
  __syncthreads();
  const uint32_t g0 = k0 / GROUP, groups = k / GROUP;
  for (uint32_t i = threadIdx.x; i < kGroups * kTileRows; i += kWarps * 32) {
    const uint32_t g = i / kTileRows, r = i % kTileRows;
    if (g0 + g >= groups || row0 + r >= n) continue;
    scales[(uint64_t)(g0 + g) * n + row0 + r] = tile_s[g][r];
    if (ZEROS) zeros[(uint64_t)(g0 + g) * n + row0 + r] = tile_z[g][r];
  }
}

template <typename T, uint32_t GROUP>
cudaError_t launch_group(const T *w, uint64_t ldw, uint32_t n, uint32_t k, uint32_t *packed, bf16 *scales, uint8_t *zeros, cudaStream_t stream) {
  const uint32_t tiles_k = (k + kTileK<T> - 1) / kTileK<T>, tiles_n = (n + kTileRows - 1) / kTileRows;
  const auto kernel = zeros ? w4_quantize_kernel<T, GROUP, true> : w4_quantize_kernel<T, GROUP, false>;
  return launch_pdl(kernel, dim3(tiles_k * tiles_n), dim3(kWarps * 32), 0, stream, w, ldw, n, k, tiles_k, packed, scales, zeros);
}

}  // namespace

template <typename T>
int launch_w4_quantize(const T *w, uint64_t ldw, uint32_t n, uint32_t k, uint32_t group, uint32_t *packed, bf16 *scales, uint8_t *zeros, cudaStream_t stream) {
  const auto launch = group == 32 ? launch_group<T, 32> : group == 64 ? launch_group<T, 64> : launch_group<T, 128>;
  ORION_CUDA_CHECK("4-bit quantiser", launch(w, ldw, n, k, packed, scales, zeros, stream));
  count_launch();
  return ORION_OK;
}
template int launch_w4_quantize<float>(const float *, uint64_t, uint32_t, uint32_t, uint32_t, uint32_t *, bf16 *, uint8_t *, cudaStream_t);
template int launch_w4_quantize<bf16>(const bf16 *, uint64_t, uint32_t, uint32_t, uint32_t, uint32_t *, bf16 *, uint8_t *, cudaStream_t);

}  // namespace orion
