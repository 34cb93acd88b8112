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
// Bound by HBM: every weight is read once, in 16-byte loads, four rows in flight per lane. A lane keeps eight weights of a row, the lanes of a group share
// its extremes by shuffles, and a CTA of 32 rows x 256 k gathers its scales in shared memory, since neighbours in memory are neighbours in n.
#include "kernels.h"
#include "w4.cuh"

namespace orion {
namespace {

constexpr uint32_t kRowsPerWarp = 4, kWarps = 8, kTileRows = kRowsPerWarp * kWarps, kTileK = 256;

// (d + e) / divisor rounded to bf16 in one rounding, d >= 0: the quotient in f32 is moved to the neighbour with an odd last bit where it is not exact
// (rounding to odd), after which rounding to 8 bits gives what a single rounding would.
__device__ __forceinline__ float scale_of(float d, float e, float divisor) {
  const float q = __fdiv_rn(d, divisor);
  const float rest = fmaf(-q, divisor, d) + e;
  uint32_t bits = __float_as_uint(q);
  if (rest != 0.f && (bits & 1u) == 0 && q > 0.f) bits += rest > 0.f ? 1u : 0xffffffffu;
  const float s = __bfloat162float(__float2bfloat16_rn(__uint_as_float(bits)));
  return s < 1.17549435e-38f ? 0.f : s;  // NaN stays
}

// w / s to the nearest whole number, ties to even, s > 0 finite and |w / s| below 2^20; `guess` is at most one off.
__device__ __forceinline__ float nearest(float w, float s, float guess) {
  const float rest = fmaf(-guess, s, w), twice = 2.f * fabsf(rest);
  const bool odd = (int)guess & 1;
  return twice > s || (twice == s && odd) ? guess + copysignf(1.f, rest) : guess;
}

template <typename T>
__device__ __forceinline__ void load8(const T *p, float (&v)[8]) {
  if constexpr (sizeof(T) == 2) {
    const uint4 r = __ldg(reinterpret_cast<const uint4 *>(p));
    const uint32_t u[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(u[i] << 16), v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
  } else {
    const float4 a = __ldg(reinterpret_cast<const float4 *>(p)), b = __ldg(reinterpret_cast<const float4 *>(p) + 1);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  }
}

template <typename T, uint32_t GROUP, bool ZEROS>
__global__ void __launch_bounds__(kWarps * 32)
w4_quantize_kernel(const T *__restrict__ w, uint64_t ldw, uint32_t n, uint32_t k, uint32_t tiles_k, uint32_t *__restrict__ packed,
                   bf16 *__restrict__ scales, uint8_t *__restrict__ zeros) {
  constexpr uint32_t kLanes = GROUP / 8, kGroups = kTileK / GROUP;
  __shared__ bf16 tile_s[kGroups][kTileRows];
  __shared__ uint8_t tile_z[kGroups][kTileRows];
  pdl_wait();
  pdl_trigger();
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t row0 = blockIdx.x / tiles_k * kTileRows, k0 = blockIdx.x % tiles_k * kTileK, kk = k0 + lane * 8;
  const bool inside = kk < k;  // whole groups: all lanes of a group agree
  float v[kRowsPerWarp][8];
#pragma unroll
  for (uint32_t r = 0; r < kRowsPerWarp; ++r) {
    const uint32_t row = row0 + warp * kRowsPerWarp + r;
    if (inside && row < n) {
      load8(w + (uint64_t)row * ldw + kk, v[r]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[r][i] = 0.f;
    }
  }
#pragma unroll
  for (uint32_t r = 0; r < kRowsPerWarp; ++r) {
    float hi = 0.f, lo = 0.f;
    bool finite = true;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (ZEROS) lo = fminf(lo, v[r][i]), hi = fmaxf(hi, v[r][i]);
      else hi = fmaxf(hi, fabsf(v[r][i]));
      finite = finite && fabsf(v[r][i]) <= 3.4028234663852886e38f;  // false for NaN
    }
    uint32_t bad = finite ? 0u : 1u;
#pragma unroll
    for (uint32_t o = kLanes / 2; o > 0; o >>= 1) {
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      if (ZEROS) lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      bad |= __shfl_xor_sync(0xffffffffu, bad, o);
    }
    float s, zero = 8.f;
    if (ZEROS) {
      // what the subtraction rounds off goes along (two-sum); halves where the span of f32 weights would not be finite
      const float shrink = hi > 1.7e38f || lo < -1.7e38f ? 0.5f : 1.f;
      const float a = shrink * hi, b = -shrink * lo, span = a + b, bb = span - a, off = (a - (span - bb)) + (b - bb);
      s = scale_of(span, off, 15.f) / shrink;
      const float inv = s > 0.f ? 1.f / s : 0.f;
      zero = s > 0.f ? fminf(nearest(-lo, s, rintf(-lo * inv)), 15.f) : 0.f;
    } else {
      s = scale_of(hi, 0.f, 7.f);
    }
    if (bad) s = __uint_as_float(0x7fc00000u), zero = ZEROS ? 0.f : 8.f;
    const bool some = s > 0.f;  // false for 0 and NaN: every code is the zero point
    const float inv = some ? 1.f / s : 0.f;
    // t = 1.5 * 2^23 + code: its last bits are the code
    constexpr float kMagic = 12582912.f;
    uint32_t word = 0;
    float near = 0.f;
    float code[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float value = some ? v[r][i] : 0.f;
      const float c = fmaf(value, inv, kMagic) - kMagic;
      near = fmaxf(near, fabsf(fmaf(value, inv, -c)));
      code[i] = c;
    }
    if (near > 0.49999f) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (some) code[i] = nearest(v[r][i], s, code[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float c = code[i] + zero;
      if (ZEROS) c = fminf(fmaxf(c, 0.f), 15.f);  // symmetric codes stay within 1 .. 15 by themselves: max|w| / scale is at most 7 (1 + 2^-8)
      word |= (__float_as_uint(c + kMagic) & 15u) << (4 * (i / 2) + 16 * (i & 1));
    }
    const uint32_t row = row0 + warp * kRowsPerWarp + r;
    if (inside && row < n) packed[(uint64_t)row * (k / 8) + kk / 8] = word;
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
  const uint32_t tiles_k = (k + kTileK - 1) / kTileK, tiles_n = (n + kTileRows - 1) / kTileRows;
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
