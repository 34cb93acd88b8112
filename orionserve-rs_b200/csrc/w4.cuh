// 4-bit weights with a scale, and where wanted a zero point, per group of 32, 64 or 128 consecutive k:
//   W[n][k] = (code[n][k] - zero[k / group][n]) * scale[k / group][n],    code and zero 0..15, scale bf16.
// Without zero points every zero is 8.
//
// A 32-bit word holds eight consecutive k: number 2i in bits 4i .. 4i + 3, number 2i + 1 in bits 16 + 4i .. 19 + 4i. So one AND leaves a pair of
// neighbours in the two halves of a register, where a packed 16-bit instruction or a matrix fragment takes them, and eight weights cost one shift and
// four ANDs. Scales and zeros are stored group by group ([in / group][out]), so that the lanes of a warp, which hold different rows, read neighbours.
//
// Scales have the eight significant bits of bf16: (code - 8) * scale then has at most eleven, which an f16 operand holds exactly.
#pragma once

#include "common.cuh"

namespace orion {

struct W4View {
  const uint32_t *packed = nullptr;  // [n][k / 8], 16-byte aligned
  const bf16 *scales = nullptr;      // [k / group][n]
  const uint8_t *zeros = nullptr;    // [k / group][n]; null: 8 everywhere
};

// What a projection reads and writes. up.packed set: y = act(x W^T) * (x up^T); else y = x W^T + bias (bias may be null).
struct W4Call {
  const void *x = nullptr;   // [rows][ldx], T
  void *out = nullptr;       // [rows][ldo], T
  W4View w, up;
  const float *bias = nullptr;
  uint64_t ldx = 0, ldo = 0;
  uint32_t rows = 0, n = 0, k = 0, group = 0;
  GatedKind act = kGatedSilu;
};

template <typename T>
int launch_w4_few(const W4Call &c, cudaStream_t stream);

// bf16 activations of many rows; `workspace` holds w4_tiles_workspace() bytes, `error` is the word that waits which run out set.
uint64_t w4_tiles_workspace(uint32_t rows, uint32_t weight_rows, uint32_t k, uint32_t group);
int launch_w4_tiles(const W4Call &c, void *workspace, uint32_t *error, cudaStream_t stream);

template <typename T>
int launch_w4_quantize(const T *w, uint64_t ldw, uint32_t n, uint32_t k, uint32_t group, uint32_t *packed, bf16 *scales, uint8_t *zeros, cudaStream_t stream);

}  // namespace orion
