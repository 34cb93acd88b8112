// Entry points of the 4-bit operators (include/orion_cuda.h): arguments are checked on the host, nothing is allocated, work is enqueued on the caller's
// stream.
#include "kernels.h"
#include "w4.cuh"

#include <atomic>

namespace orion {
namespace {

constexpr uint64_t kMostRows = 1u << 30, kMostFeatures = 1u << 30;

int check_sizes(uint64_t out_features, uint64_t in_features, uint32_t group) {
  if (group != 32 && group != 64 && group != 128)
    return set_error(ORION_ERR_INVALID_REQUEST, "groups of 4-bit weights hold 32, 64 or 128 values, got %u", group);
  if (in_features == 0 || in_features % group != 0 || in_features > kMostFeatures)
    return set_error(ORION_ERR_INVALID_REQUEST, "%llu input features are no whole number of groups of %u (at most 2^30)", (unsigned long long)in_features, group);
  if (out_features == 0 || out_features > kMostFeatures)
    return set_error(ORION_ERR_INVALID_REQUEST, "%llu output features: 1 to 2^30 are possible", (unsigned long long)out_features);
  return ORION_OK;
}

int check_dtype(int dtype) {
  if (dtype != ORION_DTYPE_F32 && dtype != ORION_DTYPE_BF16)
    return set_error(ORION_ERR_INVALID_REQUEST, "4-bit operators take f32 or bf16 values, got dtype %d", dtype);
  return ORION_OK;
}
uint64_t size_of(int dtype) { return dtype == ORION_DTYPE_F32 ? 4 : 2; }
bool aligned(const void *p, uint64_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

// Rows that the kernels read in pieces of 16 bytes.
int check_matrix(const char *what, const void *p, uint64_t rows, uint64_t cols, uint64_t stride, int dtype) {
  if (!p) return set_error(ORION_ERR_INVALID_REQUEST, "%s: null pointer argument", what);
  if (rows > 1 && stride < cols)
    return set_error(ORION_ERR_INVALID_REQUEST, "%s: a row stride of %llu is less than a row of %llu", what, (unsigned long long)stride, (unsigned long long)cols);
  if (stride > (1ull << 40)) return set_error(ORION_ERR_INVALID_REQUEST, "%s: a row stride of %llu is too large", what, (unsigned long long)stride);
  if (!aligned(p, 16) || (rows > 1 && stride * size_of(dtype) % 16 != 0))
    return set_error(ORION_ERR_INVALID_REQUEST, "%s: rows must start on 16-byte boundaries", what);
  return ORION_OK;
}

int check_weight(const char *what, const OrionW4Weight *w) {
  if (!w || !w->packed || !w->scales) return set_error(ORION_ERR_INVALID_REQUEST, "%s: null pointer argument", what);
  ORION_TRY(check_sizes(w->out_features, w->in_features, w->group));
  if (!aligned(w->packed, 16) || !aligned(w->scales, 4) || !aligned(w->zeros, 4))
    return set_error(ORION_ERR_INVALID_REQUEST, "%s: packed weights must start on a 16-byte boundary, scales and zeros on a 4-byte one", what);
  return ORION_OK;
}
W4View view(const OrionW4Weight *w) {
  return {static_cast<const uint32_t *>(w->packed), static_cast<const bf16 *>(w->scales), static_cast<const uint8_t *>(w->zeros)};
}

// What both products have in common; fills `c` but for the activation.
int check_product(int dtype, const void *x, uint64_t rows, uint64_t x_stride, const OrionW4Weight *w, void *out, uint64_t out_stride, W4Call *c) {
  ORION_TRY(check_dtype(dtype));
  ORION_TRY(check_weight("weight", w));
  if (rows > kMostRows) return set_error(ORION_ERR_INVALID_REQUEST, "%llu rows: at most 2^30 are possible", (unsigned long long)rows);
  if (rows == 0) return ORION_OK;
  ORION_TRY(check_matrix("x", x, rows, w->in_features, x_stride, dtype));
  if (!out) return set_error(ORION_ERR_INVALID_REQUEST, "out: null pointer argument");
  if (!aligned(out, size_of(dtype))) return set_error(ORION_ERR_INVALID_REQUEST, "out: not aligned to its type");
  if (rows > 1 && (out_stride < w->out_features || out_stride > (1ull << 40)))
    return set_error(ORION_ERR_INVALID_REQUEST, "out: a row stride of %llu for rows of %llu", (unsigned long long)out_stride, (unsigned long long)w->out_features);
  c->x = x, c->out = out, c->w = view(w), c->ldx = x_stride, c->ldo = out_stride;
  c->rows = (uint32_t)rows, c->n = (uint32_t)w->out_features, c->k = (uint32_t)w->in_features, c->group = w->group;
  return ORION_OK;
}

// Whether a product runs in tiles on tcgen05 (w4_tiles.cu), which needs bf16 and a stage of 256 k, or in the kernel for few rows. The tiles need a kernel ahead
// of theirs and some 9 us until the first of them is done; the others' rate is that of mma.sync. Times in us, tiles / few, weights from HBM: k 2048 to 2048,
// 64 rows 14 / 9, 192 rows 18 / 16, 400 rows 19 / 26; k 4096 to 4096, 32 rows 14 / 10, 64 rows 16 / 15, 128 rows 19 / 23; k 3584 to 4608, 64 rows 15 / 17;
// k 2048 to 16384, 24 rows 14 / 16, 128 rows 19 / 40.
bool takes_tiles(int dtype, uint64_t rows, uint64_t weight_rows, uint64_t k) {
  return dtype == ORION_DTYPE_BF16 && rows > 16 && k >= 256 && (double)(rows > 48 ? rows : 48) * (double)weight_rows * (double)k > 1e9;
}

// Address of the projections' error word, looked up once per device.
int error_word(int device, uint32_t **word) {
  static std::atomic<uint32_t *> known[kMaxDeviceOrdinals];
  const bool tracked = device >= 0 && device < kMaxDeviceOrdinals;
  *word = tracked ? known[device].load(std::memory_order_acquire) : nullptr;
  if (*word) return ORION_OK;
  *word = static_cast<uint32_t *>(const_cast<void *>(gemm_tc_error_word()));
  if (!*word) return set_error(ORION_ERR_BACKEND, "backend cuda failed at error word: %s", cudaGetErrorString(cudaGetLastError()));
  if (tracked) known[device].store(*word, std::memory_order_release);
  return ORION_OK;
}

int launch(int device, int dtype, const W4Call &c, void *workspace, uint64_t workspace_bytes, cudaStream_t stream) {
  const uint32_t weight_rows = c.up.packed ? 2 * c.n : c.n;
  if (!takes_tiles(dtype, c.rows, weight_rows, c.k)) {
    ScopedDevice current(device);
    ORION_CUDA_CHECK("set device", current.status);
    return dtype == ORION_DTYPE_F32 ? launch_w4_few<float>(c, stream) : launch_w4_few<bf16>(c, stream);
  }
  const uint64_t need = w4_tiles_workspace(c.rows, weight_rows, c.k, c.group);
  if (!workspace || workspace_bytes < need || !aligned(workspace, 256))
    return set_error(ORION_ERR_INVALID_REQUEST, "a workspace of %llu bytes on a 256-byte boundary is needed, got %llu", (unsigned long long)need,
                     (unsigned long long)(workspace ? workspace_bytes : 0));
  ScopedDevice current(device);
  ORION_CUDA_CHECK("set device", current.status);
  uint32_t *error = nullptr;
  ORION_TRY(error_word(device, &error));
  return launch_w4_tiles(c, workspace, error, stream);
}

}  // namespace
}  // namespace orion

extern "C" {

using namespace orion;

int orion_cuda_w4_quantize(int device, int dtype, const void *weight, uint64_t out_features, uint64_t in_features, uint64_t row_stride, uint32_t group,
                           void *packed, void *scales, void *zeros, void *stream) {
  clear_error();
  ORION_TRY(check_dtype(dtype));
  ORION_TRY(check_sizes(out_features, in_features, group));
  ORION_TRY(check_matrix("weight", weight, out_features, in_features, row_stride, dtype));
  if (!packed || !scales) return set_error(ORION_ERR_INVALID_REQUEST, "null pointer argument");
  if (!aligned(packed, 16) || !aligned(scales, 4) || !aligned(zeros, 4))
    return set_error(ORION_ERR_INVALID_REQUEST, "packed weights must start on a 16-byte boundary, scales and zeros on a 4-byte one");
  if ((out_features + 31) / 32 * ((in_features + 255) / 256) > 0x7fffffffull)
    return set_error(ORION_ERR_INVALID_REQUEST, "a matrix of %llu x %llu is too large for one call", (unsigned long long)out_features, (unsigned long long)in_features);
  ScopedDevice current(device);
  ORION_CUDA_CHECK("set device", current.status);
  const uint32_t n = (uint32_t)out_features, k = (uint32_t)in_features;
  uint32_t *p = static_cast<uint32_t *>(packed);
  bf16 *s = static_cast<bf16 *>(scales);
  uint8_t *z = static_cast<uint8_t *>(zeros);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == ORION_DTYPE_F32 ? launch_w4_quantize(static_cast<const float *>(weight), row_stride, n, k, group, p, s, z, st)
                                  : launch_w4_quantize(static_cast<const bf16 *>(weight), row_stride, n, k, group, p, s, z, st);
}

int orion_cuda_w4_workspace(int dtype, uint64_t rows, const OrionW4Weight *weight, int gated, uint64_t *bytes) {
  clear_error();
  if (!bytes) return set_error(ORION_ERR_INVALID_REQUEST, "null pointer argument");
  *bytes = 0;
  ORION_TRY(check_dtype(dtype));
  ORION_TRY(check_weight("weight", weight));
  if (rows > kMostRows) return set_error(ORION_ERR_INVALID_REQUEST, "%llu rows: at most 2^30 are possible", (unsigned long long)rows);
  const uint64_t weight_rows = weight->out_features * (gated ? 2 : 1);
  if (takes_tiles(dtype, rows, weight_rows, weight->in_features)) *bytes = w4_tiles_workspace((uint32_t)rows, (uint32_t)weight_rows, (uint32_t)weight->in_features, weight->group);
  return ORION_OK;
}

int orion_cuda_w4_linear(int device, int dtype, const void *x, uint64_t rows, uint64_t x_stride, const OrionW4Weight *weight, const float *bias, void *out,
                         uint64_t out_stride, void *workspace, uint64_t workspace_bytes, void *stream) {
  clear_error();
  W4Call c;
  ORION_TRY(check_product(dtype, x, rows, x_stride, weight, out, out_stride, &c));
  if (rows == 0) return ORION_OK;
  if (!aligned(bias, 4)) return set_error(ORION_ERR_INVALID_REQUEST, "bias: not aligned to its type");
  c.bias = bias;
  return launch(device, dtype, c, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

int orion_cuda_w4_gated(int device, int dtype, const void *x, uint64_t rows, uint64_t x_stride, const OrionW4Weight *gate, const OrionW4Weight *up,
                        int activation, void *out, uint64_t out_stride, void *workspace, uint64_t workspace_bytes, void *stream) {
  clear_error();
  W4Call c;
  ORION_TRY(check_weight("up", up));
  ORION_TRY(check_product(dtype, x, rows, x_stride, gate, out, out_stride, &c));
  if (up->out_features != gate->out_features || up->in_features != gate->in_features || up->group != gate->group)
    return set_error(ORION_ERR_INVALID_REQUEST, "gate and up projection differ: %llu x %llu in groups of %u, %llu x %llu in groups of %u",
                     (unsigned long long)gate->out_features, (unsigned long long)gate->in_features, gate->group, (unsigned long long)up->out_features,
                     (unsigned long long)up->in_features, up->group);
  if (activation != ORION_GATE_SILU && activation != ORION_GATE_GELU_TANH)
    return set_error(ORION_ERR_INVALID_REQUEST, "unknown activation %d", activation);
  if (rows == 0) return ORION_OK;
  c.up = view(up);
  c.act = activation == ORION_GATE_SILU ? kGatedSilu : kGatedGelu;
  return launch(device, dtype, c, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
