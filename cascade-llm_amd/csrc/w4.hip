// Products of a few rows with matrices of 4-bit weights (gfx950).
//
// The layout (include/cascade_hip.h) is that of a wave's load: a tile of 16
// matrix rows and 128 columns is 1 KiB, of which lane l takes the 16 bytes at
// 16 l: row l % 16, and of each 32 columns the eight from 8 (l / 16) on, which
// is its piece of an MFMA operand.
#include "cascade_device.h"
#include "cascade_internal.h"

namespace cascade {

struct W4Matrix {
  const u32x4 *packed;
  const uint16_t *scales;
  const uint8_t *zeros;  // nullable: 8
};

struct W4Args {
  const uint16_t *x;
  int64_t x_stride;
  W4Matrix w[2];  // gate and up for SwiGLU
  int32_t m, n, k;
  int32_t tiles;   // of 128 columns
  int32_t groups;  // of a row
  int32_t group_shift;
  const uint16_t *residual;
  int64_t residual_stride;
  void *y;
  int64_t y_stride;
};

enum W4Out { kW4Bf16, kW4F32, kW4Swiglu };

constexpr int kW4Threads = 64;

__device__ __forceinline__ float w4_row_product(const W4Args &a, const W4Matrix &w, int row,
                                                int col) {
  const uint32_t *words = reinterpret_cast<const uint32_t *>(w.packed);
  float total = 0.0f;
  for (int g = 0; g < a.groups; ++g) {
    const int64_t at = (static_cast<int64_t>(col / 16) * a.groups + g) * 16 + col % 16;
    const float scale = bf16_to_f32(w.scales[at]);
    const int zero = w.zeros != nullptr ? w.zeros[at] : 8;
    const int end = min(a.k, (g + 1) << a.group_shift);
    float sum = 0.0f;
    for (int k = g << a.group_shift; k < end; k += 8) {
      const int64_t tile = static_cast<int64_t>(col / 16) * a.tiles + k / 128;
      const int lane = 16 * (k / 8 % 4) + col % 16;
      uint32_t word = words[tile * 256 + lane * 4 + k / 32 % 4];
      word = (word >> 3) | (word << 29);
      for (int i = 0; i < 8; ++i) {
        const int q = (word >> (16 * (i & 1) + 4 * (i >> 1))) & 15;
        sum = fmaf(bf16_to_f32(a.x[row * a.x_stride + k + i]), static_cast<float>(q - zero), sum);
      }
    }
    total = fmaf(scale, sum, total);
  }
  return total;
}

// One thread an output.
template <int OUT>
__global__ __launch_bounds__(kW4Threads) void w4_kernel(W4Args a) {
  const int64_t i = static_cast<int64_t>(blockIdx.x) * kW4Threads + threadIdx.x;
  const int row = static_cast<int>(i / a.n), col = static_cast<int>(i % a.n);
  if (row >= a.m) return;
  float v = w4_row_product(a, a.w[0], row, col);
  if constexpr (OUT == kW4Swiglu)
    v = v / (1.0f + __expf(-v)) * w4_row_product(a, a.w[1], row, col);
  if (OUT == kW4Bf16 && a.residual != nullptr)
    v += bf16_to_f32(a.residual[row * a.residual_stride + col]);
  if constexpr (OUT == kW4F32)
    static_cast<float *>(a.y)[row * a.y_stride + col] = v;
  else
    static_cast<uint16_t *>(a.y)[row * a.y_stride + col] = f32_to_bf16(v);
}

template <int OUT>
static int launch_w4(W4Args a, int64_t x_stride, int64_t m, int64_t n, int64_t k,
                     int64_t group, void *stream) {
  if (m <= 0 || n <= 0 || k <= 0) return CASCADE_EINVAL;
  if (k & 7) return CASCADE_EALIGN;
  if ((group != 32 && group != 64 && group != 128) || m > 0x7fffff || n > 0x7fffff ||
      k > 0x7fffff)
    return CASCADE_ESHAPE;
  if (x_stride < 0 || (m > 1 && x_stride < k) || a.y_stride < 0 ||
      (m > 1 && a.y_stride < n) || a.residual_stride < 0)
    return CASCADE_EINVAL;
  if ((x_stride & 7) || !aligned16(a.x)) return CASCADE_EALIGN;
  for (int i = 0; i < (OUT == kW4Swiglu ? 2 : 1); ++i) {
    if (a.w[i].packed == nullptr || a.w[i].scales == nullptr) return CASCADE_EINVAL;
    if (!aligned16(a.w[i].packed) || !aligned16(a.w[i].scales) || !aligned16(a.w[i].zeros))
      return CASCADE_EALIGN;
  }
  if (a.x == nullptr || a.y == nullptr || a.x == a.y) return CASCADE_EINVAL;
  if (OUT == kW4Swiglu && (a.w[0].zeros == nullptr) != (a.w[1].zeros == nullptr))
    return CASCADE_EINVAL;
  if ((reinterpret_cast<uintptr_t>(a.y) & (OUT == kW4F32 ? 3 : 1)) ||
      (reinterpret_cast<uintptr_t>(a.residual) & 1))
    return CASCADE_EALIGN;
  a.x_stride = x_stride;
  a.m = static_cast<int32_t>(m);
  a.n = static_cast<int32_t>(n);
  a.k = static_cast<int32_t>(k);
  a.tiles = static_cast<int32_t>((k + 127) / 128);
  a.group_shift = group == 128 ? 7 : group == 64 ? 6 : 5;
  a.groups = static_cast<int32_t>((k + group - 1) / group);
  const int64_t blocks = (m * n + kW4Threads - 1) / kW4Threads;
  if (blocks > 0xffffffffll / kW4Threads) return CASCADE_ESHAPE;
  return launch_kernel(w4_kernel<OUT>, dim3(static_cast<unsigned>(blocks)), dim3(kW4Threads),
                       0, static_cast<hipStream_t>(stream), a);
}

}  // namespace cascade

using namespace cascade;

extern "C" size_t cascade_linear_w4_workspace_bytes(int64_t, int64_t, int64_t) { return 0; }

extern "C" int cascade_linear_w4_bf16(const void *x, int64_t x_stride, const void *packed,
                                      const void *scales, const void *zeros, int64_t m,
                                      int64_t n, int64_t k, int64_t group,
                                      const void *residual, int64_t residual_stride,
                                      void *y, int64_t y_stride, void *workspace,
                                      size_t workspace_bytes, void *stream) {
  W4Args a{};
  a.x = static_cast<const uint16_t *>(x);
  a.w[0] = {static_cast<const u32x4 *>(packed), static_cast<const uint16_t *>(scales),
            static_cast<const uint8_t *>(zeros)};
  a.residual = static_cast<const uint16_t *>(residual);
  a.residual_stride = residual_stride;
  a.y = y;
  a.y_stride = y_stride;
  return launch_w4<kW4Bf16>(a, x_stride, m, n, k, group, stream);
}

extern "C" int cascade_linear_w4_f32out_bf16(const void *x, int64_t x_stride,
                                             const void *packed, const void *scales,
                                             const void *zeros, int64_t m, int64_t n,
                                             int64_t k, int64_t group, float *y,
                                             int64_t y_stride, void *workspace,
                                             size_t workspace_bytes, void *stream) {
  W4Args a{};
  a.x = static_cast<const uint16_t *>(x);
  a.w[0] = {static_cast<const u32x4 *>(packed), static_cast<const uint16_t *>(scales),
            static_cast<const uint8_t *>(zeros)};
  a.y = y;
  a.y_stride = y_stride;
  return launch_w4<kW4F32>(a, x_stride, m, n, k, group, stream);
}

extern "C" int cascade_gate_up_swiglu_w4_bf16(
    const void *x, int64_t x_stride, const void *gate_packed, const void *gate_scales,
    const void *gate_zeros, const void *up_packed, const void *up_scales,
    const void *up_zeros, int64_t m, int64_t n_half, int64_t k, int64_t group, void *y,
    int64_t y_stride, void *stream) {
  W4Args a{};
  a.x = static_cast<const uint16_t *>(x);
  a.w[0] = {static_cast<const u32x4 *>(gate_packed),
            static_cast<const uint16_t *>(gate_scales),
            static_cast<const uint8_t *>(gate_zeros)};
  a.w[1] = {static_cast<const u32x4 *>(up_packed), static_cast<const uint16_t *>(up_scales),
            static_cast<const uint8_t *>(up_zeros)};
  a.y = y;
  a.y_stride = y_stride;
  return launch_w4<kW4Swiglu>(a, x_stride, m, n_half, k, group, stream);
}
