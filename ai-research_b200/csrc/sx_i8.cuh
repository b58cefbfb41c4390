// sx_i8.cuh -- products of int8 rows: arguments and what their kernels share (include/sx.h).
#pragma once

#include "../../include/sx.h"
#include "sx_common.cuh"

namespace sx {

constexpr uint32_t kI8MaxK = 131072;  // 128 * 128 * (kI8MaxK - 16) < 2^31

// gemm_i8, or gate_up_i8 with a second matrix.
struct I8Args {
  const int8_t *x, *w[2];
  const float *x_scale, *w_scale[2];
  void *y;
  uint32_t x_ld, w_ld, y_ld, t, n, k;
  uint32_t *err;
};

// A sum as the value it stands for.
SX_DEV float i8_value(int32_t sum, float x_scale, float w_scale) { return (float)sum * x_scale * w_scale; }
// gelu_tanh(g) * u: g / 2 (1 + tanh z) = g / (1 + e^-2z), whose e^-2z overflows where the value is 0 in f32
SX_DEV float i8_gated(float g, float u) {
  const float z = 0.7978845608f * (g + 0.044715f * g * g * g);
  return __fdividef(g, 1.0f + __expf(-2.0f * z)) * u;
}

template <typename T>
SX_DEV T i8_out(float v);
template <>
SX_DEV float i8_out<float>(float v) { return v; }
template <>
SX_DEV __nv_bfloat16 i8_out<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

constexpr uint32_t kI8GemvRows = 16;  // up to which the weights are streamed
cudaError_t prepare_gemv_i8();
cudaError_t launch_gemv_i8(uint32_t dtype, bool gated, const I8Args &a, int num_sms, cudaStream_t s);

}  // namespace sx
