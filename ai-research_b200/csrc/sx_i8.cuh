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

// A sum as the value it stands for.  (Operations are spelled out here and below: all kernels round alike, so a
// row of a product does not depend on which of them computes it.)
SX_DEV float i8_value(int32_t sum, float x_scale, float w_scale) { return __fmul_rn(__fmul_rn((float)sum, x_scale), w_scale); }
// gelu_tanh(g) * u: g / 2 (1 + tanh z) = g / (1 + e^-2z), z = 0.7978845608 (g + 0.044715 g^3).  The reciprocal is 0 where it
// would be below f32's normal numbers, from a sum of 2^126 on (g below -10): that takes at most 2^-126 |g u| away.  Above,
// e^-2z carries its exponent's rounding: some 9 + 17 |z| steps of 2^-23 in all.
constexpr float kGelu1 = -2.0f * 0.7978845608f * 1.4426950408889634f, kGelu3 = kGelu1 * 0.044715f;  // of g, g^3 in log2 e^-2z
SX_DEV float i8_ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(x));
  return r;
}
SX_DEV float i8_rcp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(x));
  return r;
}
SX_DEV float i8_gated(float g, float u) {
  const float x = __fmul_rn(g, __fmaf_rn(__fmul_rn(g, g), kGelu3, kGelu1));
  return __fmul_rn(__fmul_rn(g, i8_rcp(__fadd_rn(1.0f, i8_ex2(x)))), u);
}
// The same of two neighbours, two operations an instruction
SX_DEV float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n.reg .b64 x, y;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmul.rn.f32x2 x, x, y;\nmov.b64 {%0, %1}, x;\n}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
SX_DEV float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n.reg .b64 x, y;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nadd.rn.f32x2 x, x, y;\nmov.b64 {%0, %1}, x;\n}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
SX_DEV float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n.reg .b64 x, y, z;\nmov.b64 x, {%2, %3};\nmov.b64 y, {%4, %5};\nmov.b64 z, {%6, %7};\n"
      "fma.rn.f32x2 x, x, y, z;\nmov.b64 {%0, %1}, x;\n}\n"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
SX_DEV float2 i8_value2(int32_t s0, int32_t s1, float x_scale, float2 w_scale) {
  return mul2(mul2(make_float2((float)s0, (float)s1), make_float2(x_scale, x_scale)), w_scale);
}
SX_DEV float2 i8_gated2(float2 g, float2 u) {
  const float2 x = mul2(g, fma2(mul2(g, g), make_float2(kGelu3, kGelu3), make_float2(kGelu1, kGelu1)));
  const float2 d = add2(make_float2(1.0f, 1.0f), make_float2(i8_ex2(x.x), i8_ex2(x.y)));
  return mul2(mul2(g, make_float2(i8_rcp(d.x), i8_rcp(d.y))), u);
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
