// sx_i8_rows.cu -- rows to int8 codes, and the norms and residual between two blocks (include/sx.h,
// sx_dispatch_quantize_i8 and sx_dispatch_residual_norm).
//
// A row is read once: each thread holds groups of 8 elements, the row's maximum and sum of squares meet
// in shared memory, and what is written comes from registers.  A code is u * (127 / max|u|) with u = x * w,
// which has no sum in it, so codes do not depend on how a row is split over threads.
#include "sx_host.h"
#include "sx_i8.cuh"
#include "sx_kv8.cuh"
#include "sx_launch.cuh"

namespace sx {
namespace {

constexpr uint32_t kInf = 0x7F800000u;
constexpr float kTiny = 7.88860905e-31f;  // 2^-100
constexpr uint32_t kMaxThreads = 1024;

struct RowsArgs {
  const void *in;       // quantize: x; residual_norm: r
  const float *x;       // residual_norm: the residual
  const float *post_w, *w;
  float *x_out;
  void *y;
  float *scale;
  uint32_t in_ld, x_ld, x_out_ld, y_ld, rows, n;
  float scalar, eps;
};

template <typename T>
SX_DEV void load8(const T *p, float (&v)[8]) {
  if constexpr (sizeof(T) == 2) {
    load_vec<T, 8>(p, v);
  } else {
    float a[4], b[4];
    load_vec<T, 4>(p, a);
    load_vec<T, 4>(p + 4, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = a[i];
      v[4 + i] = b[i];
    }
  }
}
template <typename T>
SX_DEV void store8(T *p, const float (&v)[8]) {
  if constexpr (sizeof(T) == 2) {
    store_vec<T, 8>(p, v);
  } else {
    const float a[4] = {v[0], v[1], v[2], v[3]}, b[4] = {v[4], v[5], v[6], v[7]};
    store_vec<T, 4>(p, a);
    store_vec<T, 4>(p + 4, b);
  }
}
SX_DEV void store_codes(int8_t *p, const float (&u)[8], float mul) {
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    w[h] = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[h] |= ((uint32_t)__float2int_rn(__fmul_rn(u[4 * h + i], mul)) & 0xFFu) << (8 * i);
  }
  *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
}

// The largest `top` and the sum of `sum` over the CTA.
struct RowRed {
  uint32_t top[32];
  float sum[32];
};
SX_DEV void row_reduce(RowRed &red, uint32_t &top, float &sum) {
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  top = __reduce_max_sync(0xffffffffu, top);
  sum = warp_sum(sum);
  if (warps == 1) return;
  if (lane == 0) {
    red.top[warp] = top;
    red.sum[warp] = sum;
  }
  __syncthreads();
  top = __reduce_max_sync(0xffffffffu, lane < warps ? red.top[lane] : 0u);
  sum = warp_sum(lane < warps ? red.sum[lane] : 0.0f);
}

// What a row's codes are multiplied by, and its scale.
SX_DEV float code_factor(uint32_t top, float sq_sum, float inv, bool norm, float *scale) {
  const float a = __uint_as_float(top);
  if (top >= kInf || (norm && !(sq_sum < INFINITY))) {
    *scale = __uint_as_float(0x7FC00000u);
    return 0.0f;
  }
  *scale = a >= kTiny ? a / 127.0f * inv : 0.0f;
  return a >= kTiny ? 127.0f / a : 0.0f;
}

// G: groups of 8 elements that a thread holds; 0: rows too long for registers are read again (from L2).
template <typename T, uint32_t G>
__global__ void __launch_bounds__(kMaxThreads) quantize_i8_kernel(const __grid_constant__ RowsArgs a) {
  __shared__ RowRed red;
  pdl_launch_dependents();
  pdl_wait();
  const size_t row = blockIdx.x;
  const T *const in = static_cast<const T *>(a.in) + row * a.in_ld;
  int8_t *const q = static_cast<int8_t *>(a.y) + row * a.y_ld;
  uint32_t top = 0;
  float sum = 0.0f;
  // u of a group, from x there
  auto gained = [&](uint32_t d, float (&u)[8]) {
    if (!a.w) return;
    float w[8];
    load8(a.w + d, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = __fmul_rn(u[i], w[i]);
  };
  auto measure = [&](uint32_t d, float (&u)[8]) {
    if (a.w)
#pragma unroll
      for (int i = 0; i < 8; ++i) sum = fmaf(u[i], u[i], sum);
    gained(d, u);
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(u[i]) & 0x7FFFFFFFu);
  };
  const uint32_t d0 = 8 * threadIdx.x, step = 8 * blockDim.x;
  float u[G ? G : 1][8];
  if constexpr (G > 0) {
#pragma unroll
    for (uint32_t g = 0; g < G; ++g)
      if (d0 + g * step < a.n) load8(in + d0 + g * step, u[g]);
#pragma unroll
    for (uint32_t g = 0; g < G; ++g)
      if (d0 + g * step < a.n) measure(d0 + g * step, u[g]);
  } else {
    for (uint32_t d = d0; d < a.n; d += step) {
      load8(in + d, u[0]);
      measure(d, u[0]);
    }
  }
  row_reduce(red, top, sum);
  float scale;
  const float inv = a.w ? 1.0f / sqrtf(sum / (float)a.n + a.eps) : 1.0f;
  const float mul = code_factor(top, sum, inv, a.w != nullptr, &scale);
  if (threadIdx.x == 0) a.scale[row] = scale;
  if constexpr (G > 0) {
#pragma unroll
    for (uint32_t g = 0; g < G; ++g)
      if (d0 + g * step < a.n) store_codes(q + d0 + g * step, u[g], mul);
  } else {
    for (uint32_t d = d0; d < a.n; d += step) {
      load8(in + d, u[0]);
      gained(d, u[0]);
      store_codes(q + d, u[0], mul);
    }
  }
}

enum RowOut { kOutNone, kOutF32, kOutBf16, kOutI8 };

template <typename T, RowOut OUT, uint32_t G>
__global__ void __launch_bounds__(kMaxThreads) residual_norm_kernel(const __grid_constant__ RowsArgs a) {
  __shared__ RowRed red[2];
  pdl_launch_dependents();
  pdl_wait();
  const size_t row = blockIdx.x;
  const T *const r = static_cast<const T *>(a.in) + row * a.in_ld;
  const float *const x = a.x + row * a.x_ld;
  float *const x_out = a.x_out + row * a.x_out_ld;
  const uint32_t d0 = 8 * threadIdx.x, step = 8 * blockDim.x;
  constexpr uint32_t kHeld = G ? G : 1;
  float h[kHeld][8], v[kHeld][8];
  uint32_t top = 0;
  float sum = 0.0f, post = 1.0f;
  if constexpr (G > 0) {
#pragma unroll
    for (uint32_t g = 0; g < G; ++g)
      if (d0 + g * step < a.n) {
        load8(r + d0 + g * step, h[g]);
        load8(x + d0 + g * step, v[g]);
      }
  }
  auto squares = [&](const float (&u)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = fmaf(u[i], u[i], sum);
  };
  if (a.post_w) {
    if constexpr (G > 0) {
#pragma unroll
      for (uint32_t g = 0; g < G; ++g)
        if (d0 + g * step < a.n) squares(h[g]);
    } else {
      for (uint32_t d = d0; d < a.n; d += step) {
        load8(r + d, h[0]);
        squares(h[0]);
      }
    }
    row_reduce(red[0], top, sum);
    post = 1.0f / sqrtf(sum / (float)a.n + a.eps);
    sum = 0.0f;
  }
  // the new residual of a group in u, from x there
  auto residual = [&](uint32_t d, const float (&t)[8], float (&u)[8]) {
    float w[8];
    if (a.post_w) load8(a.post_w + d, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = (u[i] + (a.post_w ? t[i] * post * w[i] : t[i])) * a.scalar;
    store8(x_out + d, u);
    squares(u);
    if constexpr (OUT == kOutI8) {
      load8(a.w + d, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(__fmul_rn(u[i], w[i])) & 0x7FFFFFFFu);
    }
  };
  if constexpr (G > 0) {
#pragma unroll
    for (uint32_t g = 0; g < G; ++g)
      if (d0 + g * step < a.n) residual(d0 + g * step, h[g], v[g]);
  } else {
    for (uint32_t d = d0; d < a.n; d += step) {
      load8(r + d, h[0]);
      load8(x + d, v[0]);
      residual(d, h[0], v[0]);
    }
  }
  if constexpr (OUT == kOutNone) return;
  row_reduce(red[1], top, sum);
  const float inv = 1.0f / sqrtf(sum / (float)a.n + a.eps);
  float mul = 0.0f;
  if constexpr (OUT == kOutI8) {
    float scale;
    mul = code_factor(top, sum, inv, true, &scale);
    if (threadIdx.x == 0) a.scale[row] = scale;
  }
  auto normed = [&](uint32_t d, float (&u)[8]) {
    float w[8];
    load8(a.w + d, w);
    if constexpr (OUT == kOutI8) {
#pragma unroll
      for (int i = 0; i < 8; ++i) u[i] = __fmul_rn(u[i], w[i]);
      store_codes(static_cast<int8_t *>(a.y) + row * a.y_ld + d, u, mul);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) u[i] = u[i] * inv * w[i];
      if constexpr (OUT == kOutF32)
        store8(static_cast<float *>(a.y) + row * a.y_ld + d, u);
      else
        store8(static_cast<__nv_bfloat16 *>(a.y) + row * a.y_ld + d, u);
    }
  };
  if constexpr (G > 0) {
#pragma unroll
    for (uint32_t g = 0; g < G; ++g)
      if (d0 + g * step < a.n) normed(d0 + g * step, v[g]);
  } else {
    for (uint32_t d = d0; d < a.n; d += step) {
      load8(x_out + d, v[0]);
      normed(d, v[0]);
    }
  }
}

using RowsKernel = void (*)(const RowsArgs);

// Groups of 8 that a thread holds: one where rows are few (more threads end sooner), else up to `most`; 0 past
// kMaxThreads times that.
uint32_t groups_of(uint32_t n, uint32_t rows, uint32_t most, uint32_t sms) {
  const uint32_t groups = n / 8;
  uint32_t g = rows <= 2 * sms || groups <= 32 ? 1 : most;
  while (g < most && groups > g * kMaxThreads) g *= 2;
  return groups > g * kMaxThreads ? 0 : g;
}
cudaError_t launch_rows(RowsKernel k, const RowsArgs &a, uint32_t g, cudaStream_t s) {
  const uint32_t each = 8 * (g ? g : 1), threads = std::min(kMaxThreads, ((a.n + each - 1) / each + 31) / 32 * 32);
  return launch_chained(k, dim3(a.rows), dim3(threads), 0, s, 1, a);
}

template <typename T>
RowsKernel quantize_kernel(uint32_t g) {
  return g == 0 ? quantize_i8_kernel<T, 0> : g == 1 ? quantize_i8_kernel<T, 1> : g == 2 ? quantize_i8_kernel<T, 2> : quantize_i8_kernel<T, 4>;
}
template <typename T, RowOut OUT>
RowsKernel residual_kernel(uint32_t g) {
  return g == 0 ? residual_norm_kernel<T, OUT, 0> : g == 1 ? residual_norm_kernel<T, OUT, 1> : residual_norm_kernel<T, OUT, 2>;
}
template <typename T>
RowsKernel residual_kernel(bool none, uint32_t y_dtype, uint32_t g) {
  if (none) return residual_kernel<T, kOutNone>(g);
  return y_dtype == SX_F32 ? residual_kernel<T, kOutF32>(g) : y_dtype == SX_BF16 ? residual_kernel<T, kOutBf16>(g) : residual_kernel<T, kOutI8>(g);
}

uint32_t bytes_of(uint32_t dtype) { return dtype == SX_F32 ? 4 : dtype == SX_BF16 ? 2 : 1; }
// rows that 16-byte pieces may be taken of
bool aligned(const void *p, uint32_t ld, uint32_t dtype) { return ((uintptr_t)p | (uintptr_t)ld * bytes_of(dtype)) % 16 == 0; }

}  // namespace
}  // namespace sx

extern "C" {

SX_API sx_status sx_dispatch_quantize_i8(sx_engine *e, const sx_quantize_i8_args *a) {
  auto bad = [](const char *why) {
    sx_host_set_error("quantize_i8: %s", why);
    return SX_ERR_INVALID;
  };
  if (!a) return bad("null arguments");
  if (a->dtype != SX_F32 && a->dtype != SX_BF16) return bad("dtype must be SX_F32 or SX_BF16");
  if (!a->x || !a->q || !a->scale) return bad("null x, q or scale");
  if (a->n == 0 || a->n % 16 != 0 || a->n >= sx::kI8MaxK) return bad("n must be a multiple of 16, above 0 and below 131072");
  if (a->x_ld < a->n || a->q_ld < a->n) return bad("row strides are shorter than a row");
  if (!sx::aligned(a->x, a->x_ld, a->dtype) || !sx::aligned(a->q, a->q_ld, SX_I8) || (uintptr_t)a->norm_w % 16 != 0)
    return bad("x, q and norm_w must be 16-byte aligned and strides multiples of 16 bytes");
  if ((uintptr_t)a->scale % 4 != 0) return bad("scale must be aligned to its elements");
  if (a->norm_w && !(a->eps >= 0.0f)) return bad("eps must not be negative");
  if (a->rows >= (1u << 31)) return bad("too many rows");
  if (!e) return bad("null engine");
  if (a->rows == 0) return SX_OK;
  const cudaError_t ce = cudaSetDevice(e->device);
  if (ce != cudaSuccess) return sx_host_cuda_status(ce, "cudaSetDevice");
  sx::RowsArgs r{};
  r.in = a->x;
  r.w = a->norm_w;
  r.y = a->q;
  r.scale = a->scale;
  r.in_ld = a->x_ld;
  r.y_ld = a->q_ld;
  r.rows = a->rows;
  r.n = a->n;
  r.eps = a->eps;
  const uint32_t g = sx::groups_of(a->n, a->rows, 4, e->num_sms);
  return sx_host_cuda_status(
      sx::launch_rows(a->dtype == SX_F32 ? sx::quantize_kernel<float>(g) : sx::quantize_kernel<__nv_bfloat16>(g), r, g, e->stream),
      "quantize_i8 launch");
}

SX_API sx_status sx_dispatch_residual_norm(sx_engine *e, const sx_residual_norm_args *a) {
  auto bad = [](const char *why) {
    sx_host_set_error("residual_norm: %s", why);
    return SX_ERR_INVALID;
  };
  if (!a) return bad("null arguments");
  if (a->r_dtype != SX_F32 && a->r_dtype != SX_BF16) return bad("r_dtype must be SX_F32 or SX_BF16");
  if (!a->x || !a->r || !a->x_out) return bad("null x, r or x_out");
  if (a->n == 0 || a->n % 16 != 0 || a->n >= sx::kI8MaxK) return bad("n must be a multiple of 16, above 0 and below 131072");
  if (a->x_ld < a->n || a->r_ld < a->n || a->x_out_ld < a->n) return bad("row strides are shorter than a row");
  if (!sx::aligned(a->x, a->x_ld, SX_F32) || !sx::aligned(a->r, a->r_ld, a->r_dtype) || !sx::aligned(a->x_out, a->x_out_ld, SX_F32) ||
      (uintptr_t)a->post_w % 16 != 0)
    return bad("rows and gains must be 16-byte aligned and strides multiples of 16 bytes");
  if (a->x_out == a->x && a->x_out_ld != a->x_ld) return bad("x_out may be x with the same stride only");
  if (a->y) {
    if (a->y_dtype != SX_F32 && a->y_dtype != SX_BF16 && a->y_dtype != SX_I8) return bad("y_dtype must be SX_F32, SX_BF16 or SX_I8");
    if (!a->pre_w) return bad("null pre_w");
    if (a->y_ld < a->n) return bad("row strides are shorter than a row");
    if (!sx::aligned(a->y, a->y_ld, a->y_dtype) || (uintptr_t)a->pre_w % 16 != 0)
      return bad("rows and gains must be 16-byte aligned and strides multiples of 16 bytes");
    if ((a->y_dtype == SX_I8) != (a->y_scale != nullptr)) return bad("y_scale belongs to SX_I8");
    if ((uintptr_t)a->y_scale % 4 != 0) return bad("y_scale must be aligned to its elements");
  }
  if ((a->post_w || a->y) && !(a->eps >= 0.0f)) return bad("eps must not be negative");
  if (a->rows >= (1u << 31)) return bad("too many rows");
  if (!e) return bad("null engine");
  if (a->rows == 0) return SX_OK;
  const cudaError_t ce = cudaSetDevice(e->device);
  if (ce != cudaSuccess) return sx_host_cuda_status(ce, "cudaSetDevice");
  sx::RowsArgs r{};
  r.in = a->r;
  r.x = a->x;
  r.post_w = a->post_w;
  r.w = a->pre_w;
  r.x_out = a->x_out;
  r.y = a->y;
  r.scale = a->y_scale;
  r.in_ld = a->r_ld;
  r.x_ld = a->x_ld;
  r.x_out_ld = a->x_out_ld;
  r.y_ld = a->y_ld;
  r.rows = a->rows;
  r.n = a->n;
  r.scalar = a->scalar;
  r.eps = a->eps;
  const bool none = a->y == nullptr;
  const uint32_t g = sx::groups_of(a->n, a->rows, 2, e->num_sms);
  return sx_host_cuda_status(
      sx::launch_rows(a->r_dtype == SX_F32 ? sx::residual_kernel<float>(none, a->y_dtype, g) : sx::residual_kernel<__nv_bfloat16>(none, a->y_dtype, g),
                      r, g, e->stream),
      "residual_norm launch");
}

}  // extern "C"
