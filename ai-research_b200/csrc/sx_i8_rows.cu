// sx_i8_rows.cu -- rows to int8 codes, and the norms and residual between two blocks (include/sx.h,
// sx_dispatch_quantize_i8 and sx_dispatch_residual_norm).
//
// A row is read once: each thread holds groups of 8 elements as they came, the row's maximum and sum of squares meet
// in shared memory (or in the row's warp), and what is written comes from registers.  A code is u * (127 / max|u|)
// with u = x * w, which has no sum in it, so codes do not depend on how a row is split over threads.  A NaN or an
// infinity is found in the maximum itself, whose bits are above all others'.
//
// Measured, bound by HBM: seam of 16896 rows of 3840 (f32 stream, bf16 in and out, 12 bytes an element) 135 us, 5.8 TB/s
// or 88 % of the measured copy rate, with L1 77 % busy beside it; into codes 146 us, 75 %; codes of 2697 x 15360 bf16 20 us
// (6.2 TB/s, 95 %), of 16896 x 3840 29 (6.6 TB/s), of f32 with a gain 49 (6.6), of bf16 with one 44 (4.4: registers leave
// eight rows an SM) and of 2697 x 15360 32.5 (3.8: two): instructions and L1 count beside the bytes (bf16 magnitudes one at
// a time took 26.2 and 36 us, codes by conversions 27 and 39; gains read again for the codes 58.6 for f32's 51.4, two rows
// at a time for bf16's no faster).  CTAs that go through rows with the next one on its way were slower (45 us for 39, f32
// 89 for 59: registers), as were a warp for rows of 3840 (45) and more elements a thread.  One row of 3840 takes 1.5 us,
// with a gain 1.9, with both norms 3.0.
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

// 8 elements as they are in memory, and as f32
template <typename T>
struct Raw8 {
  uint4 v[sizeof(T) / 2];
};
template <typename T>
SX_DEV void load_raw(const T *p, Raw8<T> &r) {
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.v[i] = reinterpret_cast<const uint4 *>(p)[i];
}
template <typename T>
SX_DEV void unpack8(const Raw8<T> &r, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
    const uint32_t w[4] = {r.v[i].x, r.v[i].y, r.v[i].z, r.v[i].w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (sizeof(T) == 4) {
        v[4 * i + k] = __uint_as_float(w[k]);
      } else {
        v[2 * k] = __uint_as_float(w[k] << 16);
        v[2 * k + 1] = __uint_as_float(w[k] & 0xFFFF0000u);
      }
    }
  }
}
template <typename T>
SX_DEV void load8(const T *p, float (&v)[8]) {
  Raw8<T> r;
  load_raw(p, r);
  unpack8(r, v);
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
// The same of 4 elements and 4 of 128 elements further, zeros past n: each load of a warp is then one piece of memory.
// (Of 32 bytes a lane L1 takes twice as long: 16896 x 3840 f32 with a gain 51.5 us, so 49.7; 8000 x 8000 55.4 and 51.1.
// bf16 rows, half as many bytes for the same gains, are better off in pieces of 16 bytes: 41 and 42.)
SX_DEV void load_raw_far(const float *p, bool more, Raw8<float> &r) {
  r.v[0] = *reinterpret_cast<const uint4 *>(p);
  r.v[1] = more ? *reinterpret_cast<const uint4 *>(p + 128) : make_uint4(0, 0, 0, 0);
}
// Codes of 8 values: adding 1.5 2^23 rounds a value of up to 127 to a whole number, ties to even, which is then the
// sum's low byte.  mul 0: a row without values, whatever its elements.
SX_DEV uint2 codes_of(const float (&u)[8], float mul) {
  constexpr float kMagic = 12582912.0f;
  uint32_t w[2] = {0, 0};
  if (mul != 0.0f) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      // (products apart: a paired one and the sum after it would become one operation, with one rounding)
      const float2 c = make_float2(kMagic, kMagic);
      const float2 x = add2(make_float2(__fmul_rn(u[4 * h], mul), __fmul_rn(u[4 * h + 1], mul)), c);
      const float2 y = add2(make_float2(__fmul_rn(u[4 * h + 2], mul), __fmul_rn(u[4 * h + 3], mul)), c);
      w[h] = prmt(prmt(__float_as_uint(x.x), __float_as_uint(x.y), 0x0040), prmt(__float_as_uint(y.x), __float_as_uint(y.y), 0x0040), 0x5410);
    }
  }
  return make_uint2(w[0], w[1]);
}
SX_DEV void store_codes(int8_t *p, const float (&u)[8], float mul) { *reinterpret_cast<uint2 *>(p) = codes_of(u, mul); }
SX_DEV void store_codes_far(int8_t *p, bool more, const float (&u)[8], float mul) {
  const uint2 c = codes_of(u, mul);
  *reinterpret_cast<uint32_t *>(p) = c.x;
  if (more) *reinterpret_cast<uint32_t *>(p + 128) = c.y;
}
// the larger of top and |x|, a NaN where there is one
SX_DEV float top_of(float top, float x) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(r) : "f"(top), "f"(fabsf(x)));
  return r;
}

// the larger magnitudes of two bf16s, each of a place
SX_DEV void top_bits(uint32_t &pair, const uint4 &v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) asm("max.u16x2 %0, %0, %1;\n" : "+r"(pair) : "r"(w[i] & 0x7FFF7FFFu));
}

// The largest `top` and the sum of `sum` over the CTA.
struct RowRed {
  uint32_t top[32];
  float sum[32];
};
// WARP: a row has a warp, else the CTA.
template <bool WARP>
SX_DEV void row_reduce(RowRed &red, uint32_t &top, float &sum) {
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  top = __reduce_max_sync(0xffffffffu, top);
  sum = warp_sum(sum);
  if (WARP || warps == 1) return;
  if (lane == 0) {
    red.top[warp] = top;
    red.sum[warp] = sum;
  }
  __syncthreads();
  top = __reduce_max_sync(0xffffffffu, lane < warps ? red.top[lane] : 0u);
  sum = warp_sum(lane < warps ? red.sum[lane] : 0.0f);
}
// This thread's row, its first element and how far its next are
struct Place {
  size_t row;
  uint32_t d0, step;
};
constexpr uint32_t kWarpRows = 8;  // rows of a CTA with WARP
template <bool WARP>
SX_DEV Place place() {
  if (WARP) return {(size_t)blockIdx.x * kWarpRows + (threadIdx.x >> 5), 8 * (threadIdx.x & 31), 8 * 32};
  return {blockIdx.x, 8 * threadIdx.x, 8 * blockDim.x};
}

// 1 / sqrt(mean of squares + eps); a NaN where that is no normal number of f32: a sum of squares that has passed f32 would
// take a row's values away as 0, and below 2^-126 squares are rounded by a 2^-149, which shows in their sum.
SX_DEV float inv_rms(float mean) {
  return __float_as_uint(mean) - 0x00800000u < 0x7F000000u ? 1.0f / sqrtf(mean) : __uint_as_float(0x7FC00000u);
}

// What a row's codes are multiplied by, and its scale (inv: inv_rms with a norm, or 1).
SX_DEV float code_factor(uint32_t top, float sq_sum, float inv, bool norm, float *scale) {
  const float a = __uint_as_float(top);
  if (top >= kInf || (norm && !(sq_sum < INFINITY))) {
    *scale = __uint_as_float(0x7FC00000u);
    return 0.0f;
  }
  *scale = a >= kTiny ? a / 127.0f * inv : 0.0f;
  return a >= kTiny ? 127.0f / a : 0.0f;
}

// G: groups of 8 elements that a thread holds, as they came or with their GAIN; 0: rows too long for registers are
// read again (from L2).  (With 64 registers kMaxThreads fit.  The bound given as threads makes slower code: 2697 x 15360
// with a gain 36.9 us, so 34.8; bf16 32.8, 30.9.)
template <typename T, bool GAIN, bool WARP, uint32_t G>
__global__ void __maxnreg__(64) quantize_i8_kernel(const __grid_constant__ RowsArgs a) {
  __shared__ RowRed red;
  pdl_launch_dependents();
  pdl_wait();
  const Place p = place<WARP>();
  if (WARP && p.row >= a.rows) return;
  constexpr bool kFar = GAIN && sizeof(T) == 4;  // a warp's 256 elements as in load_raw_far
  const uint32_t d0 = kFar ? p.d0 - 4 * (threadIdx.x & 31) : p.d0, step = p.step;
  const T *const in = static_cast<const T *>(a.in) + p.row * a.in_ld;
  int8_t *const q = static_cast<int8_t *>(a.y) + p.row * a.y_ld;
  constexpr uint32_t kHeld = G ? G : 1;
  Raw8<T> raw[kHeld];
  float u[GAIN ? kHeld : 1][8], top = 0.0f, sum = 0.0f;
  // the group at d, from x in v: with its gain, and counted
  auto measure = [&](uint32_t d, float (&v)[8]) {
    if constexpr (GAIN) {
      Raw8<float> raw_w;
      if constexpr (kFar)
        load_raw_far(a.w + d, d + 128 < a.n, raw_w);
      else
        load_raw(a.w + d, raw_w);
      float w[8];
      unpack8(raw_w, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        sum = fmaf(v[i], v[i], sum);
        v[i] = __fmul_rn(v[i], w[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) top = top_of(top, v[i]);
  };
  if constexpr (G > 0) {
#pragma unroll
    for (uint32_t g = 0; g < G; ++g)
      if (d0 + g * step < a.n) {
        if constexpr (kFar)
          load_raw_far(in + d0 + g * step, d0 + g * step + 128 < a.n, raw[g]);
        else
          load_raw(in + d0 + g * step, raw[g]);
      }
    if constexpr (sizeof(T) == 2 && !GAIN) {  // two at a time: the order of bf16's bits is the values' too
      uint32_t pair = 0;
#pragma unroll
      for (uint32_t g = 0; g < G; ++g)
        if (d0 + g * step < a.n) top_bits(pair, raw[g].v[0]);
      top = __uint_as_float(max(pair << 16, pair & 0xFFFF0000u));
    } else {
#pragma unroll
      for (uint32_t g = 0; g < G; ++g)
        if (d0 + g * step < a.n) {
          unpack8(raw[g], u[GAIN ? g : 0]);
          measure(d0 + g * step, u[GAIN ? g : 0]);
        }
    }
  } else {
    for (uint32_t d = d0; d < a.n; d += step) {
      if constexpr (kFar)
        load_raw_far(in + d, d + 128 < a.n, raw[0]);
      else
        load_raw(in + d, raw[0]);
      unpack8(raw[0], u[0]);
      measure(d, u[0]);
    }
  }
  uint32_t bits = __float_as_uint(top) & 0x7FFFFFFFu;  // (their order is the values', with infinity and NaN on top)
  row_reduce<WARP>(red, bits, sum);
  float scale;
  const float inv = GAIN ? inv_rms(sum / (float)a.n + a.eps) : 1.0f;
  const float mul = code_factor(bits, sum, inv, GAIN, &scale);
  if (d0 == 0) a.scale[p.row] = scale;
  if constexpr (G > 0) {
#pragma unroll
    for (uint32_t g = 0; g < G; ++g)
      if (d0 + g * step < a.n) {
        if constexpr (!GAIN) unpack8(raw[g], u[0]);
        if constexpr (kFar)
          store_codes_far(q + d0 + g * step, d0 + g * step + 128 < a.n, u[g], mul);
        else
          store_codes(q + d0 + g * step, u[GAIN ? g : 0], mul);
      }
  } else {
    for (uint32_t d = d0; d < a.n; d += step) {
      if constexpr (kFar)
        load_raw_far(in + d, d + 128 < a.n, raw[0]);
      else
        load_raw(in + d, raw[0]);
      unpack8(raw[0], u[0]);
      measure(d, u[0]);
      if constexpr (kFar)
        store_codes_far(q + d, d + 128 < a.n, u[0], mul);
      else
        store_codes(q + d, u[0], mul);
    }
  }
}

enum RowOut { kOutNone, kOutF32, kOutBf16, kOutI8 };

// (f32 rows with four groups a thread read r again: 64 registers of a row's would leave one CTA an SM)
template <typename T, RowOut OUT, bool WARP, uint32_t G>
__global__ void __launch_bounds__(WARP ? kWarpRows * 32 : kMaxThreads) residual_norm_kernel(const __grid_constant__ RowsArgs a) {
  __shared__ RowRed red[2];
  pdl_launch_dependents();
  pdl_wait();
  const Place p = place<WARP>();
  const size_t row = p.row;
  if (WARP && row >= a.rows) return;
  const T *const r = static_cast<const T *>(a.in) + row * a.in_ld;
  const float *const x = a.x + row * a.x_ld;
  float *const x_out = a.x_out + row * a.x_out_ld;
  const uint32_t d0 = p.d0, step = p.step;
  constexpr uint32_t kHeld = G ? G : 1;
  constexpr bool kAgain = !WARP && G == 4 && sizeof(T) == 4;
  Raw8<T> held[kAgain ? 1 : kHeld];
  float h[8], v[kHeld][8];
  uint32_t bits = 0;
  float top = 0.0f, sum = 0.0f, post = 1.0f;
  if constexpr (G > 0) {
#pragma unroll
    for (uint32_t g = 0; g < G; ++g)
      if (d0 + g * step < a.n) {
        if constexpr (!kAgain) load_raw(r + d0 + g * step, held[g]);
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
        if (d0 + g * step < a.n) {
          if constexpr (kAgain)
            load8(r + d0 + g * step, h);
          else
            unpack8(held[g], h);
          squares(h);
        }
    } else {
      for (uint32_t d = d0; d < a.n; d += step) {
        load8(r + d, h);
        squares(h);
      }
    }
    row_reduce<WARP>(red[0], bits, sum);
    post = inv_rms(sum / (float)a.n + a.eps);
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
      for (int i = 0; i < 8; ++i) top = top_of(top, __fmul_rn(u[i], w[i]));
    }
  };
  if constexpr (G > 0) {
#pragma unroll
    for (uint32_t g = 0; g < G; ++g)
      if (d0 + g * step < a.n) {
        if constexpr (kAgain)
          load8(r + d0 + g * step, h);
        else
          unpack8(held[g], h);
        residual(d0 + g * step, h, v[g]);
      }
  } else {
    for (uint32_t d = d0; d < a.n; d += step) {
      load8(r + d, h);
      load8(x + d, v[0]);
      residual(d, h, v[0]);
    }
  }
  if constexpr (OUT == kOutNone) return;
  bits = __float_as_uint(top) & 0x7FFFFFFFu;
  row_reduce<WARP>(red[1], bits, sum);
  const float inv = inv_rms(sum / (float)a.n + a.eps);
  float mul = 0.0f;
  if constexpr (OUT == kOutI8) {
    float scale;
    mul = code_factor(bits, sum, inv, true, &scale);
    if (d0 == 0) a.scale[row] = scale;
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

// How rows are laid over threads.
struct RowsPlan {
  bool warp;
  uint32_t g, threads, ctas;
};
// Few rows: a CTA each with a thread for every 8 elements, which ends soonest.  Many short ones: a warp each, as CTAs
// start at most one a ns (60000 rows of 256 as CTAs 63 us).  Else a CTA each, up to `most` groups a thread.
RowsPlan rows_plan(uint32_t n, uint32_t rows, uint32_t warp_most, uint32_t most, uint32_t sms) {
  const uint32_t groups = n / 8;
  RowsPlan p{false, 1, 0, rows};
  if (rows > 2 * sms && groups <= 32 * warp_most) {
    p.warp = true;
    while (groups > 32 * p.g) p.g *= 2;
    p.threads = 32 * kWarpRows;
    p.ctas = (rows + kWarpRows - 1) / kWarpRows;
    return p;
  }
  if (rows > 2 * sms && groups > 128) p.g = std::min(rows > 32 * sms || groups > 1024 ? 4u : 2u, most);
  while (p.g < most && groups > p.g * kMaxThreads) p.g *= 2;
  if (groups > p.g * kMaxThreads) p.g = 0;
  const uint32_t each = p.g ? p.g : 1;
  p.threads = std::min(kMaxThreads, ((groups + each - 1) / each + 31) / 32 * 32);
  return p;
}

using RowsKernel = void (*)(const RowsArgs);
template <typename T, bool GAIN>
RowsKernel quantize_kernel(const RowsPlan &p) {
  if (p.warp) {
    if constexpr (sizeof(T) == 2 && !GAIN)
      if (p.g == 8) return quantize_i8_kernel<T, GAIN, true, 8>;
    return p.g == 1 ? quantize_i8_kernel<T, GAIN, true, 1> : p.g == 2 ? quantize_i8_kernel<T, GAIN, true, 2> : quantize_i8_kernel<T, GAIN, true, 4>;
  }
  return p.g == 0 ? quantize_i8_kernel<T, GAIN, false, 0> : p.g == 1 ? quantize_i8_kernel<T, GAIN, false, 1>
       : p.g == 2 ? quantize_i8_kernel<T, GAIN, false, 2> : quantize_i8_kernel<T, GAIN, false, 4>;
}
template <typename T>
RowsKernel quantize_kernel(const RowsPlan &p, bool gain) {
  return gain ? quantize_kernel<T, true>(p) : quantize_kernel<T, false>(p);
}
template <typename T, RowOut OUT>
RowsKernel residual_kernel(const RowsPlan &p) {
  if (p.warp)
    return p.g == 1 ? residual_norm_kernel<T, OUT, true, 1> : p.g == 2 ? residual_norm_kernel<T, OUT, true, 2> : residual_norm_kernel<T, OUT, true, 4>;
  return p.g == 0 ? residual_norm_kernel<T, OUT, false, 0> : p.g == 1 ? residual_norm_kernel<T, OUT, false, 1>
       : p.g == 2 ? residual_norm_kernel<T, OUT, false, 2> : residual_norm_kernel<T, OUT, false, 4>;
}
template <typename T>
RowsKernel residual_kernel(bool none, uint32_t y_dtype, const RowsPlan &p) {
  if (none) return residual_kernel<T, kOutNone>(p);
  return y_dtype == SX_F32 ? residual_kernel<T, kOutF32>(p) : y_dtype == SX_BF16 ? residual_kernel<T, kOutBf16>(p) : residual_kernel<T, kOutI8>(p);
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
  if (a->rows && (!a->x || !a->q || !a->scale)) return bad("null x, q or scale");  // (an empty tensor has no address)
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
  const sx::RowsPlan p = sx::rows_plan(a->n, a->rows, a->dtype == SX_F32 || a->norm_w ? 4 : 8, 4, e->num_sms);
  const sx::RowsKernel k = a->dtype == SX_F32 ? sx::quantize_kernel<float>(p, a->norm_w) : sx::quantize_kernel<__nv_bfloat16>(p, a->norm_w);
  return sx_host_cuda_status(sx::launch_chained(k, dim3(p.ctas), dim3(p.threads), 0, e->stream, 1, r), "quantize_i8 launch");
}

SX_API sx_status sx_dispatch_residual_norm(sx_engine *e, const sx_residual_norm_args *a) {
  auto bad = [](const char *why) {
    sx_host_set_error("residual_norm: %s", why);
    return SX_ERR_INVALID;
  };
  if (!a) return bad("null arguments");
  if (a->r_dtype != SX_F32 && a->r_dtype != SX_BF16) return bad("r_dtype must be SX_F32 or SX_BF16");
  if (a->rows && (!a->x || !a->r || !a->x_out)) return bad("null x, r or x_out");
  if (a->n == 0 || a->n % 16 != 0 || a->n >= sx::kI8MaxK) return bad("n must be a multiple of 16, above 0 and below 131072");
  if (a->x_ld < a->n || a->r_ld < a->n || a->x_out_ld < a->n) return bad("row strides are shorter than a row");
  if (!sx::aligned(a->x, a->x_ld, SX_F32) || !sx::aligned(a->r, a->r_ld, a->r_dtype) || !sx::aligned(a->x_out, a->x_out_ld, SX_F32) ||
      (uintptr_t)a->post_w % 16 != 0)
    return bad("rows and gains must be 16-byte aligned and strides multiples of 16 bytes");
  if (a->rows && a->x_out == a->x && a->x_out_ld != a->x_ld) return bad("x_out may be x with the same stride only");
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
  const sx::RowsPlan p = sx::rows_plan(a->n, a->rows, 4, a->n > 8192 ? 4 : 2, e->num_sms);
  return sx_host_cuda_status(
      sx::launch_chained(a->r_dtype == SX_F32 ? sx::residual_kernel<float>(none, a->y_dtype, p) : sx::residual_kernel<__nv_bfloat16>(none, a->y_dtype, p),
                         dim3(p.ctas), dim3(p.threads), 0, e->stream, 1, r),
      "residual_norm launch");
}

}  // extern "C"
