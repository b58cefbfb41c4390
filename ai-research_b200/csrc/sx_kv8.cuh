// sx_kv8.cuh -- the paged 8-bit KV cache on the device: layout, scales, rows of a ragged batch.
//
// Every 16 tokens of one kv head are a K and a V record of 16 * head_dim e4m3 bytes, each with a
// power-of-two scale (include/sx.h, sx_kv8).  A record is cut into 512-byte pieces of 32 elements;
// lane l = 4 g + c of a warp owns the 16 bytes at 16 l of each piece, which are the A operand of
// two mma.m16n8k16:
//   K (rows = tokens):   tokens g and g + 8, elements 8 c .. 8 c + 7 of the piece
//   V (rows = elements): elements 4 g .. 4 g + 3 of the piece, tokens 2 c, 2 c + 1, 2 c + 8, 2 c + 9
// so a warp's 16-byte loads are coalesced and no shuffle or transposition follows them.
#pragma once

#include <cuda_fp8.h>

#include "../../include/sx.h"
#include "sx_common.cuh"
#include "sx_kv8_units.h"

namespace sx {

constexpr int kKv8MinExp = -60, kKv8MaxExp = 60;
constexpr uint32_t kKv8MaxSeqs = 4096;

// Rows of sequence b; false when they do not fit.
SX_DEV bool kv8_rows(const sx_kv8 &c, const uint32_t *row_start, const uint32_t *kv_len,
                     uint32_t tokens, uint32_t b, Kv8Rows *r) {
  return kv8_rows_fit(row_start[b], row_start[b + 1], kv_len[b], tokens, c.max_pages * c.page_tokens, r);
}

// The last b < n with key(b) <= u (0 if there is none); key rises with b.  A whole warp calls it:
// 32 probes at a time, so 4096 sequences take three rounds of loads.
template <typename Key>
SX_DEV uint32_t warp_last_le(uint32_t n, uint32_t u, Key key) {
  const uint32_t lane = threadIdx.x & 31;
  uint32_t lo = 0;
  while (n > 1) {
    const uint32_t step = (n + 31) / 32;
    const uint32_t at = step * lane;
    const uint32_t k = __popc(__ballot_sync(0xffffffffu, at < n && key(lo + at) <= u));
    const uint32_t skip = k ? step * (k - 1) : 0;
    lo += skip;
    n = min(step, n - skip);
  }
  return lo;
}

// The smallest e with amax <= 448 * 2^e (448 = 1.75 * 2^8), within the scales' range.
SX_DEV int kv8_exponent(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  return min(max(e, kKv8MinExp), kKv8MaxExp);
}
SX_DEV int kv8_scale_exponent(float scale) {
  const int e = (int)((__float_as_uint(scale) >> 23) & 255u) - 127;
  return min(max(e, kKv8MinExp), kKv8MaxExp);
}
SX_DEV float exp2_int(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// four e4m3 bytes <-> four f32 (round to nearest even, saturating; NaN stays NaN)
SX_DEV uint32_t e4m3_pack4(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | hi << 16;
}
// four e4m3 bytes -> two f16x2 (exact).  The conversion takes a register's half as it is: half a
// cycle per SM and pair, against 1.5 when the half is first cut out in 32 bits.
SX_DEV void e4m3x4_f16(uint32_t w, uint32_t &lo, uint32_t &hi) {
  asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %2;\n cvt.rn.f16x2.e4m3x2 %0, l;\n"
      " cvt.rn.f16x2.e4m3x2 %1, h;\n}\n"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}
SX_DEV float4 e4m3_unpack4(uint32_t w) {
  const __half2_raw lo = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xFFFFu), __NV_E4M3);
  const __half2_raw hi = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3);
  const float2 a = __half22float2(__half2(lo)), b = __half22float2(__half2(hi));
  return make_float4(a.x, a.y, b.x, b.y);
}

// VEC consecutive elements of a vector in memory as f32, and back
template <typename T, int VEC>
SX_DEV void load_vec(const T *p, float (&v)[VEC]) {
  constexpr int kBytes = VEC * (int)sizeof(T);
  uint32_t w[(kBytes + 3) / 4];
  if constexpr (kBytes == 16) {
    const uint4 u = *reinterpret_cast<const uint4 *>(p);
    w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
  } else if constexpr (kBytes == 8) {
    const uint2 u = *reinterpret_cast<const uint2 *>(p);
    w[0] = u.x; w[1] = u.y;
  } else {
    static_assert(kBytes == 4, "4, 8 or 16 bytes");
    w[0] = *reinterpret_cast<const uint32_t *>(p);
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    if constexpr (sizeof(T) == 4)
      v[i] = __uint_as_float(w[i]);
    else
      v[i] = __uint_as_float(i & 1 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
  }
}
template <typename T, int VEC>
SX_DEV void store_vec(T *p, const float (&v)[VEC]) {
  constexpr int kBytes = VEC * (int)sizeof(T);
  uint32_t w[(kBytes + 3) / 4];
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) w[i] = __float_as_uint(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t *>(&b);
    }
  }
  if constexpr (kBytes == 16)
    *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  else if constexpr (kBytes == 8)
    *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
  else
    *reinterpret_cast<uint32_t *>(p) = w[0];
}

// ---- attention
constexpr float kLog2e = 1.4426950408889634f;

struct Kv8AttnArgs {
  sx_kv8 c;
  const void *q;
  void *out;
  uint32_t q_ld, out_ld;
  const uint32_t *row_start, *kv_len;
  uint32_t tokens, num_q, window, gqa, min_run;
  float scale;
  float *part;      // parts of split problems: [2 grid][rows] x {m, l}, then [2 grid][rows][D]
  uint32_t *cnt;    // [grid], zero at rest
  uint32_t *err;
};

SX_DEV float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(x));
  return r;
}
SX_DEV uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t *>(&h);
}
// what f16 rounding left of the pair
SX_DEV uint32_t pack_f16_rest(float lo, float hi, uint32_t rounded) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&rounded));
  return pack_f16(lo - f.x, hi - f.y);
}

// Count an arrival on behalf of a CTA whose threads met at a barrier before: their writes are
// released by it, and those of the CTAs counted before are acquired.
SX_DEV uint32_t arrive_acq_rel(uint32_t *cnt) {
  uint32_t r;
  asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;\n" : "=r"(r) : "l"(cnt) : "memory");
  return r;
}
cudaError_t launch_kv8_prompt(Kv8AttnArgs a, sx_dtype t, int num_sms, cudaStream_t s);

}  // namespace sx
