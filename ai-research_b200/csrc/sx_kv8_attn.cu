// sx_kv8_attn.cu -- attention over the paged 8-bit KV cache (include/sx.h, sx_dispatch_kv8_attn).
//
//   out_r = sum_j p_j V_j,  p = softmax_j(scale q_r . K_j),  j <= pos(r), j > pos(r) - window
//
// One warp per row and q head walks the row's keys with a running maximum and sum.
#include "sx_host.h"
#include "sx_kv8.cuh"

namespace sx {
namespace {

struct Kv8AttnArgs {
  sx_kv8 c;
  const void *q;
  void *out;
  uint32_t q_ld, out_ld;
  const uint32_t *row_start, *kv_len;
  uint32_t tokens, num_q, window;
  float scale;
  uint32_t *err;
};

template <typename T, int D>
__global__ void __launch_bounds__(128) kv8_attn_kernel(Kv8AttnArgs a) {
  constexpr int kPer = D / 32;
  const int lane = threadIdx.x & 31;
  const uint32_t t = blockIdx.x, h = blockIdx.y * 4 + (threadIdx.x >> 5);
  if (h >= a.num_q) return;
  const uint32_t b = warp_last_le(a.c.num_seqs, t, [&](uint32_t i) { return a.row_start[i]; });
  Kv8Rows r;
  if (!kv8_rows(a.c, a.row_start, a.kv_len, a.tokens, b, &r)) {
    if (lane == 0) raise_error(a.err, kDevBadParams);
    return;
  }
  if (t < r.r0 || t >= r.r0 + r.n) return;
  const uint32_t pos = r.len - r.n + (t - r.r0), kvh = h / (a.num_q / a.c.num_kv);
  const uint32_t j0 = a.window && pos >= a.window ? pos - a.window + 1 : 0;
  const T *q = static_cast<const T *>(a.q) + (size_t)t * a.q_ld + (size_t)h * D;
  float qr[kPer], o[kPer], m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    qr[i] = (float)q[32 * i + lane];
    o[i] = 0.0f;
  }
  for (uint32_t j = j0; j <= pos; ++j) {
    const uint32_t page = a.c.table[(size_t)b * a.c.max_pages + j / a.c.page_tokens];
    if (page >= a.c.num_pages) {
      if (lane == 0) raise_error(a.err, kDevBadSlot);
      continue;
    }
    const size_t rec = (((size_t)page * a.c.num_kv + kvh) * (a.c.page_tokens / 16) + j % a.c.page_tokens / 16) * 2;
    const uint8_t *k = static_cast<const uint8_t *>(a.c.data) + rec * (16 * D);
    const uint32_t s = j % 16;
    float part = 0.0f, v[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const uint32_t e = lane;
      const uint32_t kb = k[512 * i + 16 * (4 * (s % 8) + e / 8) + 8 * (s / 8) + e % 8];
      const uint32_t vb = k[16 * D + 512 * i + 16 * (4 * (e / 4) + s % 8 / 2) + 4 * (e % 4) + s % 2 + 2 * (s / 8)];
      const float2 f = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(kb | vb << 8), __NV_E4M3)));
      part = fmaf(qr[i], f.x, part);
      v[i] = f.y;
    }
    const float z = warp_sum(part) * a.c.scale[rec] * a.scale;
    const float mn = fmaxf(m, z), corr = m == -INFINITY ? 0.0f : expf(m - mn);
    const float p = expf(z - mn), pv = p * a.c.scale[rec + 1];
    l = fmaf(l, corr, p);
#pragma unroll
    for (int i = 0; i < kPer; ++i) o[i] = fmaf(o[i], corr, pv * v[i]);
    m = mn;
  }
  T *out = static_cast<T *>(a.out) + (size_t)t * a.out_ld + (size_t)h * D;
#pragma unroll
  for (int i = 0; i < kPer; ++i) out[32 * i + lane] = (T)(l == 0.0f ? 0.0f : o[i] / l);
}

using AttnKernel = void (*)(Kv8AttnArgs);
AttnKernel attn_kernel(sx_dtype t, uint32_t d) {
  if (t == SX_F32)
    return d == 64 ? kv8_attn_kernel<float, 64> : d == 128 ? kv8_attn_kernel<float, 128>
         : d == 256 ? kv8_attn_kernel<float, 256> : kv8_attn_kernel<float, 512>;
  return d == 64 ? kv8_attn_kernel<__nv_bfloat16, 64> : d == 128 ? kv8_attn_kernel<__nv_bfloat16, 128>
       : d == 256 ? kv8_attn_kernel<__nv_bfloat16, 256> : kv8_attn_kernel<__nv_bfloat16, 512>;
}

}  // namespace
}  // namespace sx

extern "C" SX_API sx_status sx_dispatch_kv8_attn(sx_engine *e, const sx_kv8 *c, sx_dtype t,
                                                 const void *q, void *out, uint32_t q_ld,
                                                 uint32_t out_ld, const uint32_t *row_start,
                                                 const uint32_t *kv_len, uint32_t tokens,
                                                 uint32_t num_q, uint32_t window, float scale) {
  auto bad = [](const char *why) {
    sx_host_set_error("kv8_attn: %s", why);
    return SX_ERR_INVALID;
  };
  if (!e) return bad("null engine");
  sx_status st = sx_host_check_kv8("kv8_attn", c, t, num_q);
  if (st != SX_OK) return st;
  if (!q || !out || !row_start || !kv_len) return bad("null q, out, row_start or kv_len");
  if (num_q == 0) return bad("num_q must be above 0");
  const uint32_t es = t == SX_F32 ? 4 : 2, row = num_q * c->head_dim;
  if (q_ld < row || out_ld < row) return bad("row strides are shorter than a row");
  if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)q_ld * es | (uintptr_t)out_ld * es) % 16 != 0)
    return bad("vectors must be 16-byte aligned and strides multiples of 16 bytes");
  if (tokens >= (1u << 30)) return bad("too many rows");
  if (tokens == 0 || c->num_seqs == 0) return SX_OK;
  cudaError_t ce = cudaSetDevice(e->device);
  if (ce != cudaSuccess) return sx_host_cuda_status(ce, "cudaSetDevice");
  sx::Kv8AttnArgs a{*c, q, out, q_ld, out_ld, row_start, kv_len, tokens, num_q, window, scale, e->err_dev};
  sx::attn_kernel(t, c->head_dim)<<<dim3(tokens, (num_q + 3) / 4), 128, 0, e->stream>>>(a);
  return sx_host_cuda_status(cudaGetLastError(), "kv8_attn launch");
}
