// sx_kv8_append.cu -- new rows into the paged 8-bit KV cache: q / k RMS norm, position rotation,
// e4m3 quantisation with one power-of-two scale per 16 tokens and kv head (include/sx.h,
// sx_dispatch_kv8_append).
//
//   q', k' = R(pos) (x / rms(x) * gain),  v' = v / rms(v),  stored = rn_e4m3(x' 2^-e),
//   e = min { e : max |record| <= 448 2^e }
//
// A record belongs to one CTA, which sees all of its new tokens, so the scale needs no atomics:
// unit u is one 16-token block of one sequence, a CTA takes one unit and a group of kv heads with
// their q heads.  The angles of a unit's tokens are computed once and kept in shared memory.
// With sequence b's rows at row_start[b], units row_start[b] / 16 + 2 b .. belong to it: n rows
// touch at most n / 16 + 2 blocks, so the grid follows from the row and sequence counts alone and
// nothing is read back.
#include "sx_host.h"
#include "sx_kv8.cuh"

namespace sx {
namespace {

constexpr int kAppWarps = 8;

struct AppendArgs {
  sx_kv8 c;
  const void *q, *k, *v;
  uint32_t q_ld, k_ld, v_ld;
  const float *q_w, *k_w;
  void *q_out;
  const uint32_t *row_start, *kv_len;
  uint32_t tokens, gqa, rot, k_eq_v, v_norm, heads_per_cta;
  const float *inv_freq;
  float eps;
  uint32_t *err;
};

// x / rms(x) * w, in the engine's order of operations (qkv_rope)
template <int N>
SX_DEV void normalise(float (&x)[N], float eps, uint32_t dim) {
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) ss = fmaf(x[i], x[i], ss);
  ss = warp_sum(ss);
  const float rs = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(ss, (float)dim), eps)));
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = __fmul_rn(x[i], rs);
}

template <typename T, int D>
__global__ void __launch_bounds__(kAppWarps * 32) kv8_append_kernel(AppendArgs a) {
  constexpr int kPer = D / 32;                                  // elements of a vector per lane
  constexpr int kVec = kPer < 16 / (int)sizeof(T) ? kPer : 16 / (int)sizeof(T);
  constexpr int kLd = D + 4;  // tile row stride: the 16-byte reads below hit all banks once
  extern __shared__ float sh[];
  __shared__ float amax[2][kKv8Block];
  float *tile = sh;                                             // [2][16][kLd]; q rows: [warps][D]
  float2 *cs = reinterpret_cast<float2 *>(sh + 2 * kKv8Block * kLd);  // [16][rot / 2]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t half = a.rot / 2;

  const uint32_t u = blockIdx.x;
  const uint32_t b = warp_last_le(a.c.num_seqs, u, [&](uint32_t i) { return a.row_start[i] / 16 + 2 * i; });
  Kv8Rows r;
  if (!kv8_rows(a.c, a.row_start, a.kv_len, a.tokens, b, &r)) {
    if (threadIdx.x == 0) raise_error(a.err, kDevBadParams);
    return;
  }
  const uint32_t pos0 = r.len - r.n;  // position of the sequence's first new row
  const uint32_t rel = u - (r.r0 / 16 + 2 * b);
  const uint32_t blk = pos0 / kKv8Block + rel;
  if (r.n == 0 || blk * kKv8Block >= r.len) return;
  const uint32_t lo = max(pos0, blk * kKv8Block), hi = min(r.len, (blk + 1) * kKv8Block);
  const uint32_t row0 = r.r0 + (lo - pos0), cnt = hi - lo, t0 = lo % kKv8Block;
  const bool fresh = t0 == 0;
  const uint32_t page = a.c.table[(size_t)b * a.c.max_pages + blk * kKv8Block / a.c.page_tokens];
  if (page >= a.c.num_pages) {
    if (threadIdx.x == 0) raise_error(a.err, kDevBadSlot);
    return;
  }
  const uint32_t in_page = blk % (a.c.page_tokens / kKv8Block);

  for (uint32_t i = threadIdx.x; i < cnt * half; i += blockDim.x) {
    const uint32_t t = i / half, f = i % half;
    float s, c;
    sincosf(__fmul_rn((float)(lo + t), a.inv_freq[f]), &s, &c);
    cs[i] = make_float2(c, s);
  }
  __syncthreads();

  // a lane's elements of a vector: chunk i is [(32 i + lane) kVec, + kVec)
  auto load = [&](const void *base, size_t off, float (&x)[kPer]) {
#pragma unroll
    for (int i = 0; i < kPer / kVec; ++i) {
      float v[kVec];
      load_vec<T, kVec>(static_cast<const T *>(base) + off + (32 * i + lane) * kVec, v);
#pragma unroll
      for (int j = 0; j < kVec; ++j) x[i * kVec + j] = v[j];
    }
  };
  auto gain = [&](const float *w, float (&x)[kPer]) {
#pragma unroll
    for (int i = 0; i < kPer / kVec; ++i)
#pragma unroll
      for (int j = 0; j < kVec; ++j)
        x[i * kVec + j] = __fmul_rn(x[i * kVec + j], w[(32 * i + lane) * kVec + j]);
  };
  // rotate token t's vector: the pairs meet in buf (one warp's row of D floats)
  auto rotate = [&](float (&x)[kPer], float *buf, uint32_t t) {
    if (half == 0) return;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kPer; ++i) buf[(32 * (i / kVec) + lane) * kVec + i % kVec] = x[i];
    __syncwarp();
    const float2 *ct = cs + t * half;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const uint32_t d = (32 * (i / kVec) + lane) * kVec + i % kVec;
      if (d < half) {
        const float2 f = ct[d];
        x[i] = __fsub_rn(__fmul_rn(x[i], f.x), __fmul_rn(buf[d + half], f.y));
      } else if (d < 2 * half) {
        const float2 f = ct[d - half];
        x[i] = __fadd_rn(__fmul_rn(buf[d - half], f.y), __fmul_rn(x[i], f.x));
      }
    }
  };

  const uint32_t h0 = blockIdx.y * a.heads_per_cta;
  const uint32_t h1 = min(a.c.num_kv, h0 + a.heads_per_cta);
  // ---- q rows
  const uint32_t nq = (h1 - h0) * a.gqa;
  for (uint32_t i = warp; i < cnt * nq; i += kAppWarps) {
    const uint32_t t = i / nq, h = h0 * a.gqa + i % nq;
    float x[kPer];
    load(a.q, (size_t)(row0 + t) * a.q_ld + (size_t)h * D, x);
    if (a.q_w) {
      normalise(x, a.eps, D);
      gain(a.q_w, x);
    }
    rotate(x, tile + warp * D, t);
    T *dst = static_cast<T *>(a.q_out) + ((size_t)(row0 + t) * a.c.num_kv * a.gqa + h) * D;
#pragma unroll
    for (int j = 0; j < kPer / kVec; ++j) {
      float v[kVec];
#pragma unroll
      for (int e = 0; e < kVec; ++e) v[e] = x[j * kVec + e];
      store_vec<T, kVec>(dst + (32 * j + lane) * kVec, v);
    }
  }

  // ---- K and V records
  for (uint32_t h = h0; h < h1; ++h) {
    __syncthreads();  // the tile is free
    for (uint32_t i = warp; i < 2 * cnt; i += kAppWarps) {
      const uint32_t t = i >> 1, is_v = i & 1;
      float *row = tile + (is_v * kKv8Block + t0 + t) * kLd;
      float x[kPer];
      if (is_v && !a.k_eq_v)
        load(a.v, (size_t)(row0 + t) * a.v_ld + (size_t)h * D, x);
      else
        load(a.k, (size_t)(row0 + t) * a.k_ld + (size_t)h * D, x);
      if (is_v) {
        if (a.v_norm) normalise(x, a.eps, D);
      } else {
        if (a.k_w) {
          normalise(x, a.eps, D);
          gain(a.k_w, x);
        }
        rotate(x, row, t);
        __syncwarp();
      }
      float m = 0.0f;
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        row[(32 * (j / kVec) + lane) * kVec + j % kVec] = x[j];
        m = fmaxf(m, fabsf(x[j]));  // a NaN does not count
      }
      m = warp_max(m);
      if (lane == 0) amax[is_v][t] = m;
    }
    __syncthreads();
    const size_t rec = (((size_t)page * a.c.num_kv + h) * (a.c.page_tokens / kKv8Block) + in_page) * 2;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      float m = 0.0f;
      for (uint32_t t = 0; t < cnt; ++t) m = fmaxf(m, amax[w][t]);
      const int e_old = fresh ? kKv8MinExp : kv8_scale_exponent(a.c.scale[rec + w]);
      const int e = max(e_old, kv8_exponent(m));
      const float inv = exp2_int(-e), shrink = exp2_int(e_old - e);
      uint8_t *out = static_cast<uint8_t *>(a.c.data) + (rec + w) * (size_t)(kKv8Block * D);
      const float *src = tile + w * kKv8Block * kLd;
      // scale is read by all before one thread writes it (the barrier below)
      for (uint32_t i = threadIdx.x; i < D; i += blockDim.x) {  // 16-byte pieces of the record
        const uint32_t p = i >> 5, g = (i & 31) >> 2, c = i & 3;
        uint4 old = make_uint4(0, 0, 0, 0);
        uint32_t v[4];
        if (w == 0) {
          const bool n0 = g >= t0 && g < t0 + cnt, n1 = g + 8 >= t0 && g + 8 < t0 + cnt;
          if (!fresh) {
            if (!n0 && !n1 && e == e_old) continue;
            if (!n0 || !n1) old = *reinterpret_cast<const uint4 *>(out + 16 * i);
          }
          v[0] = old.x; v[1] = old.y; v[2] = old.z; v[3] = old.w;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const bool is_new = q < 2 ? n0 : n1;
            if (is_new) {
              const float4 f = *reinterpret_cast<const float4 *>(src + (g + 8 * (q >> 1)) * kLd + 32 * p + 8 * c + 4 * (q & 1));
              v[q] = e4m3_pack4(f.x * inv, f.y * inv, f.z * inv, f.w * inv);
            } else if (e != e_old) {
              const float4 f = e4m3_unpack4(v[q]);
              v[q] = e4m3_pack4(f.x * shrink, f.y * shrink, f.z * shrink, f.w * shrink);
            }
          }
        } else {
          uint32_t is_new = 0;  // byte mask of the new tokens among 2 c, 2 c + 1, 2 c + 8, 2 c + 9
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            const uint32_t t = 2 * c + (s & 1) + 8 * (s >> 1);
            if (t >= t0 && t < t0 + cnt) is_new |= 0xFFu << (8 * s);
          }
          if (!fresh) {
            if (is_new == 0 && e == e_old) continue;
            if (is_new != 0xFFFFFFFFu) old = *reinterpret_cast<const uint4 *>(out + 16 * i);
          }
          v[0] = old.x; v[1] = old.y; v[2] = old.z; v[3] = old.w;
          float f[4][4];  // [token][element]
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            const uint32_t t = 2 * c + (s & 1) + 8 * (s >> 1);
            float4 x = make_float4(0, 0, 0, 0);
            if ((is_new >> (8 * s)) & 1) x = *reinterpret_cast<const float4 *>(src + t * kLd + 32 * p + 4 * g);
            f[s][0] = x.x; f[s][1] = x.y; f[s][2] = x.z; f[s][3] = x.w;
          }
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            if (e != e_old) {
              const float4 o = e4m3_unpack4(v[q]);
              v[q] = e4m3_pack4(o.x * shrink, o.y * shrink, o.z * shrink, o.w * shrink);
            }
            const uint32_t n = e4m3_pack4(f[0][q] * inv, f[1][q] * inv, f[2][q] * inv, f[3][q] * inv);
            v[q] = (n & is_new) | (v[q] & ~is_new);
          }
        }
        *reinterpret_cast<uint4 *>(out + 16 * i) = make_uint4(v[0], v[1], v[2], v[3]);
      }
    }
    __syncthreads();
    if (threadIdx.x < 2) {
      const uint32_t w = threadIdx.x;
      float m = 0.0f;
      for (uint32_t t = 0; t < cnt; ++t) m = fmaxf(m, amax[w][t]);
      const int e_old = fresh ? kKv8MinExp : kv8_scale_exponent(a.c.scale[rec + w]);
      a.c.scale[rec + w] = exp2_int(max(e_old, kv8_exponent(m)));
    }
  }
}

size_t append_smem(uint32_t d, uint32_t rot) {
  return 2 * kKv8Block * (d + 4) * sizeof(float) + (size_t)kKv8Block * (rot / 2) * sizeof(float2);
}

using AppendKernel = void (*)(AppendArgs);
AppendKernel append_kernel(sx_dtype t, uint32_t d) {
  if (t == SX_F32)
    return d == 64 ? kv8_append_kernel<float, 64> : d == 128 ? kv8_append_kernel<float, 128>
         : d == 256 ? kv8_append_kernel<float, 256> : kv8_append_kernel<float, 512>;
  return d == 64 ? kv8_append_kernel<__nv_bfloat16, 64> : d == 128 ? kv8_append_kernel<__nv_bfloat16, 128>
       : d == 256 ? kv8_append_kernel<__nv_bfloat16, 256> : kv8_append_kernel<__nv_bfloat16, 512>;
}

}  // namespace

cudaError_t prepare_kv8_append() {
  for (uint32_t d : {64u, 128u, 256u, 512u})
    for (sx_dtype t : {SX_F32, SX_BF16}) {
      const cudaError_t e = cudaFuncSetAttribute(
          append_kernel(t, d), cudaFuncAttributeMaxDynamicSharedMemorySize, (int)append_smem(d, d));
      if (e != cudaSuccess) return e;
    }
  return cudaSuccess;
}

}  // namespace sx

sx_status sx_host_check_kv8(const char *what, const sx_kv8 *c, sx_dtype t, uint32_t num_q) {
  const char *why = nullptr;
  if (!c || !c->data || !c->scale || !c->table)
    why = "null cache, data, scale or table";
  else if (t != SX_F32 && t != SX_BF16)
    why = "dtype must be SX_F32 or SX_BF16";
  else if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256 && c->head_dim != 512)
    why = "head_dim must be 64/128/256/512";
  else if (c->page_tokens == 0 || c->page_tokens % 16 != 0 || c->page_tokens > 1024)
    why = "page_tokens must be a multiple of 16, up to 1024";
  else if (c->num_pages == 0 || c->max_pages == 0 ||
           (uint64_t)c->max_pages * c->page_tokens >= (1ull << 31))
    why = "need pages, and max_pages * page_tokens below 2^31";
  else if (c->num_seqs > sx::kKv8MaxSeqs)
    why = "at most 4096 sequences";
  else if (c->num_kv == 0 || c->num_kv > 4096 || num_q % c->num_kv != 0 || num_q / c->num_kv > 64)
    why = "num_q must be a multiple of num_kv, at most 64 q heads per kv head";
  else if ((uintptr_t)c->data % 16 != 0 || (uintptr_t)c->scale % 8 != 0)
    why = "data must be 16-byte and scale 8-byte aligned";
  if (!why) return SX_OK;
  sx_host_set_error("%s: %s", what, why);
  return SX_ERR_INVALID;
}

extern "C" SX_API sx_status sx_dispatch_kv8_append(
    sx_engine *e, const sx_kv8 *c, sx_dtype t, const void *q_in, const void *k_in,
    const void *v_in, uint32_t q_ld, uint32_t k_ld, uint32_t v_ld, const float *q_norm_w,
    const float *k_norm_w, void *q_out, const uint32_t *row_start, const uint32_t *kv_len,
    uint32_t tokens, uint32_t num_q, const float *inv_freq, uint32_t rotary_dim, uint32_t flags,
    float eps) {
  auto bad = [](const char *why) {
    sx_host_set_error("kv8_append: %s", why);
    return SX_ERR_INVALID;
  };
  if (!e) return bad("null engine");
  sx_status st = sx_host_check_kv8("kv8_append", c, t, num_q);
  if (st != SX_OK) return st;
  const bool k_eq_v = (flags & SX_KV8_K_EQ_V) != 0;
  if (flags & ~(SX_KV8_K_EQ_V | SX_KV8_V_NORM)) return bad("unknown flag");
  if (!k_in || (!v_in && !k_eq_v) || !row_start || !kv_len) return bad("null k, v, row_start or kv_len");
  if (num_q > 0 && (!q_in || !q_out)) return bad("null q_in or q_out");
  if (rotary_dim % 2 != 0 || rotary_dim > c->head_dim) return bad("rotary_dim must be even and <= head_dim");
  if (rotary_dim > 0 && !inv_freq) return bad("null inv_freq");
  if (!(eps >= 0.0f)) return bad("eps must not be negative");
  const uint32_t es = t == SX_F32 ? 4 : 2, kv = c->num_kv * c->head_dim;
  if ((num_q > 0 && q_ld < num_q * c->head_dim) || k_ld < kv || (!k_eq_v && v_ld < kv))
    return bad("row strides are shorter than a row");
  uintptr_t al = (uintptr_t)k_in | (uintptr_t)k_ld * es;
  if (!k_eq_v) al |= (uintptr_t)v_in | (uintptr_t)v_ld * es;
  if (num_q > 0) al |= (uintptr_t)q_in | (uintptr_t)q_out | (uintptr_t)q_ld * es;
  if (al % 16 != 0) return bad("vectors must be 16-byte aligned and strides multiples of 16 bytes");
  if (tokens >= (1u << 30)) return bad("too many rows");
  if (tokens == 0 || c->num_seqs == 0) return SX_OK;
  cudaError_t ce = cudaSetDevice(e->device);
  if (ce != cudaSuccess) return sx_host_cuda_status(ce, "cudaSetDevice");
  sx::AppendArgs a{};
  a.c = *c;
  a.q = q_in; a.k = k_in; a.v = v_in;
  a.q_ld = q_ld; a.k_ld = k_ld; a.v_ld = v_ld;
  a.q_w = q_norm_w; a.k_w = k_norm_w;
  a.q_out = q_out;
  a.row_start = row_start;
  a.kv_len = kv_len;
  a.tokens = tokens;
  a.gqa = num_q / c->num_kv;
  a.rot = rotary_dim;
  a.k_eq_v = k_eq_v;
  a.v_norm = (flags & SX_KV8_V_NORM) != 0;
  a.inv_freq = inv_freq;
  a.eps = eps;
  a.err = e->err_dev;
  a.heads_per_cta = 1;
  const uint32_t units = tokens / sx::kKv8Block + 2 * c->num_seqs;
  const dim3 grid(units, (c->num_kv + a.heads_per_cta - 1) / a.heads_per_cta);
  sx::append_kernel(t, c->head_dim)<<<grid, sx::kAppWarps * 32,
                                      sx::append_smem(c->head_dim, rotary_dim), e->stream>>>(a);
  return sx_host_cuda_status(cudaGetLastError(), "kv8_append launch");
}
