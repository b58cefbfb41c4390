// sx_sample.cu -- logits to probabilities, and verification of drafted tokens against them
// (include/sx.h, sx_dispatch_probs and sx_dispatch_verify).
//
// Both walk rows of a vocabulary (1 MiB at 262144 tokens) and are bound by reading them, so a row
// is spread over a thread-block cluster: its CTAs exchange one partial result each through
// distributed shared memory, and the row is read once.  Many long rows take two passes instead.
// Measured, rows of 262144: probabilities of one row 4.6 us, of 40 rows 19.1 (4.4 TB/s); verification of
// 4 drafts for one sequence 7.2 us, for 64 sequences 26.5 (5.1 TB/s, 78 % of the measured copy rate).
#include "sx_common.cuh"
#include "sx_host.h"
#include "sx_launch.cuh"

namespace sx {
namespace {

constexpr int kSampleThreads = 512;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr uint32_t kMaxCluster = 16;

SX_DEV uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
  return r;
}
SX_DEV uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;\n" : "=r"(r));
  return r;
}
SX_DEV void cluster_arrive() { asm volatile("barrier.cluster.arrive.aligned;\n" ::: "memory"); }
SX_DEV void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;\n" ::: "memory"); }
// store to the same shared variable of cluster rank r
SX_DEV void st_cluster_u64(uint64_t *p, uint32_t r, uint64_t v) {
  asm volatile("{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %0, %1;\n"
               " st.shared::cluster.u64 [a], %2;\n}\n" ::"r"(smem_u32(p)),
               "r"(r), "l"(v)
               : "memory");
}
SX_DEV float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(x));
  return r;
}

// elements [i, i + 4) of a row of n; `fill` past its end
SX_DEV float4 load4(const float *p, uint32_t i, uint32_t n, bool aligned, float fill) {
  if (aligned && i + 4 <= n) return *reinterpret_cast<const float4 *>(p + i);
  float4 v = make_float4(fill, fill, fill, fill);
  if (i < n) v.x = p[i];
  if (i + 1 < n) v.y = p[i + 1];
  if (i + 2 < n) v.z = p[i + 2];
  if (i + 3 < n) v.w = p[i + 3];
  return v;
}
SX_DEV void store4(float *p, uint32_t i, uint32_t n, bool aligned, float4 v) {
  if (aligned && i + 4 <= n) {
    *reinterpret_cast<float4 *>(p + i) = v;
    return;
  }
  if (i < n) p[i] = v.x;
  if (i + 1 < n) p[i + 1] = v.y;
  if (i + 2 < n) p[i + 2] = v.z;
  if (i + 3 < n) p[i + 3] = v.w;
}
SX_DEV bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// ---------------------------------------------------------------------------------------
// p = 2^(c (z - max)) / sum, c = log2(e) / temperature.
struct ProbsArgs {
  const float *z;
  float *p;
  uint32_t z_ld, p_ld, n;
  float c;
};

// A sum of many terms whose rounding is carried along: rows of 2^24 logits leave chains of 64 (two passes) to
// 512 additions, which err alike where a row repeats itself (by 1e-6 of all its probabilities in two passes).
struct LongSum {
  float s = 0.0f, rest = 0.0f;
  SX_DEV void scale(float f) {
    s *= f;
    rest *= f;
  }
  SX_DEV void add(float x) {
    const float y = __fadd_rn(x, rest), t = __fadd_rn(s, y);
    rest = __fsub_rn(y, __fsub_rn(t, s));
    s = t;
  }
};

// NV > 0: a thread holds NV float4 of the row in registers, so the row is read once; NV = 0: rows
// of any length, read a second time (from L2) for the division.
template <int NV>
__global__ void __launch_bounds__(kSampleThreads) probs_kernel(ProbsArgs a) {
  __shared__ float red_m[kSampleWarps], red_s[kSampleWarps];
  __shared__ uint64_t part[kMaxCluster];  // {max, sum} of every CTA of the row
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t rank = cluster_rank(), ctas = cluster_size(), row = blockIdx.x / ctas;
  const float *z = a.z + (size_t)row * a.z_ld;
  float *p = a.p + (size_t)row * a.p_ld;
  const bool az = aligned16(z), ap = aligned16(p);
  cluster_arrive();  // met before the first store to another CTA: it has started by then
  pdl_launch_dependents();
  pdl_wait();

  float4 x[NV > 0 ? NV : 1];
  float m = -INFINITY, s = 0.0f;
  const uint32_t seg = NV > 0 ? kSampleThreads * 4 * NV : (a.n + ctas - 1) / ctas + 3 & ~3u;
  const uint32_t i0 = rank * seg + threadIdx.x * 4;
  auto local = [&](float top) { return top == -INFINITY ? 0.0f : top; };
  auto exps = [&](float4 v, float top) {
    return make_float4(ex2((v.x - top) * a.c), ex2((v.y - top) * a.c), ex2((v.z - top) * a.c),
                       ex2((v.w - top) * a.c));
  };
  if constexpr (NV > 0) {
#pragma unroll
    for (int k = 0; k < NV; ++k) x[k] = load4(z, i0 + k * kSampleThreads * 4, a.n, az, -INFINITY);
#pragma unroll
    for (int k = 0; k < NV; ++k) m = fmaxf(fmaxf(m, fmaxf(x[k].x, x[k].y)), fmaxf(x[k].z, x[k].w));
  } else {
    const uint32_t end = min(a.n, (rank + 1) * seg);
    LongSum sum;
    for (uint32_t i = i0; i < end; i += kSampleThreads * 4) {
      const float4 v = load4(z, i, end, az, -INFINITY);
      const float t = fmaxf(m, fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)));
      if (t > m) {
        sum.scale(m == -INFINITY ? 0.0f : ex2((m - t) * a.c));
        m = t;
      }
      const float4 e = exps(v, local(m));
      sum.add((e.x + e.y) + (e.z + e.w));
    }
    s = sum.s;
  }
  const float mine = m;
  m = warp_max(m);
  if (lane == 0) red_m[warp] = m;
  __syncthreads();
  m = warp_max(red_m[lane % kSampleWarps]);
  if constexpr (NV > 0) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      x[k] = exps(x[k], local(m));
      s += (x[k].x + x[k].y) + (x[k].z + x[k].w);
    }
  } else {
    s *= mine == -INFINITY ? 1.0f : ex2((mine - m) * a.c);
  }
  s = warp_sum(s);
  if (lane == 0) red_s[warp] = s;
  __syncthreads();
  s = lane < kSampleWarps ? red_s[lane] : 0.0f;
  s = warp_sum(s);
  float top = m, sum = s;
  cluster_wait();
  if (ctas > 1) {
    if (threadIdx.x < ctas)
      st_cluster_u64(part + rank, threadIdx.x, (uint64_t)__float_as_uint(s) << 32 | __float_as_uint(m));
    cluster_arrive();
    cluster_wait();
    const uint64_t v = part[lane % ctas];
    const float mk = __uint_as_float((uint32_t)v), sk = __uint_as_float((uint32_t)(v >> 32));
    top = warp_max(mk);
    sum = warp_sum((uint32_t)lane < ctas ? sk * (mk == -INFINITY ? 1.0f : ex2((mk - top) * a.c)) : 0.0f);
  }
  // a row of -inf alone has sum 0 and stays 0; a NaN or +inf has made the sum NaN
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  if constexpr (NV > 0) {
    const float f = (m == -INFINITY ? 1.0f : ex2((m - top) * a.c)) * inv;
#pragma unroll
    for (int k = 0; k < NV; ++k)
      store4(p, i0 + k * kSampleThreads * 4, a.n, ap,
             make_float4(x[k].x * f, x[k].y * f, x[k].z * f, x[k].w * f));
  } else {
    const uint32_t end = min(a.n, (rank + 1) * seg);
    for (uint32_t i = i0; i < end; i += kSampleThreads * 4) {
      const float4 e = exps(load4(z, i, end, az, -INFINITY), local(top));
      store4(p, i, end, ap, make_float4(e.x * inv, e.y * inv, e.z * inv, e.w * inv));
    }
  }
}

// Many long rows in two passes: {max, sum} of every chunk of a row, then the division, with the logits
// from L2 (126 MB; the chunks read last come first).  Clusters of 16 CTAs leave SMs empty and run in
// waves that wait for their sums; here every CTA streams.  40 rows of 262144: 19.1 us, of which 13.0
// are the bytes at the measured copy rate, the rest two launches' starts and ends.
constexpr int kChunkThreads = 256, kChunkVecs = 8;
constexpr uint32_t kChunk = kChunkThreads * 4 * kChunkVecs;

SX_DEV void load_chunk(const ProbsArgs &a, const float *z, uint32_t i0, float4 (&x)[kChunkVecs]) {
  const bool az = aligned16(z);
#pragma unroll
  for (int k = 0; k < kChunkVecs; ++k) x[k] = load4(z, i0 + k * kChunkThreads * 4, a.n, az, -INFINITY);
}
SX_DEV float max_of(const float4 (&x)[kChunkVecs]) {
  float m = -INFINITY;
#pragma unroll
  for (int k = 0; k < kChunkVecs; ++k) m = fmaxf(fmaxf(m, fmaxf(x[k].x, x[k].y)), fmaxf(x[k].z, x[k].w));
  return m;
}

__global__ void __launch_bounds__(kChunkThreads) probs_chunk_kernel(ProbsArgs a, uint32_t chunks, float2 *part) {
  __shared__ float2 red[kChunkThreads / 32];
  const uint32_t row = blockIdx.x / chunks, i0 = blockIdx.x % chunks * kChunk + threadIdx.x * 4;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  pdl_wait();
  pdl_launch_dependents();  // after the wait: the next pass may read logits before this one ends
  float4 x[kChunkVecs];
  load_chunk(a, a.z + (size_t)row * a.z_ld, i0, x);
  const float m = warp_max(max_of(x)), top = m == -INFINITY ? 0.0f : m;
  float s = 0.0f;
#pragma unroll
  for (int k = 0; k < kChunkVecs; ++k)
    s += (ex2((x[k].x - top) * a.c) + ex2((x[k].y - top) * a.c)) + (ex2((x[k].z - top) * a.c) + ex2((x[k].w - top) * a.c));
  s = warp_sum(s);
  if (lane == 0) red[warp] = make_float2(m, s);
  __syncthreads();
  if (warp == 0) {
    const float2 v = lane < kChunkThreads / 32 ? red[lane] : make_float2(-INFINITY, 0.0f);
    const float all = warp_max(v.x);
    const float sum = warp_sum(v.y * (v.x == -INFINITY ? 1.0f : ex2((v.x - all) * a.c)));
    if (lane == 0) part[blockIdx.x] = make_float2(all, sum);
  }
}

__global__ void __launch_bounds__(kChunkThreads) probs_divide_kernel(ProbsArgs a, uint32_t chunks, const float2 *part) {
  const uint32_t block = gridDim.x - 1 - blockIdx.x, row = block / chunks;
  const uint32_t i0 = block % chunks * kChunk + threadIdx.x * 4;
  const uint32_t lane = threadIdx.x & 31;
  float4 x[kChunkVecs];
  load_chunk(a, a.z + (size_t)row * a.z_ld, i0, x);
  pdl_launch_dependents();
  pdl_wait();
  float m = -INFINITY;
  LongSum s;
  for (uint32_t k = lane; k < chunks; k += 32) {  // (the same order in every warp)
    const float2 v = __ldcg(part + (size_t)row * chunks + k);
    const float top = fmaxf(m, v.x);
    s.scale(m == -INFINITY ? 1.0f : ex2((m - top) * a.c));
    s.add(v.y * (v.x == -INFINITY ? 1.0f : ex2((v.x - top) * a.c)));
    m = top;
  }
  const float all = warp_max(m), top = all == -INFINITY ? 0.0f : all;
  const float sum = warp_sum(s.s * (m == -INFINITY ? 1.0f : ex2((m - all) * a.c)));
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // -inf alone stays 0; a NaN or +inf made the sum NaN
  float *p = a.p + (size_t)row * a.p_ld;
  const bool ap = aligned16(p);
#pragma unroll
  for (int k = 0; k < kChunkVecs; ++k)
    store4(p, i0 + k * kChunkThreads * 4, a.n, ap,
           make_float4(ex2((x[k].x - top) * a.c) * inv, ex2((x[k].y - top) * a.c) * inv,
                       ex2((x[k].z - top) * a.c) * inv, ex2((x[k].w - top) * a.c) * inv));
}

// ---------------------------------------------------------------------------------------
struct VerifyArgs {
  const float *p, *q;
  const uint32_t *tok, *n_draft;
  const float *u_accept, *u_sample;
  uint32_t *out, *accepted;
  uint32_t p_ld, q_ld, drafts, vocab;
  uint32_t *err;
};

// floor(min(w, 1) 2^38), NaN and negative 0: 2^14 + w rounded toward zero in 64 bits has exactly
// that many units of 2^-38 past 2^14, and its bits count them.
constexpr uint64_t kWholeZero = 0x40D0000000000000ull;  // bits of 2^14
SX_DEV uint64_t whole_bits(float w) {
  return (uint64_t)__double_as_longlong(__dadd_rz((double)fminf(fmaxf(w, 0.0f), 1.0f), 16384.0));
}

SX_DEV uint64_t warp_sum_u64(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
SX_DEV uint64_t warp_scan_u64(uint64_t v) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t u = __shfl_up_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) >= o) v += u;
  }
  return v;
}

// One cluster per sequence.  The row is cut into one contiguous run per warp, a run into lines of
// 128 tokens (a float4 per lane); the warp keeps the sum of every line, lane i those of lines i,
// i + 32, ..., so that once the total is known the token is found by three prefix sums (warps,
// lines, tokens) and one line is read again.
constexpr uint32_t kLine = 128;

__global__ void __launch_bounds__(kSampleThreads, 2) verify_kernel(VerifyArgs a) {
  __shared__ uint64_t warp_sums[kSampleWarps];
  __shared__ uint64_t part[2][kMaxCluster];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t rank = cluster_rank(), ctas = cluster_size(), b = blockIdx.x / ctas;
  const float *p = a.p + (size_t)b * (a.drafts + 1) * a.p_ld;
  const float *q = a.q ? a.q + (size_t)b * a.drafts * a.q_ld : nullptr;
  const uint32_t *tok = a.tok + (size_t)b * a.drafts;
  cluster_arrive();  // met before the first store to another CTA
  pdl_launch_dependents();
  pdl_wait();
  const bool lead = rank == 0 && threadIdx.x == 0;
  const float us = a.u_sample[b];
  uint32_t nd = a.drafts;
  if (a.n_draft) {
    nd = a.n_draft[b];
    if (nd > a.drafts) {
      if (lead) raise_error(a.err, kDevBadParams);
      nd = a.drafts;
    }
  }
  // ---- how many drafts are accepted: a lane each, every warp alike
  uint32_t m = 0;
  for (; m < nd; m += 32) {
    const uint32_t i = m + lane;
    bool ok = false, bad = false;
    if (i < nd) {
      const uint32_t x = tok[i];
      bad = x >= a.vocab;
      if (!bad) {
        const float qx = q ? q[(size_t)i * a.q_ld + x] : 1.0f;
        ok = __fmul_rn(a.u_accept[(size_t)b * a.drafts + i], qx) < p[(size_t)i * a.p_ld + x];
      }
    }
    const uint32_t no = __ballot_sync(0xffffffffu, !ok);
    if (no) {
      const uint32_t at = __ffs(no) - 1;
      if (rank == 0 && warp == 0 && lane == (int)at && bad) raise_error(a.err, kDevBadParams);
      m += at;
      break;
    }
  }
  m = min(m, nd);
  const bool refused = m < nd;
  const float *pr = p + (size_t)m * a.p_ld;
  const float *qr = refused && q ? q + (size_t)m * a.q_ld : nullptr;
  const uint32_t gone = refused && !q ? tok[m] : SX_NO_TOKEN;  // q = 1 there, 0 elsewhere
  const bool ap = aligned16(pr), aq = aligned16(qr);

  const uint32_t lines = (a.vocab + kLine - 1) / kLine;
  const uint32_t per = (lines + ctas * kSampleWarps - 1) / (ctas * kSampleWarps);  // lines of a warp
  const uint32_t l0 = min(lines, (rank * kSampleWarps + warp) * per), l1 = min(lines, l0 + per);
  uint32_t drawn = SX_NO_TOKEN;
  bool here = false, none = true;  // this lane found the token; nothing has any weight
#pragma unroll 1
  for (int pass = 0; pass < 2; ++pass) {  // the difference; if it has no weight, the row itself
    // values of a line, and their weights
    auto fetch = [&](uint32_t line, float4 &v, float4 &d) {
      const uint32_t i = line * kLine + 4 * lane;
      v = load4(pr, i, a.vocab, ap, 0.0f);
      d = pass == 0 && qr ? load4(qr, i, a.vocab, aq, 0.0f) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    };
    auto weights = [&](uint32_t line, float4 v, float4 d, uint64_t (&w)[4]) {
      const uint32_t i = line * kLine + 4 * lane;
      w[0] = whole_bits(__fsub_rn(v.x, d.x)) - kWholeZero;
      w[1] = whole_bits(__fsub_rn(v.y, d.y)) - kWholeZero;
      w[2] = whole_bits(__fsub_rn(v.z, d.z)) - kWholeZero;
      w[3] = whole_bits(__fsub_rn(v.w, d.w)) - kWholeZero;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (pass == 0 && gone == i + k) w[k] = 0;
    };
    // Sums of groups of `step` of the warp's lines (four, or more so that 32 groups hold the run),
    // four lines in flight; lane i keeps that of group i.
    const uint32_t step = 4 * ((l1 - l0 + 127) / 128);
    uint64_t kept = 0, sum = 0;
    uint32_t in_group = 0, group = 0;
    for (uint32_t l = l0; l < l1; l += 4) {
      float4 v[4], d[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) fetch(l + k, v[k], d[k]);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint64_t w[4];
        weights(l + k, v[k], d[k], w);
        if (l + k < l1) sum += (w[0] + w[1]) + (w[2] + w[3]);
      }
      in_group += 4;
      if (in_group == step || l + 4 >= l1) {
        sum = warp_sum_u64(sum);
        if (lane == (int)group) kept = sum;
        ++group;
        sum = 0;
        in_group = 0;
      }
    }
    const uint64_t incl = warp_scan_u64(kept);
    const uint64_t mine = __shfl_sync(0xffffffffu, incl, 31);
    if (lane == 31) warp_sums[warp] = mine;
    __syncthreads();
    const uint64_t ws = lane < kSampleWarps ? warp_sums[lane] : 0;
    const uint64_t cta = warp_sum_u64(ws);
    const uint64_t before_warp = warp_sum_u64(lane < warp ? ws : 0);
    if (pass == 0) cluster_wait();
    if (threadIdx.x < ctas) st_cluster_u64(&part[pass][rank], threadIdx.x, cta);
    cluster_arrive();
    cluster_wait();
    const uint64_t ps = (uint32_t)lane < ctas ? part[pass][lane] : 0;
    const uint64_t total = warp_sum_u64(ps);
    if (total == 0) continue;  // the same in every CTA
    none = false;
    const uint64_t before = warp_sum_u64((uint32_t)lane < rank ? ps : 0) + before_warp;
    const uint64_t u = (uint64_t)(fminf(fmaxf(us, 0.0f), 1.0f - 0x1p-24f) * 16777216.0f);  // (a NaN is 0)
    const uint64_t goal = (total >> 24) * u + (((total & 0xFFFFFFull) * u) >> 24);
    if (before <= goal && goal < before + mine) {  // this warp's run
      const uint32_t who = __popc(__ballot_sync(0xffffffffu, before + incl <= goal));
      uint64_t c = before + __shfl_sync(0xffffffffu, incl - kept, who);
      for (uint32_t l = l0 + who * step; l < l1 && drawn == SX_NO_TOKEN; l += 4) {
        float4 v[4], d[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) fetch(l + k, v[k], d[k]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint64_t w[4];
          weights(l + k, v[k], d[k], w);
          const uint64_t sum = (w[0] + w[1]) + (w[2] + w[3]), in = warp_scan_u64(sum);
          const uint64_t line = __shfl_sync(0xffffffffu, in, 31);
          if (drawn == SX_NO_TOKEN && goal < c + line) {
            uint64_t t = c + in - sum;
            here = t <= goal && goal < t + sum;
            drawn = (l + k) * kLine + 4 * lane;
            if (t + w[0] <= goal) ++drawn;
            if (t + w[0] + w[1] <= goal) ++drawn;
            if (t + w[0] + w[1] + w[2] <= goal) ++drawn;
          }
          c += line;
        }
      }
    }
    break;
  }
  uint32_t *out = a.out + (size_t)b * (a.drafts + 1);
  if (here) out[m] = drawn;
  if (rank == 0) {
    for (uint32_t i = threadIdx.x; i <= a.drafts; i += kSampleThreads)
      if (i != m || none) out[i] = i < m ? tok[i] : SX_NO_TOKEN;
    if (threadIdx.x == 0) a.accepted[b] = m;
  }
}

using ProbsKernel = void (*)(ProbsArgs);
struct ProbsVariant {
  ProbsKernel fn;
  uint32_t ctas;
};
// Up to 8192 logits one CTA holds the row in registers, up to 16 x 16384 as many CTAs as it needs
// do; past that they read it twice.
ProbsVariant probs_variant(uint32_t n) {
  if (n <= 2048) return {probs_kernel<1>, 1};
  if (n <= 2 * 2048) return {probs_kernel<2>, 1};
  if (n <= 4 * 2048) return {probs_kernel<4>, 1};
  uint32_t ctas = 1;
  while (ctas < kMaxCluster && ctas * (8 * 2048) < n) ctas *= 2;
  return {n <= ctas * (8 * 2048) ? probs_kernel<8> : probs_kernel<0>, ctas};
}

// Rows of four CTAs and more that do not all fit at once (two CTAs an SM, less what clusters leave
// empty) take two passes: 40 rows of 262144 19.1 us for 25.6, 18 rows 11.2 for 14.8, 100 rows of 65536
// 14.0 for 16.7; those that fit one, 10 rows of 262144 7.0 us either way, 40 of 65536 6.9.
constexpr uint32_t kTwoPassCtas = 4;

}  // namespace

cudaError_t prepare_sample_kernels() {
  const void *k[] = {(const void *)probs_kernel<0>, (const void *)probs_kernel<8>, (const void *)verify_kernel};
  for (const void *f : k) {
    const cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace sx

extern "C" {

SX_API sx_status sx_dispatch_probs(sx_engine *e, const float *logits, uint32_t logits_ld,
                                   float *probs, uint32_t probs_ld, uint32_t rows, uint32_t n,
                                   float temperature) {
  auto bad = [](const char *why) {
    sx_host_set_error("probs: %s", why);
    return SX_ERR_INVALID;
  };
  if (!e || !logits || !probs) return bad("null engine, logits or probs");
  if (n == 0 || n > (1u << 24)) return bad("n must be 1 .. 2^24");
  if (!(temperature >= 1e-30f) || !(temperature <= 1e30f)) return bad("temperature must be 1e-30 .. 1e30");
  if ((logits_ld && logits_ld < n) || (probs_ld && probs_ld < n)) return bad("strides are shorter than a row");
  if (logits == probs && (logits_ld ? logits_ld : n) != (probs_ld ? probs_ld : n))
    return bad("in place needs equal strides");
  if (rows >= (1u << 26)) return bad("too many rows");
  if (rows == 0) return SX_OK;
  cudaError_t ce = cudaSetDevice(e->device);
  if (ce != cudaSuccess) return sx_host_cuda_status(ce, "cudaSetDevice");
  sx::ProbsArgs a{logits, probs, logits_ld ? logits_ld : n, probs_ld ? probs_ld : n, n,
                  1.4426950408889634f / temperature};
  const sx::ProbsVariant v = sx::probs_variant(n);
  if (v.ctas >= sx::kTwoPassCtas && 2ull * rows * v.ctas > 3ull * e->num_sms) {
    const uint32_t chunks = (n + sx::kChunk - 1) / sx::kChunk;
    float2 *const part = e->probs_part;
    e->scratch_used = true;
    const uint32_t most = (uint32_t)(sx::kProbsPartBytes / sizeof(float2)) / chunks;
    for (uint32_t r = 0; r < rows && ce == cudaSuccess; r += most) {
      sx::ProbsArgs b = a;
      b.z += (size_t)r * a.z_ld;
      b.p += (size_t)r * a.p_ld;
      const dim3 grid(std::min(most, rows - r) * chunks), block(sx::kChunkThreads);
      ce = sx::launch_chained(sx::probs_chunk_kernel, grid, block, 0, e->stream, 1, b, chunks, part);
      if (ce == cudaSuccess)
        ce = sx::launch_chained(sx::probs_divide_kernel, grid, block, 0, e->stream, 1, b, chunks, (const float2 *)part);
    }
    return sx_host_cuda_status(ce, "probs launch");
  }
  return sx_host_cuda_status(
      sx::launch_chained(v.fn, dim3(rows * v.ctas), dim3(sx::kSampleThreads), 0, e->stream, v.ctas, a),
      "probs launch");
}

SX_API sx_status sx_dispatch_verify(sx_engine *e, const float *target, uint32_t target_ld,
                                    const float *draft, uint32_t draft_ld, const uint32_t *tok,
                                    const uint32_t *n_draft, const float *u_accept,
                                    const float *u_sample, uint32_t *out, uint32_t *accepted,
                                    uint32_t seqs, uint32_t drafts, uint32_t vocab) {
  auto bad = [](const char *why) {
    sx_host_set_error("verify: %s", why);
    return SX_ERR_INVALID;
  };
  if (!e || !target || !u_sample || !out || !accepted) return bad("null argument");
  if (drafts > 0 && (!tok || !u_accept)) return bad("null drafted tokens or u_accept");
  if (vocab == 0 || vocab > (1u << 24)) return bad("vocab must be 1 .. 2^24");
  if (drafts > 1024) return bad("at most 1024 drafts");
  if ((target_ld && target_ld < vocab) || (draft_ld && draft_ld < vocab))
    return bad("strides are shorter than a row");
  if (seqs >= (1u << 26)) return bad("too many sequences");
  if (seqs == 0) return SX_OK;
  cudaError_t ce = cudaSetDevice(e->device);
  if (ce != cudaSuccess) return sx_host_cuda_status(ce, "cudaSetDevice");
  sx::VerifyArgs a{target, drafts ? draft : nullptr, tok, n_draft, u_accept, u_sample, out, accepted,
                   target_ld ? target_ld : vocab, draft_ld ? draft_ld : vocab, drafts, vocab, e->err_dev};
  // a CTA per 8192 tokens of the vocabulary, while they fit the GPU at once (two per SM)
  uint32_t ctas = 1;
  while (ctas < sx::kMaxCluster && ctas * 8192 < vocab && (uint64_t)seqs * ctas * 2 <= 2ull * e->num_sms) ctas *= 2;
  return sx_host_cuda_status(
      sx::launch_chained(sx::verify_kernel, dim3(seqs * ctas), dim3(sx::kSampleThreads), 0, e->stream, ctas, a),
      "verify launch");
}

}  // extern "C"
