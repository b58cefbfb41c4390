// sx_i8_gemv.cu -- products of up to 16 int8 rows: streaming the weights (include/sx.h, sx_dispatch_gemm_i8 and
// sx_dispatch_gate_up_i8).
//
// mma.m16n8k32 with 16 weight rows as A and 8 rows of x as B.  A sum does not care for the order of K, so a lane
// takes 16 consecutive bytes of a row, of weights and of x alike, for both halves of two products: the rows go from
// memory to the tensor core in wide copies as they are.  A CTA takes 32 rows of weights (gate_up: 16 of each
// matrix); its warps take pieces of 64 bytes of K in turn, each through a ring of its own that every lane fills
// and reads back alone, and their sums meet in shared memory.  Where the rows alone are too few CTAs, those of
// a cluster share them, each with a part of K.
//
// Measured, bound by HBM: 262144 rows of 3840 143 us (7.0 TB/s, 107 % of the measured copy rate); gate and up of one
// token (118 MB) 20.6 us (5.7 TB/s), 8 tokens 21.3; the down projection of one token (59 MB) 11.6 us (5.1 TB/s), 8
// tokens 12.6, 16 14.5; 3 us of each are the launch, the first bytes, the cluster's and the CTA's sums.  Three CTAs an
// SM with three pieces each on their way against two with four: 20.5 and 22.9 us for gate and up, but 13.9 and 11.9
// for the down projection, whose 240 CTAs all run at once.  Rows of x that are not there are not copied: eight lanes
// asking for the same bytes of the one row took 14.9 us for 11.9.  All of a CTA's weights asked into L2 at its start
// took longer (26.9 us for 22.9): they queue ahead of what is needed first.
#include "sx_host.h"
#include "sx_i8.cuh"
#include "sx_launch.cuh"

namespace sx {
namespace {

constexpr uint32_t kWarps = 8, kTileRows16 = 16, kPiece = 64;

SX_DEV void mma_s8_16832(int32_t (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 16 bytes, or zeros without reading src
SX_DEV void cp_async16_zfill(uint32_t dst, const void *src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(there ? 16u : 0u) : "memory");
}
SX_DEV void prefetch_l2(const void *p) { asm volatile("prefetch.global.L2 [%0];\n" ::"l"(p)); }
SX_DEV void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory"); }
SX_DEV void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory"); }

// NT: 8 rows of x each.  STAGES pieces of K on their way to a warp.
template <int NT, uint32_t STAGES>
struct GemvShape {
  static constexpr uint32_t kTok = 8 * NT, kSums = 2 * kTok * kTileRows16;  // of a CTA
  static constexpr uint32_t kStage = 2 * 1024 + NT * 512;                   // weights of two tiles, x
  static constexpr uint32_t kRing = STAGES * kStage;                        // of a warp; its sums in the end
  static_assert(kSums * 4 <= kRing, "a warp's sums");
  static constexpr uint32_t smem(uint32_t cluster) { return kWarps * kRing + (cluster - 1) * kSums * 4; }
};

template <typename T, bool GATED, int NT, uint32_t STAGES>
__global__ void __launch_bounds__(kWarps * 32, STAGES == 3 ? 3 : 2) gemv_i8_kernel(const __grid_constant__ I8Args a, uint32_t cluster) {
  using S = GemvShape<NT, STAGES>;
  constexpr uint32_t kCols = GATED ? kTileRows16 : 2 * kTileRows16;  // of y
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const uint32_t rank = blockIdx.x % cluster, n0 = blockIdx.x / cluster * kCols;
  uint8_t *const ring = smem + warp * S::kRing;
  const uint32_t ring_u = smem_u32(ring) + lane * 16;
  if (cluster > 1) cluster_arrive();  // that it runs
  pdl_launch_dependents();
  const int8_t *w[2][2], *x[NT];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int h = 0; h < 2; ++h)  // (past the end: not stored)
      w[m][h] = a.w[GATED ? m : 0] + (size_t)min(n0 + (GATED ? 0 : 16 * m) + g + 8 * h, a.n - 1) * a.w_ld;
#pragma unroll
  for (int t = 0; t < NT; ++t) x[t] = a.x + (size_t)min(g + 8 * t, a.t - 1) * a.x_ld;
  // this CTA's pieces of K, and of those the warp's
  const uint32_t pieces = (a.k + kPiece - 1) / kPiece;
  const uint32_t p0 = pieces * rank / cluster + warp, p1 = pieces * (rank + 1) / cluster;
  const uint32_t steps = p0 < p1 ? (p1 - p0 + kWarps - 1) / kWarps : 0;
  // What the ring takes first is asked into L2 while the kernel before this one ends (a prefetch gives no stale
  // bytes: L2 is where its writes go).  2 to 6 % of calls of 10 to 60 MB.
  if (c == 0) {
#pragma unroll
    for (uint32_t i = 0; i < STAGES - 1; ++i)
      if (i < steps) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int h = 0; h < 2; ++h) prefetch_l2(w[m][h] + (p0 + i * kWarps) * kPiece);
      }
  }
  pdl_wait();
  auto fetch = [&](uint32_t i) {
    const uint32_t at = ring_u + i % STAGES * S::kStage, k = (p0 + i * kWarps) * kPiece + 16 * c;
    const bool there = i < steps && k < a.k;
    const uint32_t from = there ? k : 0;
    if (i < steps) {
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) cp_async16_zfill(at + m * 1024 + h * 512, w[m][h] + from, there);
#pragma unroll
      for (int t = 0; t < NT; ++t) cp_async16_zfill(at + 2048 + t * 512, x[t] + from, there && g + 8 * t < a.t);
    }
    cp_async_commit();
  };
#pragma unroll
  for (uint32_t i = 0; i < STAGES - 1; ++i) fetch(i);
  int32_t s[2][NT][4];
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[m][t][i] = 0;
#pragma unroll 1
  for (uint32_t i = 0; i < steps; ++i) {
    fetch(i + STAGES - 1);
    cp_async_wait<STAGES - 1>();
    const uint8_t *const at = ring + i % STAGES * S::kStage + lane * 16;
    uint4 v[2][2];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) v[m][h] = *reinterpret_cast<const uint4 *>(at + m * 1024 + h * 512);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const uint4 b = *reinterpret_cast<const uint4 *>(at + 2048 + t * 512);
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        mma_s8_16832(s[m][t], v[m][0].x, v[m][1].x, v[m][0].y, v[m][1].y, b.x, b.y);
        mma_s8_16832(s[m][t], v[m][0].z, v[m][1].z, v[m][0].w, v[m][1].w, b.z, b.w);
      }
    }
  }
  cp_async_wait<0>();
  __syncwarp();
  // sums of the warps: [tile][row of x][row of the tile]
  auto sums_of = [&](uint32_t k) { return reinterpret_cast<int32_t *>(smem + k * S::kRing); };
#pragma unroll
  for (int m = 0; m < 2; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        sums_of(warp)[(m * S::kTok + 8 * t + 2 * c + (i & 1)) * kTileRows16 + g + 8 * (i >> 1)] = s[m][t][i];
  __syncthreads();
  auto sum_at = [&](uint32_t i) {
    int32_t v = 0;
#pragma unroll
    for (uint32_t k = 0; k < kWarps; ++k) v += sums_of(k)[i];
    return v;
  };
  int32_t *const others = reinterpret_cast<int32_t *>(smem + kWarps * S::kRing);  // the cluster's, in its first CTA
  if (cluster > 1) {
    cluster_wait();
    if (rank > 0) {
      uint32_t to;
      asm volatile("mapa.shared::cluster.u32 %0, %1, 0;\n" : "=r"(to) : "r"(smem_u32(others + (rank - 1) * S::kSums)));
      for (uint32_t i = threadIdx.x; i < S::kSums; i += kWarps * 32)
        asm volatile("st.shared::cluster.s32 [%0], %1;\n" ::"r"(to + 4 * i), "r"(sum_at(i)) : "memory");
    }
    cluster_arrive();
    cluster_wait();
    if (rank > 0) return;
  }
  for (uint32_t o = threadIdx.x; o < S::kTok * kCols; o += kWarps * 32) {
    const uint32_t t = o / kCols, col = o % kCols, n = n0 + col;
    if (t >= a.t || n >= a.n) continue;
    int32_t sum[2];
#pragma unroll
    for (uint32_t m = 0; m < (GATED ? 2 : 1); ++m) {
      const uint32_t i = ((GATED ? m : col / 16) * S::kTok + t) * kTileRows16 + col % 16;
      sum[m] = sum_at(i);
      for (uint32_t k = 0; k + 1 < cluster; ++k) sum[m] += others[k * S::kSums + i];
    }
    const float xs = a.x_scale[t];
    float v = i8_value(sum[0], xs, a.w_scale[0][n]);
    if constexpr (GATED) v = i8_gated(v, i8_value(sum[1], xs, a.w_scale[1][n]));
    static_cast<T *>(a.y)[(size_t)t * a.y_ld + n] = i8_out<T>(v);
  }
}

using GemvKernel = void (*)(const I8Args, uint32_t);
struct GemvVariant {
  GemvKernel fn;
  uint32_t ring, more;  // shared memory of a CTA, and for each further one of a cluster
};
template <typename T, bool GATED, int NT, uint32_t STAGES>
GemvVariant gemv_variant() {
  using S = GemvShape<NT, STAGES>;
  return {gemv_i8_kernel<T, GATED, NT, STAGES>, S::smem(1), S::smem(2) - S::smem(1)};
}
template <typename T, bool GATED>
GemvVariant gemv_variant(bool two, bool deep) {
  if (two) return deep ? gemv_variant<T, GATED, 2, 4>() : gemv_variant<T, GATED, 2, 3>();
  return deep ? gemv_variant<T, GATED, 1, 4>() : gemv_variant<T, GATED, 1, 3>();
}
GemvVariant gemv_variant(uint32_t dtype, bool gated, bool two, bool deep) {
  if (dtype == SX_F32) return gated ? gemv_variant<float, true>(two, deep) : gemv_variant<float, false>(two, deep);
  return gated ? gemv_variant<__nv_bfloat16, true>(two, deep) : gemv_variant<__nv_bfloat16, false>(two, deep);
}
constexpr uint32_t kMaxCluster = 8;

}  // namespace

cudaError_t prepare_gemv_i8() {
  for (uint32_t dtype : {SX_F32, SX_BF16})
    for (uint32_t i = 0; i < 8; ++i) {
      const GemvVariant v = gemv_variant(dtype, i & 1, i & 2, i & 4);
      const cudaError_t e =
          cudaFuncSetAttribute(v.fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(v.ring + (kMaxCluster - 1) * v.more));
      if (e != cudaSuccess) return e;
    }
  return cudaSuccess;
}

cudaError_t launch_gemv_i8(uint32_t dtype, bool gated, const I8Args &a, int num_sms, cudaStream_t s) {
  const uint32_t cols = gated ? kTileRows16 : 2 * kTileRows16, tiles = (a.n + cols - 1) / cols, sms = num_sms;
  // Where all CTAs run at once, two an SM with four pieces each on their way; three with three pieces where
  // one starts as another ends.
  const bool deep = tiles <= 2 * sms;
  const GemvVariant v = gemv_variant(dtype, gated, a.t > 8, deep);
  // CTAs of a cluster share rows as long as all run at once and each warp has two pieces of K
  uint32_t cluster = 1;
  while (cluster < kMaxCluster && cluster * tiles <= sms && a.k >= 4 * cluster * kWarps * kPiece) cluster *= 2;
  return launch_chained(v.fn, dim3(tiles * cluster), dim3(kWarps * 32), v.ring + (cluster - 1) * v.more, s, cluster, a, cluster);
}

}  // namespace sx
