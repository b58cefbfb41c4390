// sx_i8_gemm.cu -- products of int8 rows on the tcgen05 tensor cores (include/sx.h, sx_dispatch_gemm_i8 and
// sx_dispatch_gate_up_i8).
//
// A CTA takes 128 rows of x and 128 columns of y: the tiles come by TMA, 128 codes of K a stage, and
// tcgen05.mma (kind::i8) sums them in 32 bits in tensor memory.  gate_up: 64 columns of each matrix.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <mutex>

#include "sx_host.h"
#include "sx_i8.cuh"
#include "sx_launch.cuh"
#include "sx_tcgen05.cuh"

namespace sx {
namespace {

constexpr uint32_t kBM = 128, kBN = 128, kBK = 128, kStages = 4;
constexpr uint32_t kATile = kBM * kBK, kBTile = kBN * kBK, kStage = kATile + kBTile;
constexpr uint32_t kSmem = kStages * kStage + 1024;
constexpr int kThreads = 6 * 32;

SX_DEV void tma_load_2d(uint32_t dst, const CUtensorMap *map, int32_t x, int32_t y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], "
      "[%1, {%2, %3}], [%4];\n" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
// D[tmem] (+)= A[smem desc] . B[smem desc]^T of int8, 32 of K
SX_DEV void umma_i8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
// Instruction descriptor: D s32, A and B s8, both K-major, N >> 3, M >> 4.
constexpr uint32_t umma_idesc_i8(uint32_t m, uint32_t n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((m >> 4) << 24);
}

struct Maps {
  CUtensorMap x, w[2];
};

template <typename T, bool GATED>
__global__ void __launch_bounds__(kThreads, 1) gemm_i8_kernel(const __grid_constant__ Maps maps, const __grid_constant__ I8Args a) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bars[2 * kStages + 1];
  __shared__ uint32_t tmem_slot, abort_flag;
  constexpr uint32_t kCols = GATED ? kBN / 2 : kBN;  // of y
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t base = (smem_u32(smem_raw) + 1023) & ~1023u, bar0 = smem_u32(bars);
  auto full = [&](uint32_t s) { return bar0 + 8 * s; };
  auto empty = [&](uint32_t s) { return bar0 + 8 * (kStages + s); };
  const uint32_t done = bar0 + 16 * kStages;
  const uint32_t m0 = blockIdx.x * kBM, n0 = blockIdx.y * kCols, steps = (a.k + kBK - 1) / kBK;
  volatile uint32_t *const stop = &abort_flag;
  if (threadIdx.x == 0) {
    for (uint32_t s = 0; s < kStages; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    mbar_init(done, 1);
    abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0) {
    tmem_alloc(smem_u32(&tmem_slot), kBN);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  auto wait = [&](uint32_t bar, uint32_t parity) {
    if (*stop) return false;
    if (mbar_wait_bounded(bar, parity & 1)) return true;
    *stop = 1;
    raise_error(a.err, kDevWaitTimeout);
    return false;
  };
  pdl_launch_dependents();
  pdl_wait();
  uint32_t issued = 0;
  if (warp == 0 && lane == 0) {
    for (uint32_t i = 0; i < steps; ++i) {
      const uint32_t s = i % kStages, st = base + s * kStage;
      if (i >= kStages && !wait(empty(s), i / kStages - 1)) break;
      mbar_arrive_expect_tx(full(s), kStage);
      tma_load_2d(st, &maps.x, i * kBK, m0, full(s));
      tma_load_2d(st + kATile, &maps.w[0], i * kBK, n0, full(s));
      if constexpr (GATED) tma_load_2d(st + kATile + kBTile / 2, &maps.w[1], i * kBK, n0, full(s));
      issued = i + 1;
    }
  } else if (warp == 1 && lane == 0) {
    for (uint32_t i = 0; i < steps; ++i) {
      const uint32_t s = i % kStages, st = base + s * kStage;
      if (!wait(full(s), i / kStages)) break;
      tc_fence_after();
      const uint64_t x = umma_desc_sw128(st), w = umma_desc_sw128(st + kATile);
#pragma unroll
      for (uint32_t k = 0; k < kBK / 32; ++k) umma_i8(tmem, x + 2 * k, w + 2 * k, umma_idesc_i8(kBM, kBN), i > 0 || k > 0);
      umma_commit(empty(s));
    }
    umma_commit(done);
  } else if (warp >= 2) {
    const uint32_t q = warp & 3, t = m0 + 32 * q + lane;
    const bool ok = wait(done, 0);
    __syncwarp();
    tc_fence_after();
    if (__all_sync(0xffffffffu, ok)) {
      const float xs = t < a.t ? a.x_scale[t] : 0.0f;
      T *const y = static_cast<T *>(a.y) + (size_t)min(t, a.t - 1) * a.y_ld;
#pragma unroll 1
      for (uint32_t c = 0; c < kCols; c += 32) {
        uint32_t r[32], u[32];
        tmem_ld32(tmem + ((32 * q) << 16) + c, r);
        if constexpr (GATED) tmem_ld32(tmem + ((32 * q) << 16) + kBN / 2 + c, u);
        tmem_wait_ld(r);
        if constexpr (GATED) tmem_wait_ld(u);
#pragma unroll
        for (uint32_t j = 0; j < 32; ++j) {
          const uint32_t n = n0 + c + j;
          if (t < a.t && n < a.n) {
            float v = i8_value((int32_t)r[j], xs, a.w_scale[0][n]);
            if constexpr (GATED) v = i8_gated(v, i8_value((int32_t)u[j], xs, a.w_scale[1][n]));
            y[n] = i8_out<T>(v);
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0 && lane == 0 && *stop)  // a stopped CTA waits (bounded) for the copies that it issued
    for (uint32_t s = 0; s < kStages; ++s)
      if (issued > s) mbar_wait_bounded(full(s), ((issued - 1 - s) / kStages) & 1);
  __syncwarp();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, kBN);
  }
}

PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess && q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

// rows of k codes, in boxes of `box` rows x 128 codes
bool encode_rows(CUtensorMap *map, const int8_t *p, uint32_t rows, uint32_t k, uint32_t ld, uint32_t box_rows) {
  auto encode = tensor_map_encoder();
  const cuuint64_t dims[2] = {k, rows}, strides[1] = {ld};
  const cuuint32_t box[2] = {kBK, box_rows}, one[2] = {1, 1};
  return encode && encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<int8_t *>(p), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool GATED>
cudaError_t launch_gemm(uint32_t dtype, const I8Args &a, cudaStream_t s) {
  Maps maps;
  constexpr uint32_t cols = GATED ? kBN / 2 : kBN;
  if (!encode_rows(&maps.x, a.x, a.t, a.k, a.x_ld, kBM) || !encode_rows(&maps.w[0], a.w[0], a.n, a.k, a.w_ld, cols)) return cudaErrorInvalidValue;
  if (GATED && !encode_rows(&maps.w[1], a.w[1], a.n, a.k, a.w_ld, cols)) return cudaErrorInvalidValue;
  auto kern = dtype == SX_F32 ? gemm_i8_kernel<float, GATED> : gemm_i8_kernel<__nv_bfloat16, GATED>;
  return launch_chained(kern, dim3((a.t + kBM - 1) / kBM, (a.n + cols - 1) / cols), dim3(kThreads), kSmem, s, 1, maps, a);
}

}  // namespace

cudaError_t prepare_gemm_i8() {
  for (auto k : {gemm_i8_kernel<float, false>, gemm_i8_kernel<float, true>, gemm_i8_kernel<__nv_bfloat16, false>, gemm_i8_kernel<__nv_bfloat16, true>}) {
    const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmem);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace sx

namespace {

sx_status dispatch_i8(const char *what, sx_engine *e, uint32_t dtype, sx::I8Args &a, bool gated) {
  auto bad = [&](const char *why) {
    sx_host_set_error("%s: %s", what, why);
    return SX_ERR_INVALID;
  };
  if (dtype != SX_F32 && dtype != SX_BF16) return bad("dtype must be SX_F32 or SX_BF16");
  uintptr_t al = (uintptr_t)a.x | a.x_ld | a.w_ld;
  for (int i = 0; i < (gated ? 2 : 1); ++i) {
    if (!a.w[i] || !a.w_scale[i]) return bad("null weights or scales");
    al |= (uintptr_t)a.w[i];
    if ((uintptr_t)a.w_scale[i] % 4 != 0) return bad("scales must be aligned to their elements");
  }
  if (!a.x || !a.x_scale || !a.y) return bad("null x, x_scale or y");
  if ((uintptr_t)a.x_scale % 4 != 0) return bad("scales must be aligned to their elements");
  if (a.k == 0 || a.k % 16 != 0 || a.k >= sx::kI8MaxK) return bad("k must be a multiple of 16, above 0 and below 131072");
  if (a.n == 0) return bad("n must be above 0");
  if (a.x_ld < a.k || a.w_ld < a.k || a.y_ld < a.n) return bad("row strides are shorter than a row");
  if (al % 16 != 0) return bad("x and weights must be 16-byte aligned and their strides multiples of 16");
  if ((uintptr_t)a.y % (dtype == SX_F32 ? 4 : 2) != 0) return bad("y must be aligned to its elements");
  if (a.t >= (1u << 31) || a.n >= (1u << 31)) return bad("t and n must be below 2^31");
  if (!e) return bad("null engine");
  if (a.t == 0) return SX_OK;
  const cudaError_t ce = cudaSetDevice(e->device);
  if (ce != cudaSuccess) return sx_host_cuda_status(ce, "cudaSetDevice");
  a.err = e->err_dev;
  return sx_host_cuda_status(gated ? sx::launch_gemm<true>(dtype, a, e->stream) : sx::launch_gemm<false>(dtype, a, e->stream), what);
}

}  // namespace

extern "C" {

SX_API sx_status sx_dispatch_gemm_i8(sx_engine *e, const sx_gemm_i8_args *p) {
  if (!p) {
    sx_host_set_error("gemm_i8: null arguments");
    return SX_ERR_INVALID;
  }
  sx::I8Args a{p->x, {p->w, nullptr}, p->x_scale, {p->w_scale, nullptr}, p->y, p->x_ld, p->w_ld, p->y_ld, p->t, p->n, p->k, nullptr};
  return dispatch_i8("gemm_i8", e, p->dtype, a, false);
}

SX_API sx_status sx_dispatch_gate_up_i8(sx_engine *e, const sx_gate_up_i8_args *p) {
  if (!p) {
    sx_host_set_error("gate_up_i8: null arguments");
    return SX_ERR_INVALID;
  }
  sx::I8Args a{p->x, {p->wg, p->wu}, p->x_scale, {p->wg_scale, p->wu_scale}, p->y, p->x_ld, p->w_ld, p->y_ld, p->t, p->n, p->k, nullptr};
  return dispatch_i8("gate_up_i8", e, p->dtype, a, true);
}

SX_API uint32_t sx_i8_args_bytes(uint32_t which) {
  const size_t n[4] = {sizeof(sx_quantize_i8_args), sizeof(sx_residual_norm_args), sizeof(sx_gemm_i8_args), sizeof(sx_gate_up_i8_args)};
  return which < 4 ? (uint32_t)n[which] : 0;
}

}  // extern "C"
