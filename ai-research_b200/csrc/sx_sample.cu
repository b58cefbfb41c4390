// sx_sample.cu -- logits to probabilities, and verification of drafted tokens against them
// (include/sx.h, sx_dispatch_probs and sx_dispatch_verify).
#include "sx_host.h"
#include "sx_common.cuh"

namespace sx {
namespace {

constexpr int kSampleThreads = 1024;

struct ProbsArgs {
  const float *z;
  float *p;
  uint32_t z_ld, p_ld, n;
  float temperature;
};

// max that keeps a NaN
SX_DEV float max_nan(float a, float b) { return a != a ? a : (b != b ? b : fmaxf(a, b)); }

__global__ void __launch_bounds__(kSampleThreads) probs_kernel(ProbsArgs a) {
  __shared__ float red[32];
  const float *z = a.z + (size_t)blockIdx.x * a.z_ld;
  float *p = a.p + (size_t)blockIdx.x * a.p_ld;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float m = -INFINITY;
  for (uint32_t i = threadIdx.x; i < a.n; i += blockDim.x) m = max_nan(m, z[i]);
  for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) red[warp] = m;
  __syncthreads();
  m = red[lane];
  for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  __syncthreads();
  const float shift = m == -INFINITY ? 0.0f : m;
  float s = 0.0f;
  for (uint32_t i = threadIdx.x; i < a.n; i += blockDim.x) s += expf(__fdiv_rn(z[i] - shift, a.temperature));
  s = block_sum(s, red);
  for (uint32_t i = threadIdx.x; i < a.n; i += blockDim.x) {
    const float e = expf(__fdiv_rn(z[i] - shift, a.temperature));
    p[i] = m == -INFINITY ? 0.0f : __fdiv_rn(e, s);
  }
}

struct VerifyArgs {
  const float *p, *q;
  const uint32_t *tok, *n_draft;
  const float *u_accept, *u_sample;
  uint32_t *out, *accepted;
  uint32_t p_ld, q_ld, drafts, vocab;
  uint32_t *err;
};

// a probability as a multiple of 2^-38 (NaN and negative: 0)
SX_DEV uint64_t whole(float w) { return w > 0.0f ? (uint64_t)(fminf(w, 1.0f) * 0x1p38f) : 0ull; }

SX_DEV uint64_t warp_sum_u64(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__global__ void __launch_bounds__(kSampleThreads) verify_kernel(VerifyArgs a) {
  __shared__ uint64_t sums[32];
  __shared__ uint32_t drawn;
  const uint32_t b = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float *p = a.p + (size_t)b * (a.drafts + 1) * a.p_ld;
  const float *q = a.q ? a.q + (size_t)b * a.drafts * a.q_ld : nullptr;
  const uint32_t *tok = a.tok + (size_t)b * a.drafts;
  uint32_t nd = a.drafts;
  if (a.n_draft) {
    nd = a.n_draft[b];
    if (nd > a.drafts) {
      if (threadIdx.x == 0) raise_error(a.err, kDevBadParams);
      nd = a.drafts;
    }
  }
  uint32_t m = 0;
  for (; m < nd; ++m) {
    const uint32_t x = tok[m];
    if (x >= a.vocab) {
      if (threadIdx.x == 0) raise_error(a.err, kDevBadParams);
      break;
    }
    const float qx = q ? q[(size_t)m * a.q_ld + x] : 1.0f;
    if (!(__fmul_rn(a.u_accept[(size_t)b * a.drafts + m], qx) < p[(size_t)m * a.p_ld + x])) break;
  }
  const float *pr = p + (size_t)m * a.p_ld;
  const float *qr = m < nd && q ? q + (size_t)m * a.q_ld : nullptr;
  const uint32_t gone = m < nd && !q ? tok[m] : SX_NO_TOKEN;
  if (threadIdx.x == 0) drawn = SX_NO_TOKEN;
  for (int pass = 0; pass < 2; ++pass) {  // the difference; if it has no weight, the row itself
    auto weight = [&](uint32_t i) -> uint64_t {
      if (pass == 1) return whole(pr[i]);
      return whole(qr ? __fsub_rn(pr[i], qr[i]) : i == gone ? 0.0f : pr[i]);
    };
    // thread's run of consecutive tokens
    const uint32_t per = (a.vocab + blockDim.x - 1) / blockDim.x;
    const uint32_t i0 = min(a.vocab, threadIdx.x * per), i1 = min(a.vocab, i0 + per);
    uint64_t mine = 0;
    for (uint32_t i = i0; i < i1; ++i) mine += weight(i);
    uint64_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= (uint32_t)o) incl += v;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = incl;
    __syncthreads();
    uint64_t before = warp_sum_u64(lane < warp ? sums[lane] : 0ull);
    const uint64_t total = warp_sum_u64(sums[lane]);
    if (total == 0) continue;
    const uint64_t u = (uint64_t)(a.u_sample[b] * 16777216.0f);
    const uint64_t goal = (total >> 24) * u + (((total & 0xFFFFFFull) * u) >> 24);
    before += incl - mine;
    if (before <= goal && goal < before + mine) {
      uint64_t c = before;
      for (uint32_t i = i0; i < i1; ++i) {
        c += weight(i);
        if (c > goal) {
          drawn = i;
          break;
        }
      }
    }
    break;
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i <= a.drafts; i += blockDim.x)
    a.out[(size_t)b * (a.drafts + 1) + i] = i < m ? tok[i] : i == m ? drawn : SX_NO_TOKEN;
  if (threadIdx.x == 0) a.accepted[b] = m;
}

}  // namespace
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
  if (!(temperature > 0.0f) || !(temperature < 3.0e38f)) return bad("temperature must be positive and finite");
  if ((logits_ld && logits_ld < n) || (probs_ld && probs_ld < n)) return bad("strides are shorter than a row");
  if (logits == probs && (logits_ld ? logits_ld : n) != (probs_ld ? probs_ld : n))
    return bad("in place needs equal strides");
  if (rows == 0) return SX_OK;
  cudaError_t ce = cudaSetDevice(e->device);
  if (ce != cudaSuccess) return sx_host_cuda_status(ce, "cudaSetDevice");
  sx::ProbsArgs a{logits, probs, logits_ld ? logits_ld : n, probs_ld ? probs_ld : n, n, temperature};
  sx::probs_kernel<<<rows, sx::kSampleThreads, 0, e->stream>>>(a);
  return sx_host_cuda_status(cudaGetLastError(), "probs launch");
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
  if (seqs == 0) return SX_OK;
  cudaError_t ce = cudaSetDevice(e->device);
  if (ce != cudaSuccess) return sx_host_cuda_status(ce, "cudaSetDevice");
  sx::VerifyArgs a{target, drafts ? draft : nullptr, tok, n_draft, u_accept, u_sample, out, accepted,
                   target_ld ? target_ld : vocab, draft_ld ? draft_ld : vocab, drafts, vocab, e->err_dev};
  sx::verify_kernel<<<seqs, sx::kSampleThreads, 0, e->stream>>>(a);
  return sx_host_cuda_status(cudaGetLastError(), "verify launch");
}

}  // extern "C"
