// sx_i8_gemm.cu -- products of int8 rows on the tcgen05 tensor cores (include/sx.h, sx_dispatch_gemm_i8 and
// sx_dispatch_gate_up_i8).
//
//   y[t][n] = x_scale[t] w_scale[n] sum_k x[t][k] w[n][k]        gate_up: gelu_tanh(y_gate) y_up
//
// Sums are whole numbers below 2^31 in 32 bits: no order of summation, split of K or kernel changes them, and a
// value is rounded three times in f32 (the sum, two scales), then to y's type.
//
// Many rows: tiles.  Two CTAs of a cluster take a tile of 256 rows of x and 256 columns of y (gate_up: 128 of each
// matrix), 128 rows in the tensor memory of each: tcgen05.mma of the pair (kind::i8) reads 128 rows of x and half of
// the columns' weights from each CTA's shared memory, so both operands are fetched once per pair.  The grid is one
// pair per two SMs, which goes through the tiles; tensor memory holds two tiles' sums, so that one is scaled and
// stored while the next is summed.  Warps of a CTA:
//   0       TMA: 128 codes of K a stage, six stages, completing on the leader's barrier
//   1       the leader's issues the products and commits stages and sums to both CTAs
//   2 .. 9  sums to values, 32 rows each and every other box of columns, staged in shared memory and stored by TMA
//           (rows of y that do not begin on 16 bytes, and ends of rows inside them: by lanes)
// Measured: 16896 x 8192 x 3840 into f32 411 us (box to box up to 433), 2.6 POP/s or 159 % of the measured bf16
// rate; gate and up of 16896 x 15360 x 3840 1323 us, 3.0 POP/s, 184 %.  What bounds it is the power cap: the clock
// falls to 1.3 GHz, and bringing tiles from L2 takes nearly as much power as the products.  (Zeros as data leave it
// at 1.97 GHz, and the same call takes 252 us; products without copies 271, copies without products 243; no stores
// 351 of 433, stores that stay in L2 395.)  So tiles that read less for a product were tried: 256 x 512 with one set
// of sums ran at 1.5 GHz and took 391 us for 365, since four stages of 48 KB are too few; 256 x 128 takes 456 for
// 369.  A thread that issues by itself costs the products of 128 columns a third (516 us for 343, without copies):
// what is alike in a warp has to be known to be so.
//
// Few rows of x, or few tiles: see below.
#include <algorithm>
#include <type_traits>

#include "sx_host.h"
#include "sx_i8.cuh"
#include "sx_kv8.cuh"
#include "sx_launch.cuh"
#include "sx_tcgen05.cuh"
#include "sx_tma.cuh"

namespace sx {
namespace {

constexpr uint32_t kBM = 256, kBN = 256, kBK = 128;  // of a pair
constexpr uint32_t kHalf = kBM / 2;             // rows of a CTA
constexpr int kEpiWarps = 8, kThreads = (2 + kEpiWarps) * 32;
constexpr uint32_t kBox = 4096;                 // 32 rows of 128 bytes of y
constexpr uint32_t kTmemCols = 512;             // two tiles' sums

constexpr uint32_t kATile = kHalf * kBK, kBTile = kBN / 2 * kBK, kStage = kATile + kBTile, kStages = 196608 / kStage;
constexpr uint32_t kData = kStages * kStage + kEpiWarps * kBox;
// What the CTA's threads share behind the stages and boxes: no static shared memory beside them, so that they begin
// on the 1024 bytes that the swizzle asks for, with room for a little less than that.
template <int MATS>
struct PairShared {
  float col_scale[kEpiWarps][MATS][32];
  uint64_t bars[2 * kStages + 4];
  uint32_t tmem_slot, abort_flag;
};
constexpr uint32_t kMaxSmem = 227 * 1024;

// ---- TMA, cluster and pair wrappers
SX_DEV uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(r));
  return r;
}
SX_DEV void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
// the address of a shared-memory word of this CTA in CTA `rank` of the cluster
SX_DEV uint32_t in_cta(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
// Nothing in memory is handed over by it, only sums that have been read: a release would wait for the lanes' stores to
// y too (8192 x 8191 x 512 into bf16 76 us, so 55; gate and up of it into f32 143, 110).
SX_DEV void mbar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];\n" ::"r"(bar) : "memory");
}
// 2-D tiled load into this CTA's shared memory that completes on a barrier of either CTA of the pair
SX_DEV void tma_load_pair(uint32_t dst, const CUtensorMap *map, int32_t x, int32_t y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], "
      "[%1, {%2, %3}], [%4];\n" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
      : "memory");
}
SX_DEV void tma_prefetch_2d(const CUtensorMap *map, int32_t x, int32_t y) {
  asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];\n" ::"l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y)
               : "memory");
}
// a store of what is not to stay in L2
SX_DEV void tma_store_2d_far(const CUtensorMap *map, int32_t x, int32_t y, uint32_t src, uint64_t policy) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group.L2::cache_hint [%0, {%1, %2}], [%3], %4;\n" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y), "r"(src), "l"(policy)
               : "memory");
}

SX_DEV void tmem_alloc_pair(uint32_t dst_smem, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(dst_smem), "r"(cols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
}
SX_DEV void tmem_dealloc_pair(uint32_t taddr, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(taddr), "r"(cols) : "memory");
}
// D[tmem] (+)= A[smem desc] . B[smem desc]^T of int8, 32 of K, A and B from both CTAs of the pair
SX_DEV void umma_i8_pair(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
// arrive once on the barrier at this place in both CTAs when every operation this thread issued has completed
SX_DEV void umma_commit_pair(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n" ::"r"(bar),
               "h"((uint16_t)3)
               : "memory");
}
// Instruction descriptor: D s32, A and B s8, both K-major, N >> 3, M >> 4.
constexpr uint32_t umma_idesc_i8(uint32_t m, uint32_t n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((m >> 4) << 24);
}

// A wait that runs out ends this CTA's waiting: what follows is skipped, and the error word says so.
__device__ __noinline__ bool wait_longer(uint32_t bar, uint32_t parity, volatile uint32_t *stop, uint32_t *err) {
  if (*stop) return false;
  if (mbar_wait_bounded(bar, parity)) return true;
  *stop = 1;
  raise_error(err, kDevWaitTimeout);
  return false;
}

template <typename T>
SX_DEV T ld_shared(uint32_t src) {
  if constexpr (sizeof(T) == 4) {
    float f;
    asm volatile("ld.shared.f32 %0, [%1];\n" : "=f"(f) : "r"(src) : "memory");
    return f;
  } else {
    uint16_t h;
    asm volatile("ld.shared.u16 %0, [%1];\n" : "=h"(h) : "r"(src) : "memory");
    return __ushort_as_bfloat16(h);
  }
}

struct Maps {
  CUtensorMap x, w[2], part[2], y;  // part: the weights in boxes for a part of a tile
};
struct Tiles {
  uint32_t rows, cols;  // tiles of rows and of columns
  uint32_t group;       // tiles of rows that go through all columns together
  uint32_t whole;       // tiles taken whole; those after them in 2^part parts, by columns
  uint32_t part, units; // units: whole tiles and parts
  uint32_t boxes;       // boxes of y that end before this column are stored by copies, the others by lanes
  uint32_t far;         // y is more than L2 holds: its lines leave L2 before those of x and the weights
};
// What a pair takes at a time: columns [part, + 1) of 2^lg of a tile
struct Unit {
  uint32_t row, col, lg, part;
};
// Tile i: what runs at a time reads few rows of either matrix, and the rows of x of a group stay in L2 meanwhile.
SX_DEV Unit unit_at(const Tiles &g, uint32_t i) {
  Unit u;
  u.lg = i < g.whole ? 0 : g.part;
  const uint32_t tile = i < g.whole ? i : g.whole + ((i - g.whole) >> u.lg);
  u.part = (i - g.whole) & ((1u << u.lg) - 1);
  const uint32_t band = tile / (g.group * g.cols), in = tile - band * g.group * g.cols;
  const uint32_t high = min(g.group, g.rows - band * g.group);
  u.col = in / high;
  u.row = band * g.group + in % high;
  return u;
}

template <typename T, bool GATED>
__global__ void __launch_bounds__(kThreads, 1)
    gemm_i8_pair_kernel(const __grid_constant__ Maps maps, const __grid_constant__ I8Args a, const __grid_constant__ Tiles g) {
  constexpr uint32_t kCols = GATED ? kBN / 2 : kBN;  // columns of y of a tile
  using Shared = PairShared<GATED ? 2 : 1>;
  static_assert(kData + sizeof(Shared) <= kMaxSmem, "shared memory");
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023) & ~1023u, skip = base - smem_u32(smem_raw);
  if (skip + kData + sizeof(Shared) > kMaxSmem) {  // (alike in all CTAs: never where shared memory is laid out as it is)
    raise_error(a.err, kDevBadParams);
    return;
  }
  Shared &sh = *reinterpret_cast<Shared *>(smem_raw + skip + kData);
  uint32_t &tmem_slot = sh.tmem_slot, &abort_flag = sh.abort_flag;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = cluster_rank(), bar0 = smem_u32(sh.bars);
  auto full = [&](uint32_t s) { return bar0 + 8 * s; };                   // the leader's: both CTAs' copies
  auto empty = [&](uint32_t s) { return bar0 + 8 * (kStages + s); };      // each CTA's
  auto sums_full = [&](uint32_t c) { return bar0 + 8 * (2 * kStages + c); };
  auto sums_empty = [&](uint32_t c) { return bar0 + 8 * (2 * kStages + 2 + c); };  // the leader's
  volatile uint32_t *const stop = &abort_flag;
  if (threadIdx.x == 0) {
    for (uint32_t s = 0; s < kStages; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (uint32_t c = 0; c < 2; ++c) {
      mbar_init(sums_full(c), 1);
      mbar_init(sums_empty(c), 2 * kEpiWarps);
    }
    abort_flag = 0;
    fence_mbar_init();
  }
  __syncwarp();
  if (warp == 0) tmem_alloc_pair(smem_u32(&tmem_slot), kTmemCols);
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  auto wait = [&](uint32_t bar, uint32_t parity) { return mbar_try_wait(bar, parity & 1) || wait_longer(bar, parity & 1, stop, a.err); };
  const uint32_t pair = blockIdx.x / 2, pairs = gridDim.x / 2, steps = (a.k + kBK - 1) / kBK;
  // this CTA's first row of weights of a unit, and the copies that bring its rows
  auto w_row = [&](const Unit &u) -> int32_t { return u.col * kCols + u.part * (kCols >> u.lg) + (GATED ? 0 : rank * (kBN / 2 >> u.lg)); };
  auto w_map = [&](const Unit &u) { return u.lg ? &maps.part[GATED ? rank : 0] : &maps.w[GATED ? rank : 0]; };
  if (threadIdx.x == 0 && pair < g.units) {  // the first weights are asked into L2 while the kernel before this one ends
    const Unit u = unit_at(g, pair);
    for (uint32_t k = 0; k < steps && k < kStages; ++k) tma_prefetch_2d(w_map(u), k * kBK, w_row(u));
  }
  __syncwarp();
  pdl_launch_dependents();
  pdl_wait();
  uint32_t it = 0;  // stages used, over all tiles
  if (warp == 0) {  // (the whole warp, so that addresses are the same in all lanes; one thread issues)
    const uint32_t leader_full = in_cta(full(0), 0);
    for (uint32_t i = pair; i < g.units; i += pairs) {
      const Unit u = unit_at(g, i);
      const int32_t x_row = u.row * kBM + rank * kHalf, w0 = w_row(u);
      const CUtensorMap *const w = w_map(u);
      const uint32_t bytes = 2 * (kATile + (kBTile >> u.lg));  // of both CTAs
      bool ok = true;
      for (uint32_t k = 0; k < steps; ++k, ++it) {
        const uint32_t s = it % kStages, at = base + s * kStage, bar = leader_full + 8 * s;
        if (it >= kStages && !(ok = __all_sync(0xffffffffu, wait(empty(s), it / kStages - 1)))) break;
        if (elect_one()) {
          if (rank == 0) mbar_arrive_expect_tx(full(s), bytes);
          tma_load_pair(at, &maps.x, k * kBK, x_row, bar);
          tma_load_pair(at + kATile, w, k * kBK, w0, bar);
        }
        __syncwarp();
      }
      if (!ok) break;
    }
  } else if (warp == 1 && rank == 0) {
    // (the whole warp, so that descriptors are the same in all lanes; one thread issues)
    uint32_t n = 0;
    for (uint32_t i = pair; i < g.units; i += pairs, ++n) {
      const uint32_t d = tmem + n % 2 * kBN, idesc = umma_idesc_i8(kBM, kBN >> (i < g.whole ? 0 : g.part));
      if (n >= 2 && !__all_sync(0xffffffffu, wait(sums_empty(n & 1), n / 2 - 1))) break;
      tc_fence_after();
      bool ok = true;
      for (uint32_t k = 0; k < steps; ++k, ++it) {
        const uint32_t s = it % kStages, at = base + s * kStage;
        if (!(ok = __all_sync(0xffffffffu, wait(full(s), it / kStages)))) break;
        tc_fence_after();
        const uint64_t x = umma_desc_sw128(at), w = umma_desc_sw128(at + kATile);
        if (elect_one()) {
#pragma unroll
          for (uint32_t j = 0; j < kBK / 32; ++j) umma_i8_pair(d, x + 2 * j, w + 2 * j, idesc, k > 0 || j > 0);
          umma_commit_pair(empty(s));
          if (k + 1 == steps) umma_commit_pair(sums_full(n & 1));
        }
        __syncwarp();
      }
      if (!ok) break;
    }
  } else if (warp >= 2) {
    constexpr uint32_t kBoxCols = 128 / sizeof(T), kPer = kBoxCols / 32;  // columns of a box, loads of 32 of them
    constexpr uint32_t kBoxes = kCols / kBoxCols, kMine = (kBoxes + 1) / 2 * kPer;  // of a tile; of a warp, loads
    static_assert(kCols % kBoxCols == 0, "whole boxes");
    const uint32_t q = warp & 3, odd = (warp - 2) / 4, box = base + kStages * kStage + (warp - 2) * kBox;
    float(&cs)[GATED ? 2 : 1][32] = sh.col_scale[warp - 2];
    const uint64_t first_out = l2_evict_first_policy();
    auto first = [&](uint32_t i) { return (odd + 2 * (i / kPer)) * kBoxCols + i % kPer * 32; };  // column of load i
    // Scales of a tile, a row's and the columns' a lane each: a tile ahead, as they come from L2.
    struct Scales {
      uint32_t t0, n0, lg;
      float x, w[GATED ? 2 : 1][kMine];
    };
    auto scales_of = [&](uint32_t i, Scales &sc) {
      if (i >= g.units) return;
      const Unit u = unit_at(g, i);
      sc.t0 = u.row * kBM + rank * kHalf + 32 * q;
      sc.n0 = u.col * kCols + u.part * (kCols >> u.lg);
      sc.lg = u.lg;
      sc.x = sc.t0 + lane < a.t ? a.x_scale[sc.t0 + lane] : 0.0f;
#pragma unroll
      for (uint32_t m = 0; m < (GATED ? 2 : 1); ++m)
#pragma unroll
        for (uint32_t k = 0; k < kMine; ++k) {
          const uint32_t nc = sc.n0 + first(k) + lane;
          sc.w[m][k] = first(k) < kCols && nc < a.n ? a.w_scale[m][nc] : 0.0f;
        }
    };
    uint32_t n = 0;
    Scales next;
    scales_of(pair, next);
    for (uint32_t i = pair; i < g.units; i += pairs, ++n) {
      Scales now = next;
      scales_of(i + pairs, next);
      const uint32_t t0 = now.t0, n0 = now.n0, src = tmem + ((32 * q) << 16) + n % 2 * kBN, cols = kCols >> now.lg;
      const float xs = now.x;
      float(&ws)[GATED ? 2 : 1][kMine] = now.w;
      const bool ok = wait(sums_full(n & 1), n / 2);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      auto drained = [&] {  // this warp has read its sums
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(in_cta(sums_empty(n & 1), 0));
      };
      if (first(0) >= cols) drained();
#pragma unroll 1
      for (uint32_t k = 0; k < kMine && first(k) < cols; ++k) {
        const uint32_t c = first(k);
        uint32_t r[32], u[GATED ? 32 : 1];
        tmem_ld32(src + c, r);
        if constexpr (GATED) tmem_ld32(src + cols + c, u);
        __syncwarp();  // the scales of the columns before have been read
#pragma unroll
        for (uint32_t m = 0; m < (GATED ? 2 : 1); ++m) {
          cs[m][lane] = ws[m][0];
#pragma unroll
          for (uint32_t w = 0; w + 1 < kMine; ++w) ws[m][w] = ws[m][w + 1];
        }
        const uint32_t half = k % kPer;
        if (half == 0 && lane == 0) bulk_wait_read<0>();  // the box's store before has read it
        __syncwarp();
        tmem_wait_ld(r);
        if constexpr (GATED) tmem_wait_ld(u);
        if (k + 1 == kMine || first(k + 1) >= cols) drained();
        float v[32];
#pragma unroll
        for (uint32_t j = 0; j < 32; j += 2) {
          float2 y = i8_value2((int32_t)r[j], (int32_t)r[j + 1], xs, *reinterpret_cast<const float2 *>(&cs[0][j]));
          if constexpr (GATED)
            y = i8_gated2(y, i8_value2((int32_t)u[j], (int32_t)u[j + 1], xs, *reinterpret_cast<const float2 *>(&cs[1][j])));
          v[j] = y.x;
          v[j + 1] = y.y;
        }
        const uint32_t line = box + lane * 128, sw = lane & 7;
#pragma unroll
        for (uint32_t j = 0; j < 32 * sizeof(T) / 16; ++j) {
          uint32_t w[4];
#pragma unroll
          for (uint32_t e = 0; e < 4; ++e) {
            if constexpr (sizeof(T) == 4) {
              w[e] = __float_as_uint(v[4 * j + e]);
            } else {
              const __nv_bfloat162 b = __floats2bfloat162_rn(v[8 * j + 2 * e], v[8 * j + 2 * e + 1]);
              w[e] = *reinterpret_cast<const uint32_t *>(&b);
            }
          }
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(line + (((half * 4 + j) ^ sw) << 4)), "r"(w[0]), "r"(w[1]),
                       "r"(w[2]), "r"(w[3])
                       : "memory");
        }
        if (half + 1 < kPer) continue;
        const uint32_t c0 = n0 + c - half * 32;
        if (c0 + kBoxCols <= g.boxes) {
          fence_proxy_async();  // generic-proxy writes -> the TMA engine's reads
          __syncwarp();
          if (lane == 0 && c0 < a.n && t0 < a.t) {
            if (g.far)  // (neither stores what is past t and n)
              tma_store_2d_far(&maps.y, (int32_t)c0, (int32_t)t0, box, first_out);
            else
              tma_store_2d(&maps.y, (int32_t)c0, (int32_t)t0, box);
            bulk_commit();
          }
        } else {
          __syncwarp();
          constexpr uint32_t kOnce = 8;
#pragma unroll 1
          for (uint32_t r0 = 0; r0 < 32 && t0 + r0 < a.t; r0 += kOnce) {
            T v[kOnce][kPer];
#pragma unroll
            for (uint32_t rr = 0; rr < kOnce; ++rr)
#pragma unroll
              for (uint32_t e = 0; e < kPer; ++e) {
                const uint32_t c = e * 32 + lane, row = r0 + rr;
                v[rr][e] = ld_shared<T>(box + row * 128 + (((c * (uint32_t)sizeof(T) / 16) ^ (row & 7)) << 4) + c * (uint32_t)sizeof(T) % 16);
              }
#pragma unroll
            for (uint32_t rr = 0; rr < kOnce; ++rr)
#pragma unroll
              for (uint32_t e = 0; e < kPer; ++e)
                if (t0 + r0 + rr < a.t && c0 + e * 32 + lane < a.n)
                  static_cast<T *>(a.y)[(size_t)(t0 + r0 + rr) * a.y_ld + c0 + e * 32 + lane] = v[rr][e];
          }
          __syncwarp();
        }
      }
    }
    if (lane == 0) bulk_wait_all();
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && rank == 0 && *stop)  // a stopped pair waits (bounded) for the copies that it issued
    for (uint32_t s = 0; s < kStages && s < it; ++s) mbar_wait_bounded(full(s), ((it - 1 - s) / kStages) & 1);
  __syncwarp();
  cluster_sync();  // no CTA leaves while the other's products, copies or arrivals may reach it
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, kTmemCols);
  }
}

// ---- few rows of x, or few tiles: weights as the rows of the products
// 128 columns of y (rows of weights) are the M of the product and up to 256 rows of x its N, so that no row of the
// tensor memory is spent on rows of x that are not there; the CTAs of a cluster share a tile, each with a part of
// K, and each then adds up what all of them have of every so-manieth row of x: whole numbers, so the order does not
// matter and no memory but theirs is needed.  It reads the rows of x once for 128 columns, which bounds it from some
// 100 rows on: 17 rows of 3840 x 15360 13.5 us (4.4 TB/s of weights), 128 rows 16, 256 rows 21, where copies from L2
// run at 110 KB a us and SM; what starting and ending costs is 3.3 us of each.  Tiles half as deep in shared
// memory, so that the next call's CTAs find room beside these, took 14.6, 21.5 and 29.8.
constexpr uint32_t kWRows = 128, kWTile = kWRows * kBK;
struct SplitShape {
  uint32_t tok;        // rows of x of a tile: a multiple of 16
  uint32_t stages, cluster, tmem_cols;
};

SX_DEV void umma_i8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
SX_DEV void ld_shared_v4(uint32_t src, int32_t (&v)[4]) {
  asm volatile("ld.shared.v4.s32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(src) : "memory");
}
SX_DEV void ld_cluster_v4(uint32_t src, int32_t (&v)[4]) {
  asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(src) : "memory");
}

template <typename T, bool GATED>
__global__ void __launch_bounds__(kThreads)
    gemm_i8_split_kernel(const __grid_constant__ Maps maps, const __grid_constant__ I8Args a, const __grid_constant__ SplitShape p) {
  constexpr uint32_t kMats = GATED ? 2 : 1, kMaxStages = 12;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bars[2 * kMaxStages + 1];
  __shared__ uint32_t tmem_slot, abort_flag;
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = blockIdx.x % p.cluster;
  const uint32_t base = (smem_u32(smem_raw) + 1023) & ~1023u, bar0 = smem_u32(bars), stage_bytes = kMats * kWTile + p.tok * kBK;
  auto full = [&](uint32_t s) { return bar0 + 8 * s; };
  auto empty = [&](uint32_t s) { return bar0 + 8 * (kMaxStages + s); };
  const uint32_t done = bar0 + 16 * kMaxStages;
  const uint32_t n0 = blockIdx.x / p.cluster * kWRows, t0 = blockIdx.y * p.tok;
  const uint32_t all = (a.k + kBK - 1) / kBK, k0 = all * rank / p.cluster, steps = all * (rank + 1) / p.cluster - k0;
  volatile uint32_t *const stop = &abort_flag;
  if (threadIdx.x == 0) {
    for (uint32_t s = 0; s < p.stages; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    mbar_init(done, 1);
    abort_flag = 0;
    fence_mbar_init();
    // asked into L2 while the kernel before this one ends
    for (uint32_t i = 0; i < steps && i < p.stages; ++i)
#pragma unroll
      for (uint32_t m = 0; m < kMats; ++m) tma_prefetch_2d(&maps.w[m], (k0 + i) * kBK, n0);
  }
  __syncwarp();
  if (warp == 0) {
    tmem_alloc(smem_u32(&tmem_slot), p.tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  auto wait = [&](uint32_t bar, uint32_t parity) { return mbar_try_wait(bar, parity & 1) || wait_longer(bar, parity & 1, stop, a.err); };
  pdl_launch_dependents();
  pdl_wait();
  uint32_t issued = 0;
  bool ok = false;
  if (warp == 0) {  // (whole warps, so that addresses are the same in all lanes; one thread issues)
    for (uint32_t i = 0, s = 0, round = 0; i < steps; ++i) {
      const uint32_t at = base + s * stage_bytes;
      if (round > 0 && !__all_sync(0xffffffffu, wait(empty(s), round - 1))) break;
      if (elect_one()) {
        mbar_arrive_expect_tx(full(s), stage_bytes);
#pragma unroll
        for (uint32_t m = 0; m < kMats; ++m) tma_load_2d(at + m * kWTile, &maps.w[m], (k0 + i) * kBK, n0, full(s));
        tma_load_2d(at + kMats * kWTile, &maps.x, (k0 + i) * kBK, t0, full(s));
      }
      __syncwarp();
      issued = i + 1;
      if (++s == p.stages) s = 0, ++round;
    }
  } else if (warp == 1) {
    const uint32_t idesc = umma_idesc_i8(kWRows, p.tok);
    for (uint32_t i = 0, s = 0, round = 0; i < steps; ++i) {
      const uint32_t at = base + s * stage_bytes;
      if (!__all_sync(0xffffffffu, wait(full(s), round))) break;
      tc_fence_after();
      const uint64_t x = umma_desc_sw128(at + kMats * kWTile);
      if (elect_one()) {
#pragma unroll
        for (uint32_t m = 0; m < kMats; ++m) {
          const uint64_t w = umma_desc_sw128(at + m * kWTile);
#pragma unroll
          for (uint32_t j = 0; j < kBK / 32; ++j) umma_i8(tmem + m * p.tok, w + 2 * j, x + 2 * j, idesc, i > 0 || j > 0);
        }
        umma_commit(empty(s));
        if (i + 1 == steps) umma_commit(done);
      }
      __syncwarp();
      if (++s == p.stages) s = 0, ++round;
    }
  }
  // ---- sums to shared memory, over the tiles: [row of x][matrix][128]
  const uint32_t rows = min(p.tok, a.t - t0), epi = warp - 2;  // rows of x
  // This warp's rows of x further on, and the scale of the lane-th of them: here before the sums are.
  const uint32_t mine = rank + p.cluster * epi, apart = p.cluster * kEpiWarps;
  static_assert(32 * kEpiWarps >= 256, "a lane for each of a warp's rows");
  const float xs_mine = warp >= 2 && mine + lane * apart < rows ? a.x_scale[t0 + mine + lane * apart] : 0.0f;
  if (warp >= 2) {
    ok = wait(done, 0);
    ok = __all_sync(0xffffffffu, ok);
    tc_fence_after();
    const uint32_t q = warp & 3, src = tmem + ((32 * q) << 16), dst = base + (32 * q + lane) * 4;
#pragma unroll 1
    for (uint32_t c = epi / 4 * 16; c < rows; c += 32)
#pragma unroll
      for (uint32_t m = 0; m < kMats; ++m) {
        uint32_t r[16];
        tmem_ld16(src + m * p.tok + c, r);
        tmem_wait_ld(r);
#pragma unroll
        for (uint32_t j = 0; j < 16; ++j)
          asm volatile("st.shared.b32 [%0], %1;\n" ::"r"(dst + ((c + j) * kMats + m) * kWRows * 4), "r"(r[j]) : "memory");
      }
  }
  __syncwarp();
  if (p.cluster > 1)
    cluster_sync();
  else
    __syncthreads();
  // ---- a warp takes rows of x, four columns a lane; a CTA's rows are every p.cluster-th
  if (warp >= 2 && ok) {
    const uint32_t n = n0 + 4 * lane, at = base + lane * 16;
    float ws[kMats][4];
#pragma unroll
    for (uint32_t m = 0; m < kMats; ++m)
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) ws[m][j] = n + j < a.n ? a.w_scale[m][n + j] : 0.0f;
    constexpr uint32_t es = sizeof(T);
    const bool wide = (reinterpret_cast<uintptr_t>(a.y) | (uintptr_t)a.y_ld * es) % (4 * es) == 0 && n + 4 <= a.n;
    auto store = [&](uint32_t c, uint32_t nth, const int32_t (&sum)[kMats][4]) {
      const float xs = __shfl_sync(0xffffffffu, xs_mine, nth);
      float v[4];
#pragma unroll
      for (uint32_t j = 0; j < 4; ++j) {
        v[j] = i8_value(sum[0][j], xs, ws[0][j]);
        if constexpr (GATED) v[j] = i8_gated(v[j], i8_value(sum[kMats - 1][j], xs, ws[kMats - 1][j]));
      }
      T *const y = static_cast<T *>(a.y) + (size_t)(t0 + c) * a.y_ld + n;
      if (wide) {
        store_vec<T, 4>(y, v);
      } else {
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j)
          if (n + j < a.n) y[j] = i8_out<T>(v[j]);
      }
    };
    // (a load's result is hundreds of cycles away: all CTAs' parts of a row, or several rows, at a time)
    auto rows_of = [&](auto parts, auto at_once) {
      constexpr uint32_t kParts = decltype(parts)::value, kOnce = decltype(at_once)::value;
#pragma unroll 1
      for (uint32_t c = mine, nth = 0; c < rows; c += kOnce * apart, nth += kOnce) {
        int32_t v[kOnce][kParts][kMats][4];
#pragma unroll
        for (uint32_t o = 0; o < kOnce; ++o) {
          const uint32_t row = min(c + o * apart, rows - 1) * kMats * kWRows * 4 + at;
#pragma unroll
          for (uint32_t i = 0; i < kParts; ++i)
#pragma unroll
            for (uint32_t m = 0; m < kMats; ++m)
              if constexpr (kParts == 1)
                ld_shared_v4(row + m * kWRows * 4, v[o][i][m]);
              else
                ld_cluster_v4(in_cta(row + m * kWRows * 4, i), v[o][i][m]);
        }
#pragma unroll
        for (uint32_t o = 0; o < kOnce; ++o) {
#pragma unroll
          for (uint32_t i = 1; i < kParts; ++i)
#pragma unroll
            for (uint32_t m = 0; m < kMats; ++m)
#pragma unroll
              for (uint32_t j = 0; j < 4; ++j) v[o][0][m][j] += v[o][i][m][j];
          if (c + o * apart < rows) store(c + o * apart, nth + o, v[o][0]);
        }
      }
    };
    using One = std::integral_constant<uint32_t, 1>;
    using Two = std::integral_constant<uint32_t, 2>;
    using Four = std::integral_constant<uint32_t, 4>;
    using Eight = std::integral_constant<uint32_t, 8>;
    if (p.cluster == 1)
      rows_of(One{}, Four{});
    else if (p.cluster == 2)
      rows_of(Two{}, Two{});
    else if (p.cluster == 4)
      rows_of(Four{}, One{});
    else
      rows_of(Eight{}, One{});
  }
  __syncwarp();
  if (p.cluster > 1) cluster_sync();  // the others have read this CTA's sums
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *stop)  // a stopped CTA waits (bounded) for the copies that it issued
    for (uint32_t s = 0; s < p.stages && s < issued; ++s) mbar_wait_bounded(full(s), ((issued - 1 - s) / p.stages) & 1);
  __syncwarp();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, p.tmem_cols);
  }
}

bool encode(CUtensorMap *map, CUtensorMapDataType type, const void *p, uint64_t cols, uint64_t rows, uint64_t ld_bytes, uint32_t box_cols,
            uint32_t box_rows) {
  auto fn = tensor_map_encoder();
  const cuuint64_t dims[2] = {cols, rows}, strides[1] = {ld_bytes};
  const cuuint32_t box[2] = {box_cols, box_rows}, one[2] = {1, 1};
  return fn && fn(map, type, 2, const_cast<void *>(p), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

using PairKernel = void (*)(const Maps, const I8Args, const Tiles);
PairKernel pair_kernel(uint32_t dtype, bool gated) {
  if (dtype == SX_F32) return gated ? gemm_i8_pair_kernel<float, true> : gemm_i8_pair_kernel<float, false>;
  return gated ? gemm_i8_pair_kernel<__nv_bfloat16, true> : gemm_i8_pair_kernel<__nv_bfloat16, false>;
}

struct PairPlan {
  Tiles g;
  float us;
};
constexpr uint64_t kGroupBytes = 32u << 20;

// Tiles that are left when all pairs have had as many whole ones are taken in parts of half or a quarter of the
// columns, so that more pairs have one (768 x 8192 x 3840 23.8 us, in halves 21.4; 1024 x 5000 x 4096 27.2, in quarters
// 22.2).  The time, by what was measured: 5 us beside the steps of 128 of K, and those 0.31 us (0.42 and more at the
// clock that the power cap leaves in calls of 100 us, where there is no other choice), three quarters of it for a half.
// Tiles with little K wait for their values (2.7 us each), and lanes store for 0.4 us longer.  Weights that L2 does
// not hold come at 5 TB/s.
PairPlan pair_plan(uint32_t dtype, bool gated, const I8Args &a, uint32_t pairs) {
  PairPlan p{};
  const uint32_t es = dtype == SX_F32 ? 4 : 2, steps = (a.k + kBK - 1) / kBK, cols = gated ? kBN / 2 : kBN;
  p.g.rows = (a.t + kBM - 1) / kBM;
  p.g.cols = (a.n + cols - 1) / cols;
  const uint32_t all = p.g.rows * p.g.cols, left = all % pairs;
  p.g.whole = all - left;
  // (quarters only behind whole tiles: 1024 x 1024 x 1024 in halves 5.5 us, in quarters 6.7; and a box of y is 128
  // bytes, where a quarter of a gated tile has 32 columns)
  p.g.part = left * 4 <= pairs && p.g.whole > 0 && !(gated && es == 2) ? 2 : left * 2 <= pairs ? 1 : 0;
  if (left == 0) p.g.part = 0;
  p.g.units = p.g.whole + (left << p.g.part);
  // Rows of x that stay in L2 while the columns' weights go by: the more there are, the fewer times that weights which
  // do not fit L2 come from memory (118 MB of gate and up, 16896 rows of 3840: 8, 16, 32 tiles 1466, 1419, 1400 us), but
  // not past what L2 keeps (16384 rows of 15360: 696, 725, 788).
  p.g.group = (uint32_t)std::min<uint64_t>(32, std::max<uint64_t>(1, kGroupBytes / ((uint64_t)kBM * a.k)));
  // Copies store rows that begin on 16 bytes, and of those whole 16 bytes: where a row ends inside them, its last box
  // is left to lanes (8192 x 8191 x 512, rows 8192 apart: f32 67 -> 60 us, bf16 54 -> 36).  Rows that begin anywhere are
  // the lanes' (8191 apart: 95 and 55 us).  Their stores cut sectors in two; shifted by rows into whole lines, through
  // registers that keep what is left of a box, they take twelve instructions a row and box for four, and 135 us.
  p.g.boxes = ((uintptr_t)a.y | (uintptr_t)a.y_ld * es) % 16 != 0 ? 0 : (uint64_t)a.n * es % 16 != 0 ? a.n : ~0u;
  // (16896 x 8192 of f32: 438 -> 433 us; 8192 x 8192 x 512 72.6 -> 69)
  p.g.far = (uint64_t)a.t * a.n * es > (128u << 20);
  const float memory = (gated ? 2.0f : 1.0f) * (float)a.n * (float)a.k * (1.0f / 5.0e6f);
  const float turns = (float)(all / pairs), waves = turns + (left ? 1.0f : 0.0f);
  const float ragged = (a.w_ld | a.x_ld) % 128 != 0 ? 1.2f : 1.0f;  // rows that begin inside a line
  const float step = 0.31f * ragged, last = left == 0 ? 0.0f : std::max((p.g.part == 2 ? 0.5f : p.g.part == 1 ? 0.75f : 1.0f) * step * steps, p.g.part ? 1.5f : 2.7f);
  p.us = (turns > 0.0f || p.g.part == 0 ? 5.0f : gated ? 3.5f : 4.0f) + std::max(turns * std::max(step * steps, 2.7f) + last, memory);
  if (p.g.boxes == 0) p.us += waves * 0.4f;
  return p;
}

cudaError_t launch_pair(uint32_t dtype, bool gated, const I8Args &a, const PairPlan &p, uint32_t pairs, cudaStream_t s) {
  const uint32_t es = dtype == SX_F32 ? 4 : 2;
  Maps maps{};
  bool ok = encode(&maps.x, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.x, a.k, a.t, a.x_ld, kBK, kHalf);
  for (int i = 0; i < (gated ? 2 : 1); ++i) {
    if (p.g.whole || !p.g.part) ok = ok && encode(&maps.w[i], CU_TENSOR_MAP_DATA_TYPE_UINT8, a.w[i], a.k, a.n, a.w_ld, kBK, kBN / 2);
    if (p.g.part) ok = ok && encode(&maps.part[i], CU_TENSOR_MAP_DATA_TYPE_UINT8, a.w[i], a.k, a.n, a.w_ld, kBK, kBN / 2 >> p.g.part);
  }
  if (p.g.boxes != 0)
    ok = ok && encode(&maps.y, dtype == SX_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, a.y, a.n, a.t,
                      (uint64_t)a.y_ld * es, 128 / es, 32);
  if (!ok) return cudaErrorInvalidValue;
  return launch_chained(pair_kernel(dtype, gated), dim3(2 * std::min(p.g.units, pairs)), dim3(kThreads), kMaxSmem, s, 2, maps, a, p.g);
}

using SplitKernel = void (*)(const Maps, const I8Args, const SplitShape);
SplitKernel split_kernel(uint32_t dtype, bool gated) {
  if (dtype == SX_F32) return gated ? gemm_i8_split_kernel<float, true> : gemm_i8_split_kernel<float, false>;
  return gated ? gemm_i8_split_kernel<__nv_bfloat16, true> : gemm_i8_split_kernel<__nv_bfloat16, false>;
}
constexpr uint32_t kSplitSmem = 220 * 1024, kSplitSmemTwo = 108 * 1024;  // one CTA an SM, two

struct SplitPlan {
  SplitShape p;
  uint32_t n_tiles, t_tiles, smem;
  float us;
};
// The time, by what was measured: 3.3 us, the stages at 110 KB a us and SM or the weights at 6.2 TB/s, whichever is
// longer, and 13 ns for each row of a tile and matrix.
SplitPlan split_plan(bool gated, const I8Args &a, const uint32_t (&clusters)[4]) {
  const uint32_t mats = gated ? 2 : 1, most = gated ? 128 : 256, steps = (a.k + kBK - 1) / kBK;
  SplitPlan s{};
  s.t_tiles = (a.t + most - 1) / most;
  s.n_tiles = (a.n + kWRows - 1) / kWRows;
  s.p.tok = ((a.t + s.t_tiles - 1) / s.t_tiles + 15) / 16 * 16;
  s.t_tiles = (a.t + s.p.tok - 1) / s.p.tok;
  const uint64_t tiles = (uint64_t)s.n_tiles * s.t_tiles;
  const uint32_t stage = mats * kWTile + s.p.tok * kBK;
  s.p.cluster = 1;
  for (uint32_t i = 1; i < 4 && tiles <= clusters[i] && (2u << i) <= steps; ++i) s.p.cluster = 1u << i;
  s.p.tmem_cols = 32;
  while (s.p.tmem_cols < mats * s.p.tok) s.p.tmem_cols *= 2;
  const uint32_t sums = s.p.tok * mats * kWRows * 4;
  const bool two = tiles > clusters[0];  // CTAs an SM, where there are more than SMs
  s.p.stages = std::min(12u, ((two ? kSplitSmemTwo : kSplitSmem) - 1024) / stage);
  s.smem = std::max(s.p.stages * stage, sums) + 1024;  // the stages, then the sums
  const float waves = !two ? 1.0f : s.smem <= kSplitSmemTwo ? (float)tiles / (float)clusters[0] : (float)((tiles + clusters[0] - 1) / clusters[0]);
  const float ragged = (a.w_ld | a.x_ld) % 128 != 0 ? 1.3f : 1.0f;  // rows that begin inside a line
  const float few = two && s.p.stages < 3 ? 1.6f : 1.0f;  // (275 x 16078 x 2688, gate and up: 45 us; tiles of pairs 31.5)
  const float load = few * ragged * (float)((steps + s.p.cluster - 1) / s.p.cluster) * (float)stage * (1.0f / 110e3f);
  const float memory = (float)mats * (float)a.n * (float)a.k * (1.0f / 6.2e6f);
  const float values = 0.013f * (float)(s.p.tok * mats);
  // (CTAs that have an SM for themselves start when the ones before have ended)
  s.us = two && s.smem > kSplitSmemTwo ? waves * (3.3f + load + values) : 3.3f + std::max(waves * load, memory) + waves * values;
  return s;
}

cudaError_t launch_split(uint32_t dtype, bool gated, const I8Args &a, const SplitPlan &p, cudaStream_t s) {
  Maps maps{};
  bool ok = encode(&maps.x, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.x, a.k, a.t, a.x_ld, kBK, p.p.tok);
  for (int i = 0; i < (gated ? 2 : 1); ++i) ok = ok && encode(&maps.w[i], CU_TENSOR_MAP_DATA_TYPE_UINT8, a.w[i], a.k, a.n, a.w_ld, kBK, kWRows);
  if (!ok) return cudaErrorInvalidValue;
  return launch_chained(split_kernel(dtype, gated), dim3(p.n_tiles * p.p.cluster, p.t_tiles), dim3(kThreads), p.smem, s, p.p.cluster, maps, a, p.p);
}

// Few rows or few tiles: weights as the rows of the products; else tiles of pairs.
cudaError_t launch_tiles(uint32_t dtype, bool gated, const I8Args &a, const uint32_t (&clusters)[4], cudaStream_t s) {
  const PairPlan pair = pair_plan(dtype, gated, a, clusters[1]);
  const SplitPlan split = split_plan(gated, a, clusters);
  if (split.t_tiles <= 65535 && split.us < pair.us) return launch_split(dtype, gated, a, split, s);
  return launch_pair(dtype, gated, a, pair, clusters[1], s);
}

}  // namespace

cudaError_t prepare_gemm_i8(uint32_t (&clusters)[4]) {
  for (uint32_t dtype : {SX_F32, SX_BF16})
    for (bool gated : {false, true}) {
      const cudaError_t e = cudaFuncSetAttribute(split_kernel(dtype, gated), cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSplitSmem);
      if (e != cudaSuccess) return e;
    }
  for (uint32_t i = 0; i < 4; ++i) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = 1u << i;
    at.val.clusterDim.y = at.val.clusterDim.z = 1;
    cfg.gridDim = dim3(1u << i);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSplitSmem;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    int n = 0;
    const cudaError_t e = cudaOccupancyMaxActiveClusters(&n, split_kernel(SX_F32, false), &cfg);
    if (e != cudaSuccess) return e;
    clusters[i] = (uint32_t)std::max(n, 1);
  }
  for (uint32_t dtype : {SX_F32, SX_BF16})
    for (bool gated : {false, true}) {
      const cudaError_t e = cudaFuncSetAttribute(pair_kernel(dtype, gated), cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMaxSmem);
      if (e != cudaSuccess) return e;
    }
  return prepare_gemv_i8();
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
  if (a.t && (!a.x || !a.x_scale || !a.y)) return bad("null x, x_scale or y");  // (an empty tensor has no address)
  if ((uintptr_t)a.x_scale % 4 != 0) return bad("scales must be aligned to their elements");
  if (a.k == 0 || a.k % 16 != 0 || a.k >= sx::kI8MaxK) return bad("k must be a multiple of 16, above 0 and below 131072");
  if (a.n == 0) return bad("n must be above 0");
  if (a.x_ld < a.k || a.w_ld < a.k || a.y_ld < a.n) return bad("row strides are shorter than a row");
  if (al % 16 != 0) return bad("x and weights must be 16-byte aligned and their strides multiples of 16");
  if ((uintptr_t)a.y % (dtype == SX_F32 ? 4 : 2) != 0) return bad("y must be aligned to its elements");
  if (a.t >= (1u << 31) || a.n >= (1u << 31)) return bad("t and n must be below 2^31");
  if ((uint64_t)a.t * a.n >= (1ull << 42)) return bad("t * n must be below 2^42");  // (tiles are counted in 32 bits)
  if (!e) return bad("null engine");
  if (a.t == 0) return SX_OK;
  const cudaError_t ce = cudaSetDevice(e->device);
  if (ce != cudaSuccess) return sx_host_cuda_status(ce, "cudaSetDevice");
  a.err = e->err_dev;
  // Streaming the weights; many short rows of them are few steps for each of its CTAs (32768 x 1024: 1 row 9.7 us, as
  // tiles 8.1; 16 rows 11.9, 8.0; 32768 x 4096: 1 row 22.7 us).
  const bool stream = a.t <= sx::kI8GemvRows && (a.k > 2048 || a.n <= (gated ? 48u : 96u) * (uint32_t)e->num_sms);
  return sx_host_cuda_status(stream ? sx::launch_gemv_i8(dtype, gated, a, e->num_sms, e->stream)
                                    : sx::launch_tiles(dtype, gated, a, e->i8_clusters, e->stream), what);
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
