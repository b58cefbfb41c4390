// sx_kv8_append.cu -- new rows into the paged 8-bit KV cache: q / k RMS norm, position rotation,
// e4m3 quantisation with one power-of-two scale per 16 tokens and kv head (include/sx.h,
// sx_dispatch_kv8_append).
//
//   q', k' = R(pos) (x / rms(x) * gain),  v' = v / rms(v),  stored = rn_e4m3(x' 2^-e),
//   e = min { e : max |record| <= 448 2^e }
//
// A record belongs to one CTA, which sees all of its new tokens, so the scale needs no atomics: a CTA
// takes one unit (sx_kv8_units.h), a 16-token block of one sequence, and a group of kv heads with their
// q heads.  The grid follows from the row and sequence counts alone and nothing is read back.
//
// Bound by the rows' bytes, and close behind by instructions: a vector of 256 has 45 cycles of an SM
// at the copy rate.  Half a warp takes a vector (a token of the unit each, when all 16 are new):
// its sums are four shuffle steps for two vectors at once.  Lane l of the half holds elements
// 64 k + 4 l .. + 3 of every chunk k, so that a rotation whose half is a multiple of 64 needs no
// exchange and a shorter one meets its pairs by shuffles within chunk 0.  The angles are computed
// once per unit.  K and V stay in registers until the block's maxima have met in shared memory, are
// converted by their owners, and leave through a byte tile that turns rows of tokens into the
// record's pieces.  Measured: 64 prompts of 16 to 512 tokens (16 q and 8 kv heads of 256, bf16) 135 us,
// 4.2 TB/s or 65 % of the measured copy rate, with 59 % of the issue slots used and warps that wait for their
// loads most (4.0 of the stalls per issue, at the 46 % of an SM's warps that registers leave); one token of 8
// sessions 6.5 us, the latency of its chain of loads (rows and lengths, page ids, the records' old bytes and
// scales).
#include "sx_host.h"
#include "sx_kv8.cuh"
#include "sx_launch.cuh"

namespace sx {
namespace {

constexpr int kAppThreads = 256;
constexpr int kWorkers = kAppThreads / 16;  // half warps

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

// shared memory: the byte tile (or a row of f32 per worker, for rotations whose pairs meet there),
// the gains of q and k, the angles' cosines and sines
SX_HD constexpr uint32_t append_tile_bytes(uint32_t d, bool rows) {
  return rows ? kWorkers * d * 4 : 2 * kKv8Block * (d + 32);
}

// Head size D: chunks of 16 lanes x 4 elements.
constexpr int kVec = 4, kChunk = 64;
template <int D>
using Elems = float[D / kChunk][kVec];

// the lanes of this thread's half warp, and sums and maxima over them
SX_DEV uint32_t half_mask() { return 0xFFFFu << (threadIdx.x & 16); }
SX_DEV float half_sum(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(half_mask(), v, o);
  return v;
}
SX_DEV float half_max(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(half_mask(), v, o));
  return v;
}

// A lane's part of a vector as it stands in memory.
template <typename T, int D>
struct Raw {
  static constexpr int kWords = kVec * (int)sizeof(T) / 4;
  uint32_t w[D / kChunk][kWords];
  SX_DEV void load(const T *p, uint32_t l) {
#pragma unroll
    for (int k = 0; k < D / kChunk; ++k) {
      const T *src = p + kChunk * k + kVec * l;
      if constexpr (kWords == 4) {
        const uint4 u = *reinterpret_cast<const uint4 *>(src);
        w[k][0] = u.x; w[k][1] = u.y; w[k][2] = u.z; w[k][3] = u.w;
      } else {
        const uint2 u = *reinterpret_cast<const uint2 *>(src);
        w[k][0] = u.x; w[k][1] = u.y;
      }
    }
  }
  SX_DEV void unpack(Elems<D> &x) const {
#pragma unroll
    for (int k = 0; k < D / kChunk; ++k)
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        if constexpr (sizeof(T) == 4)
          x[k][j] = __uint_as_float(w[k][j]);
        else
          x[k][j] = __uint_as_float(j & 1 ? w[k][j / 2] & 0xFFFF0000u : w[k][j / 2] << 16);
      }
  }
};
template <typename T, int D>
SX_DEV void store_vector(T *p, uint32_t l, const Elems<D> &x) {
#pragma unroll
  for (int k = 0; k < D / kChunk; ++k) store_vec<T, kVec>(p + kChunk * k + kVec * l, x[k]);
}

// x / rms(x)
template <int D>
SX_DEV void normalise(Elems<D> &x, float eps) {
  float ss = 0.0f;
#pragma unroll
  for (int k = 0; k < D / kChunk; ++k)
#pragma unroll
    for (int j = 0; j < kVec; ++j) ss = fmaf(x[k][j], x[k][j], ss);
  const float rs = rsqrtf(half_sum(ss) * (1.0f / D) + eps);
#pragma unroll
  for (int k = 0; k < D / kChunk; ++k)
#pragma unroll
    for (int j = 0; j < kVec; ++j) x[k][j] = __fmul_rn(x[k][j], rs);
}
template <int D>
SX_DEV void gain(Elems<D> &x, const float *w, uint32_t l) {
#pragma unroll
  for (int k = 0; k < D / kChunk; ++k) {
    float g[kVec];
    load_vec<float, kVec>(w + kChunk * k + kVec * l, g);
#pragma unroll
    for (int j = 0; j < kVec; ++j) x[k][j] = __fmul_rn(x[k][j], g[j]);
  }
}

// The rotation of one lane's elements.  Angles of a token: [cosines of the pairs | their sines].
enum TurnMode : int { kTurnShuffle, kTurnChunks, kTurnMemory };
inline TurnMode turn_mode(uint32_t half) {
  if (half <= kChunk / 2 && half % kVec == 0) return kTurnShuffle;
  return half == 64 || half == 128 || half == 256 ? kTurnChunks : kTurnMemory;
}
template <int D, TurnMode MODE>
struct Turn {
  uint32_t half;
  uint32_t peer, at;  // shuffles: the lane of the partners, this lane's first pair
  bool low, in;       //           first of the pairs; rotated at all
  SX_DEV Turn(uint32_t half_, uint32_t l) : half(half_), peer(0), at(0), low(false), in(false) {
    if (MODE == kTurnShuffle) {
      const uint32_t o = half / kVec;
      low = l < o;
      in = l < 2 * o;
      peer = (threadIdx.x & 16) | (low ? l + o : in ? l - o : l);
      at = in ? kVec * (low ? l : l - o) : 0;
    }
  }
  // every product and sum rounded by itself, as the engine's own rotation
  template <int H>
  SX_DEV void chunks(Elems<D> &x, const float *cs, uint32_t l) const {
    if constexpr (2 * H <= D / kChunk) {
#pragma unroll
      for (int k = 0; k < H; ++k) {
        float c[kVec], s[kVec];
        load_vec<float, kVec>(cs + kChunk * k + kVec * l, c);
        load_vec<float, kVec>(cs + half + kChunk * k + kVec * l, s);
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
          const float x0 = x[k][j], x1 = x[k + H][j];
          x[k][j] = __fsub_rn(__fmul_rn(x0, c[j]), __fmul_rn(x1, s[j]));
          x[k + H][j] = __fadd_rn(__fmul_rn(x0, s[j]), __fmul_rn(x1, c[j]));
        }
      }
    }
  }
  SX_DEV void operator()(Elems<D> &x, const float *cs, float *buf, uint32_t l) const {
    if constexpr (MODE == kTurnShuffle) {
      if (half == 0) return;  // no angles to read either
      float c[kVec], s[kVec];
      load_vec<float, kVec>(cs + at, c);
      load_vec<float, kVec>(cs + half + at, s);
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        const float y = __fmul_rn(__shfl_sync(half_mask(), x[0][j], peer), s[j]);
        const float r = __fadd_rn(__fmul_rn(x[0][j], c[j]), low ? -y : y);
        if (in) x[0][j] = r;
      }
    } else if constexpr (MODE == kTurnChunks) {
      if (half == 64)
        chunks<1>(x, cs, l);
      else if (half == 128)
        chunks<2>(x, cs, l);
      else
        chunks<4>(x, cs, l);
    } else {
      __syncwarp(half_mask());
#pragma unroll
      for (int k = 0; k < D / kChunk; ++k)
#pragma unroll
        for (int j = 0; j < kVec; ++j) buf[kChunk * k + kVec * l + j] = x[k][j];
      __syncwarp(half_mask());
#pragma unroll
      for (int k = 0; k < D / kChunk; ++k)
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
          const uint32_t d = kChunk * k + kVec * l + j;
          if (d < half)
            x[k][j] = __fsub_rn(__fmul_rn(x[k][j], cs[d]), __fmul_rn(buf[d + half], cs[half + d]));
          else if (d < 2 * half)
            x[k][j] = __fadd_rn(__fmul_rn(buf[d - half], cs[d]), __fmul_rn(x[k][j], cs[d - half]));
        }
    }
  }
};

// four rows' words of 4 bytes -> four words of one byte each row (a 4 x 4 byte transposition)
SX_DEV void transpose4(uint32_t (&w)[4]) {
  const uint32_t a = prmt(w[0], w[1], 0x5140), b = prmt(w[2], w[3], 0x5140);  // bytes 0, 1
  const uint32_t c = prmt(w[0], w[1], 0x7362), d = prmt(w[2], w[3], 0x7362);  // bytes 2, 3
  w[0] = prmt(a, b, 0x5410);
  w[1] = prmt(a, b, 0x7632);
  w[2] = prmt(c, d, 0x5410);
  w[3] = prmt(c, d, 0x7632);
}

struct Unit : Kv8Unit {
  uint32_t page, in_page;  // page and block of the page
};

// The kv heads [h0, h1) of a unit with their q heads.  FULL: all 16 tokens are new.
template <typename T, int D, TurnMode MODE, bool FULL>
SX_DEV void append_heads(const AppendArgs &a, const Unit &u, uint32_t h0, uint32_t h1, uint8_t *sh,
                         float (*amax)[2][kKv8Block]) {
  constexpr int kLd = D + 32;  // bytes of a tile row
  uint8_t *const tile = sh;    // [K, V][16][kLd]
  const int lane = threadIdx.x & 31;
  const uint32_t worker = threadIdx.x >> 4, l = threadIdx.x & 15;
  float *const buf = reinterpret_cast<float *>(sh) + worker * D;
  const float *const q_w = reinterpret_cast<const float *>(sh + append_tile_bytes(D, MODE == kTurnMemory));
  const float *const k_w = q_w + D, *const angles = k_w + D;  // [16][2 half]
  const uint32_t cnt = FULL ? kKv8Block : u.cnt, t0 = FULL ? 0 : u.t0;
  const bool fresh = t0 == 0;
  const Turn<D, MODE> turn(a.rot / 2, l);

  // Worker w takes token w % tw; with few tokens the vectors of one (K, V, then q heads) are dealt
  // to the workers that share it (tw and subs: powers of two).
  uint32_t tw = kWorkers;
  if (!FULL)
    while (tw > 1 && tw / 2 >= cnt) tw /= 2;
  const uint32_t t = worker & (tw - 1), sub = FULL ? 0 : worker / tw, subs = FULL ? 1 : kWorkers / tw;
  auto mine = [&](uint32_t w) { return FULL || (t < cnt && (w & (subs - 1)) == sub); };
  const size_t row = u.row0 + t;
  const T *const k_row = static_cast<const T *>(a.k) + row * a.k_ld;
  const T *const v_row = a.k_eq_v ? k_row : static_cast<const T *>(a.v) + row * a.v_ld;
  const T *const q_row = static_cast<const T *>(a.q) + row * a.q_ld;
  T *const q_dst = static_cast<T *>(a.q_out) + row * ((size_t)a.c.num_kv * a.gqa * D);
  const float *const cs = angles + t * a.rot;
  for (uint32_t h = h0; h < h1; ++h) {
    const uint32_t par = (h - h0) & 1;
    Raw<T, D> raw[2];  // K, V: on their way while the q heads are worked on
    if (mine(0)) raw[0].load(k_row + (size_t)h * D, l);
    if (mine(1)) raw[1].load(v_row + (size_t)h * D, l);
    if (MODE == kTurnMemory) __syncthreads();  // the rows of buf lie over the tile
    // ---- q heads of kv head h, the next one's load in flight
    if (FULL || t < cnt) {
      // vector 2 + g of a token belongs to worker (2 + g) % subs of it
      uint32_t g = (sub - 2) & (subs - 1);
      const T *src = q_row + (size_t)(h * a.gqa + g) * D;
      T *dst = q_dst + (size_t)(h * a.gqa + g) * D;
      Raw<T, D> next;
      if (g < a.gqa) next.load(src, l);
      for (; g < a.gqa; g += subs, dst += subs * D) {
        Elems<D> y;
        next.unpack(y);
        src += subs * D;
        if (g + subs < a.gqa) next.load(src, l);
        if (a.q_w) {
          normalise<D>(y, a.eps);
          gain<D>(y, q_w, l);
        }
        turn(y, cs, buf, l);
        store_vector<T, D>(dst, l, y);
      }
    }
    // ---- K and V
    Elems<D> x[2];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      if (!mine(w)) continue;
      raw[w].unpack(x[w]);
      if (w == 1) {
        if (a.v_norm) normalise<D>(x[w], a.eps);
      } else {
        if (a.k_w) {
          normalise<D>(x[w], a.eps);
          gain<D>(x[w], k_w, l);
        }
        turn(x[w], cs, buf, l);
      }
      float m = 0.0f;
#pragma unroll
      for (int k = 0; k < D / kChunk; ++k)
#pragma unroll
        for (int j = 0; j < kVec; ++j) m = fmaxf(m, fabsf(x[w][k][j]));  // a NaN does not count
      m = half_max(m);
      if (l == 0) amax[par][w][t] = m;
    }
    __syncthreads();
    // ---- the block's scales, and the owners' conversion
    const size_t rec = (((size_t)u.page * a.c.num_kv + h) * (a.c.page_tokens / kKv8Block) + u.in_page) * 2;
    int e_old[2], e[2];
    {
      float m = FULL || l < cnt ? amax[par][lane >> 4][l] : 0.0f;
      m = half_max(m);
      int was = kKv8MinExp;
      if (!fresh) was = kv8_scale_exponent(a.c.scale[rec + (lane >> 4)]);
      const int now = max(was, kv8_exponent(m));
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        e_old[w] = __shfl_sync(0xffffffffu, was, 16 * w);
        e[w] = __shfl_sync(0xffffffffu, now, 16 * w);
      }
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      if (!mine(w)) continue;
      const float inv = exp2_int(-e[w]);
      uint8_t *dst = tile + (w * kKv8Block + t0 + t) * kLd + kVec * l;
#pragma unroll
      for (int k = 0; k < D / kChunk; ++k)
        *reinterpret_cast<uint32_t *>(dst + kChunk * k) =
            e4m3_pack4(x[w][k][0] * inv, x[w][k][1] * inv, x[w][k][2] * inv, x[w][k][3] * inv);
    }
    __syncthreads();
    if (threadIdx.x < 2) a.c.scale[rec + threadIdx.x] = exp2_int(threadIdx.x ? e[1] : e[0]);
    // ---- 16-byte pieces of the K record, then of the V record
    uint8_t *const out = static_cast<uint8_t *>(a.c.data) + rec * (size_t)(kKv8Block * D);
    for (uint32_t i = threadIdx.x; i < 2 * D; i += kAppThreads) {
      const uint32_t w = i / D, p = i % D >> 5, g = (i & 31) >> 2, c = i & 3;
      const uint8_t *src = tile + w * kKv8Block * kLd + 32 * p;
      uint32_t v[4], is_new[4];  // the piece and which of its bytes are new
      if (w == 0) {
        const uint2 lo8 = *reinterpret_cast<const uint2 *>(src + g * kLd + 8 * c);
        const uint2 hi8 = *reinterpret_cast<const uint2 *>(src + (g + 8) * kLd + 8 * c);
        v[0] = lo8.x; v[1] = lo8.y; v[2] = hi8.x; v[3] = hi8.y;
        is_new[0] = is_new[1] = g - t0 < cnt ? 0xFFFFFFFFu : 0u;
        is_new[2] = is_new[3] = g + 8 - t0 < cnt ? 0xFFFFFFFFu : 0u;
      } else {
        uint32_t m = 0;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const uint32_t t = 2 * c + (s & 1) + 8 * (s >> 1);
          v[s] = *reinterpret_cast<const uint32_t *>(src + t * kLd + 4 * g);
          if (t - t0 < cnt) m |= 0xFFu << (8 * s);
        }
        transpose4(v);
        is_new[0] = is_new[1] = is_new[2] = is_new[3] = m;
      }
      uint4 *dst = reinterpret_cast<uint4 *>(out + 16 * i);
      if (!FULL && (is_new[0] & is_new[2]) != 0xFFFFFFFFu) {
        uint4 old = make_uint4(0, 0, 0, 0);
        if (!fresh) {
          const int grow = w ? e[1] - e_old[1] : e[0] - e_old[0];
          if (is_new[0] == 0 && is_new[2] == 0 && grow == 0) continue;
          old = *dst;
          if (grow != 0) {
            const float shrink = exp2_int(-grow);
            uint32_t o[4] = {old.x, old.y, old.z, old.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float4 f = e4m3_unpack4(o[k]);
              o[k] = e4m3_pack4(f.x * shrink, f.y * shrink, f.z * shrink, f.w * shrink);
            }
            old = make_uint4(o[0], o[1], o[2], o[3]);
          }
        }
        v[0] = (v[0] & is_new[0]) | (old.x & ~is_new[0]);
        v[1] = (v[1] & is_new[1]) | (old.y & ~is_new[1]);
        v[2] = (v[2] & is_new[2]) | (old.z & ~is_new[2]);
        v[3] = (v[3] & is_new[3]) | (old.w & ~is_new[3]);
      }
      *dst = make_uint4(v[0], v[1], v[2], v[3]);
    }
  }
}

// The owners' search needs a row_start that rises, up to `tokens`: the grid's last CTA looks at all of it.
// (In every CTA that took 5 % of long prompts' time and 0.5 us of a small call's 6.3.)
__device__ __noinline__ void report_falls(const uint32_t *row_start, uint32_t seqs, uint32_t tokens, uint32_t *err) {
  for (uint32_t i = threadIdx.x; i < seqs; i += kAppThreads) {
    const uint32_t r0 = row_start[i], r1 = row_start[i + 1];
    if (r0 > r1 || r1 > tokens) raise_error(err, kDevBadParams);
  }
}

template <typename T, int D, TurnMode MODE>
__global__ void __launch_bounds__(kAppThreads, D * sizeof(T) <= 512 ? 4 : D <= 256 ? 3 : 2)
    kv8_append_kernel(AppendArgs a) {
  extern __shared__ __align__(16) uint8_t sh[];
  __shared__ float amax[2][2][kKv8Block];  // [parity][K, V][token]
  pdl_launch_dependents();
  pdl_wait();

  const uint32_t u = blockIdx.x;
  if (u == gridDim.x - 1) {
    report_falls(a.row_start, a.c.num_seqs, a.tokens, a.err);
    return;
  }
  const uint32_t b = warp_last_le(a.c.num_seqs, u, [&](uint32_t i) { return kv8_unit_base(a.row_start[i], i); });
  Kv8Rows r;
  if (!kv8_rows(a.c, a.row_start, a.kv_len, a.tokens, b, &r)) {
    if (threadIdx.x == 0) raise_error(a.err, kDevBadParams);
    return;
  }
  Unit unit;
  if (!kv8_unit(r, u - kv8_unit_base(r.r0, b), &unit)) return;
  unit.page = a.c.table[(size_t)b * a.c.max_pages + unit.block * kKv8Block / a.c.page_tokens];
  unit.in_page = unit.block % (a.c.page_tokens / kKv8Block);
  if (unit.page >= a.c.num_pages) {
    if (threadIdx.x == 0) raise_error(a.err, kDevBadSlot);
    return;
  }

  float *const q_w = reinterpret_cast<float *>(sh + append_tile_bytes(D, MODE == kTurnMemory)), *const k_w = q_w + D;
  float *const angles = k_w + D;
  const uint32_t half = a.rot / 2, pos = unit.block * kKv8Block + unit.t0;
  for (uint32_t i = threadIdx.x; i < unit.cnt * half; i += blockDim.x) {
    const uint32_t t = i / half, f = i - t * half;
    float s, c;
    sincosf(__fmul_rn((float)(pos + t), a.inv_freq[f]), &s, &c);
    angles[t * a.rot + f] = c;
    angles[t * a.rot + half + f] = s;
  }
  for (uint32_t i = threadIdx.x; i < D; i += blockDim.x) {
    if (a.q_w) q_w[i] = a.q_w[i];
    if (a.k_w) k_w[i] = a.k_w[i];
  }
  __syncthreads();
  const uint32_t h0 = blockIdx.y * a.heads_per_cta;
  const uint32_t h1 = min(a.c.num_kv, h0 + a.heads_per_cta);
  if (unit.cnt == kKv8Block)
    append_heads<T, D, MODE, true>(a, unit, h0, h1, sh, amax);
  else
    append_heads<T, D, MODE, false>(a, unit, h0, h1, sh, amax);
}

size_t append_smem(uint32_t d, uint32_t rot) {
  return append_tile_bytes(d, turn_mode(rot / 2) == kTurnMemory) + 2 * d * sizeof(float) +
         (size_t)kKv8Block * rot * sizeof(float);
}

using AppendKernel = void (*)(AppendArgs);
template <typename T, int D>
AppendKernel append_kernel(uint32_t half) {
  switch (turn_mode(half)) {
    case kTurnShuffle: return kv8_append_kernel<T, D, kTurnShuffle>;
    case kTurnChunks: return kv8_append_kernel<T, D, kTurnChunks>;
    default: return kv8_append_kernel<T, D, kTurnMemory>;
  }
}
template <typename T>
AppendKernel append_kernel(uint32_t d, uint32_t half) {
  return d == 64 ? append_kernel<T, 64>(half) : d == 128 ? append_kernel<T, 128>(half)
       : d == 256 ? append_kernel<T, 256>(half) : append_kernel<T, 512>(half);
}
AppendKernel append_kernel(sx_dtype t, uint32_t d, uint32_t half) {
  return t == SX_F32 ? append_kernel<float>(d, half) : append_kernel<__nv_bfloat16>(d, half);
}

}  // namespace

cudaError_t prepare_kv8_append() {
  for (uint32_t d : {64u, 128u, 256u, 512u})
    for (sx_dtype t : {SX_F32, SX_BF16})
      for (uint32_t half : {0u, 64u, 1u}) {  // one of each rotation
        const cudaError_t e = cudaFuncSetAttribute(append_kernel(t, d, half),
                                                   cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   (int)(append_tile_bytes(d, true) + append_smem(d, d)));
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
  // All kv heads of a unit in one CTA compute its angles once; with few units the heads are spread
  // until every SM has work.
  const uint32_t units = sx::kv8_unit_count(tokens, c->num_seqs);
  a.heads_per_cta = c->num_kv;
  while (a.heads_per_cta > 1 && (uint64_t)units * ((c->num_kv + a.heads_per_cta - 1) / a.heads_per_cta) <
                                    12ull * e->num_sms)
    a.heads_per_cta = (a.heads_per_cta + 1) / 2;
  const dim3 grid(units + 1, (c->num_kv + a.heads_per_cta - 1) / a.heads_per_cta);
  return sx_host_cuda_status(
      sx::launch_chained(sx::append_kernel(t, c->head_dim, rotary_dim / 2), grid, dim3(sx::kAppThreads),
                         sx::append_smem(c->head_dim, rotary_dim), e->stream, 1, a),
      "kv8_append launch");
}

extern "C" SX_API uint32_t sx_kv8_append_args_bytes(void) { return (uint32_t)sizeof(sx_kv8_append_args); }
extern "C" SX_API sx_status sx_dispatch_kv8_append_args(sx_engine *e, const sx_kv8_append_args *a) {
  if (!a) {
    sx_host_set_error("kv8_append: null arguments");
    return SX_ERR_INVALID;
  }
  return sx_dispatch_kv8_append(e, &a->cache, (sx_dtype)a->dtype, a->q_in, a->k_in, a->v_in, a->q_ld, a->k_ld, a->v_ld,
                                a->q_norm_w, a->k_norm_w, a->q_out, a->row_start, a->kv_len, a->tokens, a->num_q,
                                a->inv_freq, a->rotary_dim, a->flags, a->eps);
}
