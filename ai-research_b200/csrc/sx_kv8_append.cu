// sx_kv8_append.cu -- new rows into the paged 8-bit KV cache: q / k RMS norm, position rotation,
// e4m3 quantisation with one power-of-two scale per 16 tokens and kv head (include/sx.h,
// sx_dispatch_kv8_append).
//
//   q', k' = R(pos) (x / rms(x) * gain),  v' = v / rms(v),  stored = rn_e4m3(x' 2^-e),
//   e = min { e : max |record| <= 448 2^e }
//
// A record belongs to one CTA, which sees all of its new tokens, so the scale needs no atomics:
// unit u is one 16-token block of one sequence, a CTA takes one unit and a group of kv heads with
// their q heads.  With sequence b's rows at row_start[b], units row_start[b] / 16 + 2 b .. belong to
// it: n rows touch at most n / 16 + 2 blocks, so the grid follows from the row and sequence counts
// alone and nothing is read back.
//
// Bound by the rows' bytes, and close behind by instructions: a vector of 256 has 45 cycles of an SM
// at the copy rate.  A warp takes whole vectors; lane l holds elements 128 k + 4 l .. + 3 of every
// chunk k (64 k + 2 l for heads of 64), so that a rotation whose half is a multiple of the chunk
// needs no exchange and a shorter one meets its pairs by shuffles within chunk 0.  The angles are
// computed once per unit.  K and V stay in registers until the block's maxima have met in shared
// memory, are converted by their owners, and leave through a byte tile that turns rows of tokens
// into the record's pieces.
#include "sx_host.h"
#include "sx_kv8.cuh"
#include "sx_launch.cuh"

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

// shared memory: the byte tile (or a row of f32 per warp, for rotations whose pairs meet there),
// the gains of q and k, the angles' cosines and sines
SX_HD constexpr uint32_t append_tile_bytes(uint32_t d) {
  return 2 * kKv8Block * (d + 32) > kAppWarps * d * 4 ? 2 * kKv8Block * (d + 32) : kAppWarps * d * 4;
}

// Head size D: chunks of 32 lanes x V elements.
template <int D>
struct Lane {
  static constexpr int kVec = D >= 128 ? 4 : 2;
  static constexpr int kChunk = 32 * kVec;
  static constexpr int kChunks = D / kChunk;
};
template <int D>
using Elems = float[Lane<D>::kChunks][Lane<D>::kVec];

// A lane's part of a vector as it stands in memory.
template <typename T, int D>
struct Raw {
  static constexpr int kWords = Lane<D>::kVec * (int)sizeof(T) / 4;
  uint32_t w[Lane<D>::kChunks][kWords];
  SX_DEV void load(const T *p, uint32_t lane) {
#pragma unroll
    for (int k = 0; k < Lane<D>::kChunks; ++k) {
      const T *src = p + Lane<D>::kChunk * k + Lane<D>::kVec * lane;
      if constexpr (kWords == 4) {
        const uint4 u = *reinterpret_cast<const uint4 *>(src);
        w[k][0] = u.x; w[k][1] = u.y; w[k][2] = u.z; w[k][3] = u.w;
      } else if constexpr (kWords == 2) {
        const uint2 u = *reinterpret_cast<const uint2 *>(src);
        w[k][0] = u.x; w[k][1] = u.y;
      } else {
        w[k][0] = *reinterpret_cast<const uint32_t *>(src);
      }
    }
  }
  SX_DEV void unpack(Elems<D> &x) const {
#pragma unroll
    for (int k = 0; k < Lane<D>::kChunks; ++k)
#pragma unroll
      for (int j = 0; j < Lane<D>::kVec; ++j) {
        if constexpr (sizeof(T) == 4)
          x[k][j] = __uint_as_float(w[k][j]);
        else
          x[k][j] = __uint_as_float(j & 1 ? w[k][j / 2] & 0xFFFF0000u : w[k][j / 2] << 16);
      }
  }
};
template <typename T, int D>
SX_DEV void store_vector(T *p, uint32_t lane, const Elems<D> &x) {
#pragma unroll
  for (int k = 0; k < Lane<D>::kChunks; ++k)
    store_vec<T, Lane<D>::kVec>(p + Lane<D>::kChunk * k + Lane<D>::kVec * lane, x[k]);
}

// x / rms(x)
template <int D>
SX_DEV void normalise(Elems<D> &x, float eps) {
  float ss = 0.0f;
#pragma unroll
  for (int k = 0; k < Lane<D>::kChunks; ++k)
#pragma unroll
    for (int j = 0; j < Lane<D>::kVec; ++j) ss = fmaf(x[k][j], x[k][j], ss);
  const float rs = rsqrtf(warp_sum(ss) * (1.0f / D) + eps);
#pragma unroll
  for (int k = 0; k < Lane<D>::kChunks; ++k)
#pragma unroll
    for (int j = 0; j < Lane<D>::kVec; ++j) x[k][j] = __fmul_rn(x[k][j], rs);
}
template <int D>
SX_DEV void gain(Elems<D> &x, const float *w, uint32_t lane) {
#pragma unroll
  for (int k = 0; k < Lane<D>::kChunks; ++k) {
    float g[Lane<D>::kVec];
    load_vec<float, Lane<D>::kVec>(w + Lane<D>::kChunk * k + Lane<D>::kVec * lane, g);
#pragma unroll
    for (int j = 0; j < Lane<D>::kVec; ++j) x[k][j] = __fmul_rn(x[k][j], g[j]);
  }
}

// The rotation of one lane's elements.  Angles of a token: [cosines of the pairs | their sines].
template <int D>
struct Turn {
  static constexpr int kVec = Lane<D>::kVec, kChunk = Lane<D>::kChunk, kChunks = Lane<D>::kChunks;
  uint32_t half, mode;     // 0 none, 1 shuffles in chunk 0, 2 chunks of a lane, 3 by memory
  uint32_t peer, at;       // mode 1: the lane of the partners, this lane's first pair
  bool low, in;            //         first of the pairs; rotated at all
  SX_DEV Turn(uint32_t half_, uint32_t lane) : half(half_), peer(lane), at(0), low(false), in(false) {
    mode = half == 0 ? 0 : half % kChunk == 0 ? 2 : 2 * half <= (uint32_t)kChunk && half % kVec == 0 ? 1 : 3;
    if (mode == 1) {
      const uint32_t o = half / kVec;
      low = lane < o;
      in = lane < 2 * o;
      peer = low ? lane + o : in ? lane - o : lane;
      at = in ? kVec * (low ? lane : lane - o) : 0;
    }
  }
  // every product and sum rounded by itself, as the engine's own rotation
  template <int H>
  SX_DEV void chunks(Elems<D> &x, const float *cs, uint32_t lane) const {
    if constexpr (2 * H <= kChunks) {
#pragma unroll
      for (int k = 0; k < H; ++k) {
        float c[kVec], s[kVec];
        load_vec<float, kVec>(cs + kChunk * k + kVec * lane, c);
        load_vec<float, kVec>(cs + half + kChunk * k + kVec * lane, s);
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
          const float x0 = x[k][j], x1 = x[k + H][j];
          x[k][j] = __fsub_rn(__fmul_rn(x0, c[j]), __fmul_rn(x1, s[j]));
          x[k + H][j] = __fadd_rn(__fmul_rn(x0, s[j]), __fmul_rn(x1, c[j]));
        }
      }
    }
  }
  SX_DEV void operator()(Elems<D> &x, const float *cs, float *buf, uint32_t lane) const {
    if (mode == 0) return;
    if (mode == 1) {
      float c[kVec], s[kVec];
      load_vec<float, kVec>(cs + at, c);
      load_vec<float, kVec>(cs + half + at, s);
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        const float y = __fmul_rn(__shfl_sync(0xffffffffu, x[0][j], peer), s[j]);
        const float r = __fadd_rn(__fmul_rn(x[0][j], c[j]), low ? -y : y);
        if (in) x[0][j] = r;
      }
    } else if (mode == 2) {
      if (half == kChunk)
        chunks<1>(x, cs, lane);
      else if (half == 2 * kChunk)
        chunks<2>(x, cs, lane);
    } else {
      __syncwarp();
#pragma unroll
      for (int k = 0; k < kChunks; ++k)
#pragma unroll
        for (int j = 0; j < kVec; ++j) buf[kChunk * k + kVec * lane + j] = x[k][j];
      __syncwarp();
#pragma unroll
      for (int k = 0; k < kChunks; ++k)
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
          const uint32_t d = kChunk * k + kVec * lane + j;
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

// One 16-token block of one sequence.
struct Unit {
  uint32_t row0, cnt, t0;  // its new rows, how many, the first one's place in the block
  uint32_t page, in_page;  // page and block of the page
};

// The kv heads [h0, h1) of a unit with their q heads.  FULL: all 16 tokens are new.
template <typename T, int D, bool FULL>
SX_DEV void append_heads(const AppendArgs &a, const Unit &u, uint32_t h0, uint32_t h1, uint8_t *sh,
                         float (*amax)[2][kKv8Block]) {
  constexpr int kChunks = Lane<D>::kChunks, kVec = Lane<D>::kVec, kChunk = Lane<D>::kChunk;
  constexpr int kLd = D + 32;  // bytes of a tile row
  uint8_t *const tile = sh;    // [K, V][16][kLd]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float *const buf = reinterpret_cast<float *>(sh) + warp * D;
  const float *const q_w = reinterpret_cast<const float *>(sh + append_tile_bytes(D)), *const k_w = q_w + D;
  const float *const angles = k_w + D;  // [16][2 half]
  const uint32_t cnt = FULL ? kKv8Block : u.cnt, t0 = FULL ? 0 : u.t0;
  const bool fresh = t0 == 0;
  const Turn<D> turn(a.rot / 2, lane);

  // Tokens over warps: warp w takes tokens w % tw and w % tw + 8, and with few tokens the vectors
  // of one (K, V, then q heads) are dealt to the warps that share it (tw and subs: powers of two).
  uint32_t tw = 8;
  if (!FULL)
    while (tw > 1 && tw / 2 >= cnt) tw /= 2;
  const uint32_t tok = warp & (tw - 1), sub = FULL ? 0 : warp / tw, subs = FULL ? 1 : kAppWarps / tw;
  auto skip = [&](int i, int w) { return !FULL && (tok + 8 * i >= cnt || (w & (subs - 1)) != sub); };
  const T *rows[2][2], *q_src[2];
  T *q_dst[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const size_t row = u.row0 + tok + 8 * i;
    rows[i][0] = static_cast<const T *>(a.k) + row * a.k_ld;
    rows[i][1] = a.k_eq_v ? rows[i][0] : static_cast<const T *>(a.v) + row * a.v_ld;
    q_src[i] = static_cast<const T *>(a.q) + row * a.q_ld;
    q_dst[i] = static_cast<T *>(a.q_out) + row * ((size_t)a.c.num_kv * a.gqa * D);
  }
  for (uint32_t h = h0; h < h1; ++h) {
    const uint32_t par = (h - h0) & 1;
    float x[2][2][kChunks][kVec];  // [token][K, V]
    {
      Raw<T, D> raw[2][2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int w = 0; w < 2; ++w)
          if (!skip(i, w)) raw[i][w].load(rows[i][w] + (size_t)h * D, lane);
      if (turn.mode == 3) __syncthreads();  // the rows of buf lie over the tile
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          if (skip(i, w)) continue;
          const uint32_t t = tok + 8 * i;
          raw[i][w].unpack(x[i][w]);
          if (w == 1) {
            if (a.v_norm) normalise<D>(x[i][w], a.eps);
          } else {
            if (a.k_w) {
              normalise<D>(x[i][w], a.eps);
              gain<D>(x[i][w], k_w, lane);
            }
            turn(x[i][w], angles + t * a.rot, buf, lane);
          }
          float m = 0.0f;
#pragma unroll
          for (int k = 0; k < kChunks; ++k)
#pragma unroll
            for (int j = 0; j < kVec; ++j) m = fmaxf(m, fabsf(x[i][w][k][j]));  // a NaN does not count
          m = warp_max(m);
          if (lane == 0) amax[par][w][t] = m;
        }
    }
    // ---- q heads of kv head h, the next one's load in flight
    {
      // vector 2 + g of a token belongs to warp (2 + g) % subs
      const uint32_t g0 = (sub - 2) & (subs - 1);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t t = tok + 8 * i;
        if (!FULL && t >= cnt) continue;
        const T *src = q_src[i] + (size_t)h * a.gqa * D;
        T *dst = q_dst[i] + (size_t)h * a.gqa * D;
        Raw<T, D> next;
        if (g0 < a.gqa) next.load(src + g0 * D, lane);
        for (uint32_t g = g0; g < a.gqa; g += subs) {
          Elems<D> y;
          next.unpack(y);
          if (g + subs < a.gqa) next.load(src + (g + subs) * D, lane);
          if (a.q_w) {
            normalise<D>(y, a.eps);
            gain<D>(y, q_w, lane);
          }
          turn(y, angles + t * a.rot, buf, lane);
          store_vector<T, D>(dst + g * D, lane, y);
        }
      }
    }
    __syncthreads();
    // ---- the block's scales, and the owners' conversion
    const size_t rec = (((size_t)u.page * a.c.num_kv + h) * (a.c.page_tokens / kKv8Block) + u.in_page) * 2;
    int e_old[2], e[2];
    {
      const uint32_t t = lane & 15;
      float m = FULL || t < cnt ? amax[par][lane >> 4][t] : 0.0f;
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
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
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        if (skip(i, w)) continue;
        const float inv = exp2_int(-e[w]);
        uint8_t *row = tile + (w * kKv8Block + t0 + tok + 8 * i) * kLd + kVec * lane;
#pragma unroll
        for (int k = 0; k < kChunks; ++k) {
          if constexpr (kVec == 4)
            *reinterpret_cast<uint32_t *>(row + kChunk * k) =
                e4m3_pack4(x[i][w][k][0] * inv, x[i][w][k][1] * inv, x[i][w][k][2] * inv, x[i][w][k][3] * inv);
          else
            *reinterpret_cast<uint16_t *>(row + kChunk * k) = (uint16_t)__nv_cvt_float2_to_fp8x2(
                make_float2(x[i][w][k][0] * inv, x[i][w][k][1] * inv), __NV_SATFINITE, __NV_E4M3);
        }
      }
    __syncthreads();
    if (threadIdx.x < 2) a.c.scale[rec + threadIdx.x] = exp2_int(threadIdx.x ? e[1] : e[0]);
    // ---- 16-byte pieces of the K record, then of the V record
    uint8_t *const out = static_cast<uint8_t *>(a.c.data) + rec * (size_t)(kKv8Block * D);
    for (uint32_t i = threadIdx.x; i < 2 * D; i += kAppWarps * 32) {
      const uint32_t w = i / D, p = i % D >> 5, g = (i & 31) >> 2, c = i & 3;
      const uint8_t *src = tile + w * kKv8Block * kLd + 32 * p;
      uint32_t v[4], is_new[4];  // the piece and which of its bytes are new
      if (w == 0) {
        const uint2 lo8 = *reinterpret_cast<const uint2 *>(src + g * kLd + 8 * c);
        const uint2 hi8 = *reinterpret_cast<const uint2 *>(src + (g + 8) * kLd + 8 * c);
        v[0] = lo8.x; v[1] = lo8.y; v[2] = hi8.x; v[3] = hi8.y;
        is_new[0] = is_new[1] = g >= t0 && g < t0 + cnt ? 0xFFFFFFFFu : 0u;
        is_new[2] = is_new[3] = g + 8 >= t0 && g + 8 < t0 + cnt ? 0xFFFFFFFFu : 0u;
      } else {
        uint32_t m = 0;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const uint32_t t = 2 * c + (s & 1) + 8 * (s >> 1);
          v[s] = *reinterpret_cast<const uint32_t *>(src + t * kLd + 4 * g);
          if (t >= t0 && t < t0 + cnt) m |= 0xFFu << (8 * s);
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

template <typename T, int D>
__global__ void __launch_bounds__(kAppWarps * 32, D <= 256 ? 3 : 2) kv8_append_kernel(AppendArgs a) {
  extern __shared__ __align__(16) uint8_t sh[];
  __shared__ float amax[2][2][kKv8Block];  // [parity][K, V][token]
  pdl_launch_dependents();
  pdl_wait();

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
  Unit unit;
  unit.row0 = r.r0 + (lo - pos0);
  unit.cnt = hi - lo;
  unit.t0 = lo % kKv8Block;
  unit.page = a.c.table[(size_t)b * a.c.max_pages + blk * kKv8Block / a.c.page_tokens];
  unit.in_page = blk % (a.c.page_tokens / kKv8Block);
  if (unit.page >= a.c.num_pages) {
    if (threadIdx.x == 0) raise_error(a.err, kDevBadSlot);
    return;
  }

  float *const q_w = reinterpret_cast<float *>(sh + append_tile_bytes(D)), *const k_w = q_w + D;
  float *const angles = k_w + D;
  const uint32_t half = a.rot / 2;
  for (uint32_t i = threadIdx.x; i < unit.cnt * half; i += blockDim.x) {
    const uint32_t t = i / half, f = i - t * half;
    float s, c;
    sincosf(__fmul_rn((float)(lo + t), a.inv_freq[f]), &s, &c);
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
    append_heads<T, D, true>(a, unit, h0, h1, sh, amax);
  else
    append_heads<T, D, false>(a, unit, h0, h1, sh, amax);
}

size_t append_smem(uint32_t d, uint32_t rot) {
  return append_tile_bytes(d) + 2 * d * sizeof(float) + (size_t)kKv8Block * rot * sizeof(float);
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
  // All kv heads of a unit in one CTA compute its angles once; with few units the heads are spread
  // until every SM has work.
  const uint32_t units = tokens / sx::kKv8Block + 2 * c->num_seqs;
  a.heads_per_cta = c->num_kv;
  while (a.heads_per_cta > 1 && (uint64_t)units * ((c->num_kv + a.heads_per_cta - 1) / a.heads_per_cta) <
                                    12ull * e->num_sms)
    a.heads_per_cta = (a.heads_per_cta + 1) / 2;
  const dim3 grid(units, (c->num_kv + a.heads_per_cta - 1) / a.heads_per_cta);
  return sx_host_cuda_status(
      sx::launch_chained(sx::append_kernel(t, c->head_dim), grid, dim3(sx::kAppWarps * 32),
                         sx::append_smem(c->head_dim, rotary_dim), e->stream, 1, a),
      "kv8_append launch");
}
