// sx_kv8_attn.cu -- attention over the paged 8-bit KV cache (include/sx.h, sx_dispatch_kv8_attn).
//
//   out_r = sum_j p_j V_j,  p = softmax_j(scale q_r . K_j),  j <= pos(r), j > pos(r) - window
//
// The rows that share a kv head (n new tokens x G q heads) are packed, and the two products run
// transposed on mma.m16n8k16: S^T = K Q^T with 16 tokens as the rows of A, O^T = V^T P^T with 16
// elements of the head as the rows of A.  The cache's records are those A operands byte for byte
// (sx_kv8.cuh), so a block of 16 tokens goes shared memory -> registers -> f16 -> MMA, and eight
// packed rows fill the instruction's N without waste.  P^T leaves the first product with tokens
// along the lanes' rows and enters the second with tokens along K: movmatrix transposes it.
//
// Values: e4m3 is exact in f16.  q is scaled by a power of two per row to at most 2 and split into
// two f16 terms (22 bits) for f32 rows; bf16 rows need one.  The reference m is the running maximum of
// x + log2(v scale), x the score in log2 units, rounded up to a whole number: p' = 2^(x + log2(v scale) -
// m + 15) is at most 2^15 and carries the V record's scale, and what changes m is an exact power of two.
// The softmax's sum takes p' / v scale in f32.  f16 holds 22 bits of a p' down to 2^-3 (two terms; 11 bits
// down to 2^-14 with one) and multiples of 2^-24 below.
//
// A record's scale may be far above the values that a row sees in it: its largest value may be masked, or
// have no weight.  m would then leave nothing of the p' of other records.  Where scales fall by more than
// 2^kFar the output is scaled up and m lowered to the record's own, as far as f32 holds the output.
//
// Split: the batch's work is a line of 16-token blocks -- for each sequence, kv head and group of
// packed rows the blocks it sees and kOverhead more, for what starting and ending it costs -- cut
// into equal runs, one per CTA, computed on the device from the lengths, so a ragged batch and one
// long sequence balance alike.  The warps of a CTA take blocks in turn, each with its own ring of
// bulk copies (a K or a V record a stage) and its own maximum, sum and output; they merge in shared
// memory at the end of a problem, and CTAs that share a problem through the workspace: the last to
// arrive merges (its order is that of the CTAs, so results repeat).  Runs are of 8 blocks at least, one
// per warp (640 keys of one head of 256: 11.9 us; with 16 or 32, or uncut, 2 more).  Problems of up to three
// such steps more than a run are not cut, since a merge costs as much (16 rows in a window of 512:
// 20.4 us; cut 5 more).
//
// Measured: 64 rows on up to 8192 keys (16 q and 8 kv heads of 256, bf16) 179 us, 6.1 TB/s or 94 % of the
// measured copy rate, the rest being starts and ends of 512 problems, where a CTA's copies run dry; 131k
// keys of 8 heads of 128 for one f32 row 56.4 us (74 %); batches of heads of 512 101 %, of 128 92 %, of 64
// 56 % (a block of 16 tokens costs as many instructions of softmax for a quarter of the bytes); of f32 rows
// 99, 77 and 51 %; of 16 f32 rows per kv head 41 % (128, where 16 rows' output and scores spill) and 48 % (256).  A window
// of 512 leaves 128 of 296 CTAs work, and a warp's ring two records: each of the five steps waits for its
// own (20.4 us, floor 5.3).  Two or four blocks a warp at a time were slower below 256: 15.9 us for 5.5 on
// 127 keys with 64, 5 % in full batches of 128.  So were three or four CTAs an SM (6 and 26 % in full
// batches of 64).
#include "sx_host.h"
#include "sx_kv8.cuh"
#include "sx_launch.cuh"

namespace sx {
namespace {

constexpr int kDecWarps = 8;
constexpr int kDecThreads = kDecWarps * 32;
// Blocks that starting and ending a problem is worth.  With 8, 16, 24, 32 and 48: full batches of head size
// 256 186, 180, 181, 180 and 183 us, of 128 106, 99, 91, 90 and 91, drafts of two heads of 256 115, 108, 93,
// 90 and 93.
constexpr uint32_t kOverhead = 32;
constexpr uint32_t kMergeSteps = 3;  // steps (a block a warp) that a merge over CTAs is worth
constexpr float kPOffset = 15.0f;
constexpr float kFar = 16.0f;     // p' of a scale this far below is 2^-1 at its largest: 22 bits of multiples of 2^-24
constexpr int kLargest = 100;     // exponent up to which an output is scaled up
constexpr uint32_t kMaxParts = 32, kPartGroup = 16;  // merged at once; of a first level

SX_DEV uint32_t movmatrix_trans(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(v));
  return r;
}
// a[0 .. 1] += b[0 .. 1] in one instruction
SX_DEV void add_f32x2(float *a, const float *b) {
  asm("{\n .reg .b64 x, y;\n mov.b64 x, {%0, %1};\n mov.b64 y, {%2, %3};\n add.rn.f32x2 x, x, y;\n"
      " mov.b64 {%0, %1}, x;\n}\n"
      : "+f"(a[0]), "+f"(a[1])
      : "f"(b[0]), "f"(b[1]));
}
// The blocks of 16 tokens that rows of a sequence see.
SX_DEV void seen_blocks(const Kv8Rows &r, uint32_t window, uint32_t *first, uint32_t *count) {
  const uint32_t pos0 = r.len - r.n;  // of the first row
  *first = (window && pos0 + 1 > window ? pos0 + 1 - window : 0) / kKv8Block;
  *count = r.n ? (r.len - 1) / kKv8Block - *first + 1 : 0;
}

// Shapes of the kernel for head size D and 8 NT packed rows.  The output takes D NT / 4 registers
// per thread: up to 64 two CTAs fit an SM and hide each other's starts and ends, with 128 one.
template <int D, int NT, bool SPLIT>
struct DecShape {
  static constexpr int kRows = 8 * NT;
  static constexpr int kPieces = D / 32;
  static constexpr int kCtas = D * NT <= 256 ? 2 : 1;         // per SM
  static constexpr int kRecord = 16 * D;
  // Of one warp: an SM has 128 KB on their way, three times what the copy rate needs.  Half as much again
  // only queues, and every other load behind it: 12 and 24 KB took 200 us for 187 in full batches of 256,
  // 177 for 168 with 512.
  static constexpr int kRing = (kCtas == 2 ? 8 : 16) * 1024;
  static constexpr int kStages = kRing / kRecord;
  static constexpr int kLdO = D + 4;
  static constexpr int kMerge = kDecWarps * kRows * kLdO * 4; // shares the rings' memory
  static constexpr int kArea = kDecWarps * kRing > kMerge ? kDecWarps * kRing : kMerge;
  static constexpr int kQ = NT * kPieces * 512 * (SPLIT ? 2 : 1);
  static constexpr int kSmem = kArea + kQ;
};

// What the CTA's threads share beside the rings.
template <int ROWS>
struct DecShared {
  uint32_t last_flag;
  float row_mul[ROWS], row_inv[ROWS];
  float wm[kDecWarps][ROWS], wl[kDecWarps][ROWS];  // maxima and sums of the warps
  float fac[kMaxParts][ROWS];                      // what a warp's, or a part's, output counts
};

// A problem that several CTAs hold parts of.
struct Parts {
  uint32_t c0, parts, slot0;  // its first CTA, how many, where the first part is
  uint32_t r0, row0, rows, head;
  SX_DEV uint32_t slot(uint32_t k) const { return k == 0 ? slot0 : 2 * (c0 + k); }
};

// Merges a problem's parts, by the last CTA to arrive: up to kMaxParts at once, more by groups first,
// each into its first part's place.  They count at words of CTAs inside the problem, which no other
// problem starts in.  Out of line: it would cost the loop registers.
template <typename T, int D, int ROWS>
__device__ __noinline__ void merge_parts(const Kv8AttnArgs &a, const Parts w, DecShared<ROWS> &sh) {
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float2 *const part_ml = reinterpret_cast<float2 *>(a.part);
  float *const part_o = a.part + (size_t)2 * gridDim.x * ROWS * 2;
  bool last = w.parts <= kMaxParts;  // the level is the last one
  uint32_t from = last ? 0 : (blockIdx.x - w.c0) / kPartGroup * kPartGroup, each = 1;
  uint32_t n = last ? w.parts : min(kPartGroup, w.parts - from);
  uint32_t *word = a.cnt + w.c0 + (from ? from - 1 : 0);
#pragma unroll 1
  for (;;) {
    __syncthreads();
    if (threadIdx.x == 0) sh.last_flag = arrive_acq_rel(word) == n - 1;
    __syncthreads();
    if (!sh.last_flag) return;
    if (threadIdx.x == 0) *word = 0;
    // a warp per row for the maxima, a lane per part; then all threads over the rows' elements
    for (uint32_t i = warp; i < w.rows; i += kDecWarps) {
      float2 ml = make_float2(-INFINITY, 0.0f);
      if (lane < n) ml = __ldcg(part_ml + (size_t)w.slot(from + lane * each) * ROWS + i);
      const float m = warp_max(ml.x), f = ml.x == -INFINITY ? 0.0f : ex2(ml.x - m), l = warp_sum(ml.y * f);
      sh.fac[lane][i] = f;
      if (lane == 0) {
        sh.wm[0][i] = m;
        sh.wl[0][i] = l;
      }
    }
    __syncthreads();
    for (uint32_t x = threadIdx.x; x < w.rows * (D / 4); x += kDecThreads) {
      const uint32_t i = x / (D / 4), d = x % (D / 4) * 4;
      float4 sum = make_float4(0, 0, 0, 0);
#pragma unroll 8
      for (uint32_t k = 0; k < n; ++k) {
        const float4 v =
            __ldcg(reinterpret_cast<const float4 *>(part_o + ((size_t)w.slot(from + k * each) * ROWS + i) * D + d));
        const float f = sh.fac[k][i];
        sum.x = fmaf(v.x, f, sum.x);
        sum.y = fmaf(v.y, f, sum.y);
        sum.z = fmaf(v.z, f, sum.z);
        sum.w = fmaf(v.w, f, sum.w);
      }
      if (last) {
        const float l = sh.wl[0][i], inv = l == 0.0f ? 0.0f : 1.0f / l;
        const float y[4] = {sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv};
        const uint32_t pr = w.row0 + i;
        store_vec<T, 4>(static_cast<T *>(a.out) + (size_t)(w.r0 + pr / a.gqa) * a.out_ld +
                            (size_t)(w.head * a.gqa + pr % a.gqa) * D + d, y);
      } else {
        *reinterpret_cast<float4 *>(part_o + ((size_t)w.slot(from) * ROWS + i) * D + d) = sum;
      }
    }
    if (last) return;
    if (threadIdx.x < w.rows)
      part_ml[(size_t)w.slot(from) * ROWS + threadIdx.x] = make_float2(sh.wm[0][threadIdx.x], sh.wl[0][threadIdx.x]);
    last = true;
    from = 0;
    each = kPartGroup;
    n = (w.parts + kPartGroup - 1) / kPartGroup;
    word = a.cnt + w.c0 + 1;
  }
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(kDecThreads, (DecShape<D, NT, sizeof(T) == 4>::kCtas))
    kv8_decode_kernel(const __grid_constant__ Kv8AttnArgs a) {
  constexpr bool kSplit = sizeof(T) == 4;
  using S = DecShape<D, NT, kSplit>;
  constexpr int kStages = S::kStages, kPieces = S::kPieces, kRows = S::kRows;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t full_bar[kDecWarps * kStages];
  __shared__ DecShared<kRows> sh;
  float (&row_mul)[kRows] = sh.row_mul, (&row_inv)[kRows] = sh.row_inv;
  float (&wm)[kDecWarps][kRows] = sh.wm, (&wl)[kDecWarps][kRows] = sh.wl, (&fac)[kMaxParts][kRows] = sh.fac;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  uint8_t *const qf = smem + S::kArea;
  uint8_t *const ring = smem + warp * S::kRing;
  const uint32_t ring_u = smem_u32(ring), bar_u = smem_u32(full_bar + warp * kStages);
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(bar_u + 8 * s, 1);
    fence_mbar_init();
  }

  __syncwarp();
  pdl_launch_dependents();
  pdl_wait();

  // ---- this CTA's run of the line of blocks; every warp finds it alike
  auto problems_of = [&](const Kv8Rows &r) {
    return (r.n * a.gqa + kRows - 1) / kRows * a.c.num_kv;
  };
  uint32_t longest = 0, problems = 0;  // of this lane's sequences
  auto cost = [&](uint32_t b) -> uint64_t {
    Kv8Rows r;
    if (!kv8_rows(a.c, a.row_start, a.kv_len, a.tokens, b, &r)) {
      if (blockIdx.x == 0 && warp == 0) raise_error(a.err, kDevBadParams);
      return 0;
    }
    uint32_t first, count;
    seen_blocks(r, a.window, &first, &count);
    longest = max(longest, count);
    problems += problems_of(r);
    return r.n ? (uint64_t)(count + kOverhead) * problems_of(r) : 0;
  };
  uint64_t begin, end, run, at;  // at: where the sequence of the next problem starts
  uint32_t b;
  bool uncut;  // problems are not cut: each goes to the CTA in whose run it starts
  {
    const uint32_t per = (a.c.num_seqs + 31) / 32;
    const uint32_t b0 = lane * per, b1 = min(a.c.num_seqs, b0 + per);
    uint64_t mine = 0;
    for (uint32_t i = b0; i < b1; ++i) mine += cost(i);
    uint64_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    const uint64_t total = __shfl_sync(0xffffffffu, incl, 31);
    run = (total + gridDim.x - 1) / gridDim.x;
    run = run > (uint32_t)kDecWarps ? run : (uint32_t)kDecWarps;
    longest = __reduce_max_sync(0xffffffffu, longest);
    problems = __reduce_add_sync(0xffffffffu, problems);
    uncut = longest <= kMergeSteps * kDecWarps + (problems <= gridDim.x ? run : 0);
    begin = run * blockIdx.x;
    end = begin + run < total ? begin + run : total;
    if (begin >= end) return;
    const uint32_t who = __popc(__ballot_sync(0xffffffffu, incl <= begin));  // its lane holds begin
    at = incl - mine;
    b = b0;
    if (lane == (int)who)
      for (uint64_t n; (n = cost(b)) <= begin - at; at += n) ++b;
    at = __shfl_sync(0xffffffffu, at, who);
    b = __shfl_sync(0xffffffffu, b, who);
  }

  uint32_t issued = 0, taken = 0;  // stages of this warp's ring, over all problems
  Kv8Rows r;
  uint32_t first = 0, count = 0, left = 0, problem = 0;  // problems of b that are left
  bool fresh = true;  // the first sequence: its first problems may lie before the run
  bool merged = false;
  for (; at < end; at += count + kOverhead, --left, ++problem) {
    while (left == 0 && b < a.c.num_seqs) {  // the next sequence with rows
      const bool ok = kv8_rows(a.c, a.row_start, a.kv_len, a.tokens, b, &r);
      ++b;
      if (!ok || r.n == 0) continue;
      seen_blocks(r, a.window, &first, &count);
      left = problems_of(r);
      problem = 0;
      if (fresh) {
        problem = (uint32_t)((begin - at) / (count + kOverhead));
        left -= problem;
        at += (uint64_t)problem * (count + kOverhead);
        fresh = false;
      }
    }
    if (left == 0) break;  // (the counts changed under the call)
    uint32_t s0 = begin > at ? (uint32_t)(begin - at) : 0;
    uint32_t s1 = end - at < count ? (uint32_t)(end - at) : count;
    if (uncut) {
      if (s0 != 0) continue;
      s1 = count;
    }
    if (s0 >= s1) continue;  // only its overhead lies in the run
    const uint32_t groups = (r.n * a.gqa + kRows - 1) / kRows;
    const uint32_t h = problem / groups, row0 = problem % groups * kRows;  // packed rows
    const uint32_t rows = min((uint32_t)kRows, r.n * a.gqa - row0);
    const uint32_t pos0 = r.len - r.n;
    const uint32_t tok_lo = row0 / a.gqa, tok_hi = (row0 + rows - 1) / a.gqa;

    // ---- copies: entry j is the warp's j-th block of the segment, 32 entries at a time in lanes
    const uint32_t *table = a.c.table + (size_t)(b - 1) * a.c.max_pages;
    const uint32_t steps = (s1 - s0 + kDecWarps - 1 - warp) / kDecWarps;  // of this warp
    const uint32_t busy = min((uint32_t)kDecWarps, s1 - s0);              // warps with any
    auto block_of = [&](uint32_t j) { return s0 + j * kDecWarps + warp; };
    struct Entry {
      uint64_t rec;  // record pair index; ~0: nothing to read
      float ks, vs;
    };
    auto entry = [&](uint32_t j) -> Entry {
      Entry e{~0ull, 0.0f, 1.0f};
      if (j >= steps) return e;
      const uint32_t s = block_of(j);
      const uint32_t blk = first + s;
      const uint32_t page = table[blk * kKv8Block / a.c.page_tokens];
      if (page >= a.c.num_pages) {
        raise_error(a.err, kDevBadSlot);
        return e;
      }
      const uint32_t per = a.c.page_tokens / kKv8Block;
      e.rec = ((uint64_t)page * a.c.num_kv + h) * per + blk % per;
      const float2 f = *reinterpret_cast<const float2 *>(a.c.scale + 2 * e.rec);
      e.ks = f.x;
      e.vs = f.y;
      return e;
    };
    // rows of q come first: their loads run beside the page table's
    float qx[(kRows + kDecWarps - 1) / kDecWarps][D / 32];
#pragma unroll
    for (int i = 0; i < kRows / kDecWarps; ++i) {
      const uint32_t pr = row0 + warp + i * kDecWarps;
      const bool in = warp + i * kDecWarps < rows;
      const T *src = static_cast<const T *>(a.q) + (size_t)(r.r0 + pr / a.gqa) * a.q_ld +
                     (size_t)(h * a.gqa + pr % a.gqa) * D;
#pragma unroll
      for (int k = 0; k < D / 64; ++k) {
        float v[2] = {0.0f, 0.0f};
        if (in) load_vec<T, 2>(src + 64 * k + 2 * lane, v);
        qx[i][2 * k] = v[0];
        qx[i][2 * k + 1] = v[1];
      }
    }
    Entry cur = entry(lane), nxt = entry(32 + lane);
    uint32_t batch = 0;     // cur holds entries [32 batch, + 32)
    uint32_t to_issue = 0;  // next record to issue: 2 step (K), 2 step + 1 (V)
    auto issue = [&]() {
      const uint32_t j = to_issue / 2, st = issued % kStages;
      const Entry &e = j / 32 == batch ? cur : nxt;
      if ((uint32_t)lane == j % 32) {
        const bool there = e.rec != ~0ull;
        mbar_arrive_expect_tx(bar_u + 8 * st, there ? S::kRecord : 0);
        if (there)
          bulk_g2s(ring_u + st * S::kRecord, static_cast<const uint8_t *>(a.c.data) + (2 * e.rec + (to_issue & 1)) * S::kRecord,
                   S::kRecord, bar_u + 8 * st);
      }
      ++issued;
      ++to_issue;
    };
    if (merged) {  // the merge of the problem before is done with the ring
      fence_proxy_async();
      __syncthreads();
    }
    while (to_issue < 2 * steps && to_issue < (uint32_t)kStages) issue();

    // ---- q: power-of-two scaled f16 terms as B operands
#pragma unroll
    for (int ii = 0; ii < kRows / kDecWarps; ++ii) {
      const uint32_t i = warp + ii * kDecWarps;
      const float (&x)[D / 32] = qx[ii];
      float m = 0.0f;
#pragma unroll
      for (int k = 0; k < D / 32; ++k) m = fmaxf(m, fabsf(x[k]));
      m = warp_max(m);
      int e = (int)(__float_as_uint(m) >> 23) - 127;
      if (m == 0.0f || e == 128) e = 0;  // nothing to scale; an infinity stays one
      e = min(max(e, -126), 126);
      const float inv = exp2_int(-e);
      if (lane == 0) row_mul[i] = a.scale * kLog2e * exp2_int(e);
#pragma unroll
      for (int k = 0; k < D / 64; ++k) {
        const uint32_t d = 64 * k + 2 * lane;  // elements d, d + 1 of piece d / 32
        uint8_t *dst = qf + ((i / 8) * kPieces + d / 32) * 512 + (4 * (i % 8) + d % 32 / 8) * 16 + d % 8 * 2;
        const float v0 = x[2 * k] * inv, v1 = x[2 * k + 1] * inv;
        const uint32_t hi = pack_f16(v0, v1);
        *reinterpret_cast<uint32_t *>(dst) = hi;
        if constexpr (kSplit)
          *reinterpret_cast<uint32_t *>(dst + S::kQ / 2) = pack_f16_rest(v0, v1, hi);
      }
    }
    __syncthreads();

    float o[kPieces][2][NT][4], mx[NT][2], ls[NT][2], mul[NT][2];
    float lmax = -INFINITY;  // the largest log2(v scale) that mx may stand for
    uint32_t see_lo[NT][2], see_hi[NT][2];  // keys [lo, hi] of this lane's packed rows
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint32_t i = 8 * t + 2 * c + k;
        mul[t][k] = row_mul[i];
        mx[t][k] = -INFINITY;
        ls[t][k] = 0.0f;
        const uint32_t pos = pos0 + (row0 + min(i, rows - 1)) / a.gqa;
        see_hi[t][k] = pos;
        see_lo[t][k] = a.window && pos >= a.window ? pos - a.window + 1 : 0;
      }
#pragma unroll
    for (int p = 0; p < kPieces; ++p)
#pragma unroll
      for (int mt = 0; mt < 2; ++mt)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int k = 0; k < 4; ++k) o[p][mt][t][k] = 0.0f;
    // blocks inside [all_lo, all_hi] are seen whole by every row
    const uint32_t all_hi = pos0 + tok_lo;
    const uint32_t all_lo = a.window && pos0 + tok_hi >= a.window ? pos0 + tok_hi - a.window + 1 : 0;

    for (uint32_t step = 0; step < steps; ++step) {
      if (step / 32 != batch) {
        cur = nxt;
        ++batch;
        nxt = entry(32 * (batch + 1) + lane);
      }
      const float ks = __shfl_sync(0xffffffffu, cur.ks, step % 32), vs = __shfl_sync(0xffffffffu, cur.vs, step % 32);
      const bool have = __shfl_sync(0xffffffffu, (int)(cur.rec != ~0ull), step % 32) != 0;
      auto stage = [&]() -> uint8_t * {  // the next record, once it is there
        const uint32_t st = taken % kStages;
        if (!mbar_wait_bounded(bar_u + 8 * st, (taken / kStages) & 1)) raise_error(a.err, kDevWaitTimeout);
        ++taken;
        return ring + st * S::kRecord;
      };
      auto release = [&]() {  // a record has been read: its stage takes the next copy
        __syncwarp();
        if (to_issue < 2 * steps) issue();
      };
      const uint8_t *const kr = stage();

      // ---- S^T = K Q^T
      // (two chains of accumulators: an MMA's result is 24 cycles away)
      // (the small terms apart: the tensor core cuts off a sum's last bits at every addition, and one chain
      // for both left 1.6e-6 of one f32 row's output on 640 keys for 0.4e-6, at 1 to 4 % less time)
      constexpr int kChains = kSplit ? 4 : 2;
      float s[NT][kChains][4];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int w = 0; w < kChains; ++w)
#pragma unroll
          for (int k = 0; k < 4; ++k) s[t][w][k] = 0.0f;
#pragma unroll
      for (int p = 0; p < kPieces; ++p) {
        const uint4 k4 = *reinterpret_cast<const uint4 *>(kr + p * 512 + lane * 16);
        uint32_t a0[4], a1[4];
        e4m3x4_f16(k4.x, a0[0], a0[2]);
        e4m3x4_f16(k4.y, a1[0], a1[2]);
        e4m3x4_f16(k4.z, a0[1], a0[3]);
        e4m3x4_f16(k4.w, a1[1], a1[3]);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int w = 0; w < (kSplit ? 2 : 1); ++w) {
            const uint4 q = *reinterpret_cast<const uint4 *>(qf + w * (S::kQ / 2) + (t * kPieces + p) * 512 + lane * 16);
            mma_f16_16816(s[t][2 * w], a0, q.x, q.y);
            mma_f16_16816(s[t][2 * w + 1], a1, q.z, q.w);
          }
      }

      release();

      // ---- scores, masks, running maximum
      uint8_t *const vr = stage();
      float top[NT][2];
      const float lv = (float)kv8_scale_exponent(vs);
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float x = s[t][0][k] + s[t][1][k];
          if constexpr (kSplit) x += s[t][2][k] + s[t][3][k];
          s[t][0][k] = x * ks * mul[t][k & 1];
        }
      const uint32_t key0 = (first + block_of(step)) * kKv8Block;
      if (!have || key0 < all_lo || key0 + kKv8Block - 1 > all_hi) {
        // Some row does not see all of the block.  A token no row sees is taken out of V (its
        // bytes may be anything); one whose V holds a NaN is taken out too and makes the
        // rows that do see it NaN.
        uint32_t nan = 0;
        uint4 *const own = reinterpret_cast<uint4 *>(vr) + lane;  // + 32 p
        if (have) {
#pragma unroll
          for (int p = 0; p < kPieces; ++p) {
            const uint4 v = own[32 * p];
            nan |= ((v.x & 0x7F7F7F7Fu) + 0x01010101u) | ((v.y & 0x7F7F7F7Fu) + 0x01010101u) |
                   ((v.z & 0x7F7F7F7Fu) + 0x01010101u) | ((v.w & 0x7F7F7F7Fu) + 0x01010101u);
          }
          nan &= 0x80808080u;
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) nan |= __shfl_xor_sync(0xffffffffu, nan, w);
        } else {
          nan = 0x80808080u;  // nothing was read: whatever the stage holds goes
        }
        if (__any_sync(0xffffffffu, nan != 0)) {
          const uint32_t keep = ~((nan >> 7) * 0xFFu);
#pragma unroll
          for (int p = 0; p < kPieces; ++p) {
            uint4 v = own[32 * p];
            v.x &= keep; v.y &= keep; v.z &= keep; v.w &= keep;
            own[32 * p] = v;
          }
          fence_proxy_async();  // before the stage's next copy
        }
        // token g is byte g % 2 of the lanes with c = g / 2, token g + 8 two bytes on
        const uint32_t nan_g = __shfl_sync(0xffffffffu, nan, g / 2) >> (8 * (g & 1));
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t key = key0 + g + (k >> 1) * 8;
            const bool seen = have && key >= see_lo[t][k & 1] && key <= see_hi[t][k & 1];
            float x = s[t][0][k];
            if ((nan_g >> (16 * (k >> 1))) & 0x80u) x = NAN;
            s[t][0][k] = seen ? x : -INFINITY;
          }
      }
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int k = 0; k < 2; ++k) top[t][k] = fmaxf(s[t][0][k], s[t][0][k + 2]);
      if (lv < lmax - kFar && have) {
        // mx may stand for a scale far above this one's: down to what this record's own would be
        bool later = false;  // a row that sees nothing of it: its mx stays
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float m = top[t][k], big = ls[t][k];
#pragma unroll
            for (int p = 0; p < kPieces; ++p)
#pragma unroll
              for (int mt = 0; mt < 2; ++mt) big = fmaxf(big, fmaxf(fabsf(o[p][mt][t][k]), fabsf(o[p][mt][t][k + 2])));
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) {
              m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, w));
              big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, w));
            }
            const int room = kLargest + 127 - (int)(__float_as_uint(big) >> 23);
            const float down = fminf(mx[t][k] - ceilf(m + lv), (float)min(room, 126));
            if (m == -INFINITY) {
              later |= mx[t][k] != -INFINITY;
            } else if (down > 0.0f) {
              const float f = exp2_int((int)down);
              mx[t][k] -= (float)(int)down;
              ls[t][k] *= f;
#pragma unroll
              for (int p = 0; p < kPieces; ++p)
#pragma unroll
                for (int mt = 0; mt < 2; ++mt) {
                  o[p][mt][t][k] *= f;
                  o[p][mt][t][k + 2] *= f;
                }
            }
          }
        if (!__any_sync(0xffffffffu, later)) lmax = lv;
      }
      if (have) lmax = fmaxf(lmax, lv);
      bool moved = false;
      float shift[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float m = top[t][k];
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, w));
          top[t][k] = fmaxf(ceilf(m + lv), mx[t][k]);
          moved |= top[t][k] != mx[t][k];
          shift[t][k] = top[t][k] == -INFINITY ? 0.0f : lv - (top[t][k] - kPOffset);
        }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float f = mx[t][k] == -INFINITY ? 0.0f : ex2(mx[t][k] - top[t][k]);
            mx[t][k] = top[t][k];
            ls[t][k] *= f;
#pragma unroll
            for (int p = 0; p < kPieces; ++p)
#pragma unroll
              for (int mt = 0; mt < 2; ++mt) {
                o[p][mt][t][k] *= f;
                o[p][mt][t][k + 2] *= f;
              }
          }
      }

      // ---- P^T as B operands
      uint32_t pb[NT][kSplit ? 2 : 1][2];
      const float unv = ex2(-lv);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float pr[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) pr[k] = ex2(s[t][0][k] + shift[t][k & 1]);
        ls[t][0] = fmaf(pr[0] + pr[2], unv, ls[t][0]);
        ls[t][1] = fmaf(pr[1] + pr[3], unv, ls[t][1]);
        const uint32_t p0 = pack_f16(pr[0], pr[1]), p1 = pack_f16(pr[2], pr[3]);
        pb[t][0][0] = movmatrix_trans(p0);
        pb[t][0][1] = movmatrix_trans(p1);
        if constexpr (kSplit) {
          pb[t][1][0] = movmatrix_trans(pack_f16_rest(pr[0], pr[1], p0));
          pb[t][1][1] = movmatrix_trans(pack_f16_rest(pr[2], pr[3], p1));
        }
      }

      // ---- O^T += V^T P^T
#pragma unroll
      for (int p = 0; p < kPieces; ++p) {
        const uint4 v = *reinterpret_cast<const uint4 *>(vr + p * 512 + lane * 16);
        uint32_t a0[4], a1[4];
        e4m3x4_f16(v.x, a0[0], a0[2]);
        e4m3x4_f16(v.y, a0[1], a0[3]);
        e4m3x4_f16(v.z, a1[0], a1[2]);
        e4m3x4_f16(v.w, a1[1], a1[3]);
#pragma unroll
        for (int t = 0; t < NT; ++t)
          if constexpr (kSplit) {
            // A block's sum, then f32 additions: the tensor core cuts off what is below the last bit of the sum
            // so far, always toward zero.  One row on 120000 keys of each of 96 sequences erred by 1.9e-5 so,
            // by 6e-7 now (a plain f32 softmax: 1.3e-6).  It takes 1 to 3 % more time, 5 to 8 % with 16 rows.
            float x0[4] = {0.0f, 0.0f, 0.0f, 0.0f}, x1[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 1; w >= 0; --w) {
              mma_f16_16816(x0, a0, pb[t][w][0], pb[t][w][1]);
              mma_f16_16816(x1, a1, pb[t][w][0], pb[t][w][1]);
            }
#pragma unroll
            for (int k = 0; k < 4; k += 2) {
              add_f32x2(o[p][0][t] + k, x0 + k);
              add_f32x2(o[p][1][t] + k, x1 + k);
            }
          } else {
            mma_f16_16816(o[p][0][t], a0, pb[t][0][0], pb[t][0][1]);
            mma_f16_16816(o[p][1][t], a1, pb[t][0][0], pb[t][0][1]);
          }
      }
      release();
    }

    // ---- merge the warps
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float l = ls[t][k];
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) l += __shfl_xor_sync(0xffffffffu, l, w);
        if (g == 0) {
          wm[warp][8 * t + 2 * c + k] = mx[t][k];
          wl[warp][8 * t + 2 * c + k] = l;
        }
      }
    __syncthreads();  // every warp's ring is free
    float *const mo = reinterpret_cast<float *>(smem);
    if ((uint32_t)warp < busy) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int p = 0; p < kPieces; ++p)
#pragma unroll
          for (int k = 0; k < 2; ++k)
            *reinterpret_cast<float4 *>(mo + (size_t)(warp * kRows + 8 * t + 2 * c + k) * S::kLdO + 32 * p + 4 * g) =
                make_float4(o[p][0][t][k], o[p][0][t][k + 2], o[p][1][t][k], o[p][1][t][k + 2]);
    }
    const bool whole = s0 == 0 && s1 == count;
    // a problem that starts inside the run, or at its head: at most one of each leaves a part
    const uint32_t slot = 2 * blockIdx.x + (at > begin ? 1 : 0);
    float *const part_ml = a.part, *const part_o = a.part + (size_t)2 * gridDim.x * kRows * 2;
    if (threadIdx.x < kRows) {
      const uint32_t i = threadIdx.x;
      float m = -INFINITY, l = 0.0f;
#pragma unroll
      for (int w = 0; w < kDecWarps; ++w) m = fmaxf(m, wm[w][i]);
#pragma unroll
      for (int w = 0; w < kDecWarps; ++w) {
        const float f = wm[w][i] == -INFINITY ? 0.0f : ex2(wm[w][i] - m);
        fac[w][i] = f;
        l += wl[w][i] * f;
      }
      if (whole) {
        row_inv[i] = l == 0.0f ? 0.0f : 1.0f / l;
      } else {
        row_inv[i] = 1.0f;
        part_ml[((size_t)slot * kRows + i) * 2] = m;
        part_ml[((size_t)slot * kRows + i) * 2 + 1] = l;
      }
    }
    __syncthreads();
    auto out_row = [&](uint32_t i) {
      const uint32_t pr = row0 + i;
      return static_cast<T *>(a.out) + (size_t)(r.r0 + pr / a.gqa) * a.out_ld + (size_t)(h * a.gqa + pr % a.gqa) * D;
    };
    for (uint32_t x = threadIdx.x; x < rows * (D / 4); x += kDecThreads) {
      const uint32_t i = x / (D / 4), d = x % (D / 4) * 4;
      float4 sum = make_float4(0, 0, 0, 0);
#pragma unroll 4
      for (uint32_t w = 0; w < busy; ++w) {
        const float4 v = *reinterpret_cast<const float4 *>(mo + (size_t)(w * kRows + i) * S::kLdO + d);
        const float f = fac[w][i];
        sum.x = fmaf(v.x, f, sum.x);
        sum.y = fmaf(v.y, f, sum.y);
        sum.z = fmaf(v.z, f, sum.z);
        sum.w = fmaf(v.w, f, sum.w);
      }
      if (whole) {
        const float inv = row_inv[i], y[4] = {sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv};
        store_vec<T, 4>(out_row(i) + d, y);
      } else {
        *reinterpret_cast<float4 *>(part_o + ((size_t)slot * kRows + i) * D + d) = sum;
      }
    }
    if (!whole) {
      const uint32_t c0 = (uint32_t)(at / run), c1 = (uint32_t)((at + count - 1) / run);
      merge_parts<T, D, kRows>(a, Parts{c0, c1 - c0 + 1, 2 * c0 + (at > run * c0 ? 1 : 0), r.r0, row0, rows, h}, sh);
    }
    merged = true;
  }
}

using AttnKernel = void (*)(const Kv8AttnArgs);
struct DecVariant {
  AttnKernel fn;
  uint32_t smem, ctas;
};
template <typename T, int D, int NT>
DecVariant variant() {
  using S = DecShape<D, NT, sizeof(T) == 4>;
  return {kv8_decode_kernel<T, D, NT>, (uint32_t)S::kSmem, (uint32_t)S::kCtas};
}
// Variant i (0, 1: 8, 16 packed rows) of a head size: the output of 8 NT rows takes D NT / 4 registers
// per thread, of which there may be 128.
template <typename T>
DecVariant variant(uint32_t d, uint32_t i) {
  switch (d) {
    case 64: return i == 0 ? variant<T, 64, 1>() : variant<T, 64, 2>();
    case 128: return i == 0 ? variant<T, 128, 1>() : variant<T, 128, 2>();
    case 256: return i == 0 ? variant<T, 256, 1>() : variant<T, 256, 2>();
    default: return variant<T, 512, 1>();
  }
}
DecVariant dec_variant(sx_dtype t, uint32_t d, uint32_t i) {
  return t == SX_F32 ? variant<float>(d, i) : variant<__nv_bfloat16>(d, i);
}

}  // namespace

// Two parts per CTA of the decode kernel: up to 16 rows of {m, l}, and 4096 output values with one
// CTA per SM, half as many with two.
size_t kv8_part_bytes(int num_sms) { return (size_t)2 * num_sms * (2 * 16 * 2 + 4096) * sizeof(float); }

cudaError_t prepare_kv8_attn() {
  for (uint32_t d : {64u, 128u, 256u, 512u})
    for (sx_dtype t : {SX_F32, SX_BF16})
      for (uint32_t i = 0; i < 2; ++i) {
        const DecVariant v = dec_variant(t, d, i);
        const cudaError_t e = cudaFuncSetAttribute(v.fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)v.smem);
        if (e != cudaSuccess) return e;
      }
  return cudaSuccess;
}

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
  sx::Kv8AttnArgs a{};
  a.c = *c;
  a.q = q;
  a.out = out;
  a.q_ld = q_ld;
  a.out_ld = out_ld;
  a.row_start = row_start;
  a.kv_len = kv_len;
  a.tokens = tokens;
  a.num_q = num_q;
  a.window = window;
  a.gqa = num_q / c->num_kv;
  a.scale = scale;
  a.part = e->kv8_part;
  a.cnt = e->kv8_cnt;
  e->scratch_used = true;
  a.err = e->err_dev;
  // Packed rows of an average sequence: past 16 the tcgen05 form, which takes 128 at a time, where there
  // may be enough to do: its smallest call takes 12.5 (head size 128) to 14 us (256), this form's 7 to 8, but
  // this one reads a key once for 16 rows.  The table's width (and the window) bounds the keys, which are
  // on the device.  40 rows of 30 sequences of up to 540 keys 14.3 us here, 23.3 there (head size 256); of
  // 32 sequences of 8000 49.7 and 37.9; at the limit, 64 rows and 2 kv heads of 30 sequences of 540 keys,
  // 28.0 and 23.5 (256), 18.1 and 20.3 (128).
  const uint64_t rows = (uint64_t)tokens * a.gqa;
  const uint64_t avg = (uint64_t)((tokens + c->num_seqs - 1) / c->num_seqs) * a.gqa;
  uint64_t keys = (uint64_t)c->max_pages * c->page_tokens;
  if (window) keys = std::min<uint64_t>(keys, (uint64_t)window + tokens / c->num_seqs);
  const bool little = (rows / 16 + c->num_seqs) * c->num_kv * (keys + 128) <= 800ull * e->num_sms;
  if (avg > 16 && c->head_dim <= 256 && !little)
    return sx_host_cuda_status(sx::launch_kv8_prompt(a, t, e->num_sms, e->stream), "kv8_attn launch");
  const sx::DecVariant v = sx::dec_variant(t, c->head_dim, avg <= 8 ? 0 : 1);
  return sx_host_cuda_status(
      sx::launch_chained(v.fn, dim3(std::min(e->num_sms * v.ctas, sx::kMaxParts * sx::kPartGroup)), dim3(sx::kDecThreads), v.smem, e->stream, 1, a),
      "kv8_attn launch");
}

extern "C" SX_API uint32_t sx_kv8_attn_args_bytes(void) { return (uint32_t)sizeof(sx_kv8_attn_args); }
extern "C" SX_API sx_status sx_dispatch_kv8_attn_args(sx_engine *e, const sx_kv8_attn_args *a) {
  if (!a) {
    sx_host_set_error("kv8_attn: null arguments");
    return SX_ERR_INVALID;
  }
  return sx_dispatch_kv8_attn(e, &a->cache, (sx_dtype)a->dtype, a->q, a->out, a->q_ld, a->out_ld, a->row_start,
                              a->kv_len, a->tokens, a->num_q, a->window, a->scale);
}
