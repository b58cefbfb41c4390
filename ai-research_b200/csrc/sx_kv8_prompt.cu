// sx_kv8_prompt.cu -- attention over the paged 8-bit KV cache for many rows per kv head, on
// tcgen05 tensor cores (include/sx.h, sx_dispatch_kv8_attn).
//
//   S = Q K^T (128 packed rows x kTokens keys),  P = 2^(x + log2(v scale) - m + 6),  O += P V
//
// 128 packed rows (new tokens x q heads of one kv head) are the M of both products; S and O live in
// tensor memory, P goes back there as f16 over S and is the second product's A operand.  e4m3 is
// exact in f16, so K and V are widened on the way to shared memory; f32 rows split Q and P into two
// f16 terms, with twice the products.  Warps:
//   0 .. 7   softmax, two threads per row, each for half of a tile's 64 keys: their part of the row of S
//            from tensor memory, P back.  The maximum that the exponentials refer to moves only when it
//            grows by 2^8, which the two warps of a row vote on; the row of O is then rescaled in tensor
//            memory.  P's exponent is kOffset where the reference is.  f16 holds 22 bits of a P down to 2^-3
//            (two terms; 11 bits down to 2^-14 with one) and multiples of 2^-24 below: enough while V's
//            scales are within 2^kFar of the problem's largest.  What is further below is added to O in f32
//            (add_far).
//   8 ..     widen K and V.  A warp takes a pair of blocks (32 tokens): the cache's 16-byte pieces
//            become 16-byte stores of the 128-byte-swizzled tiles for a fitting order of the tokens
//            (tile position 32 q + 8 (t % 8 / 2) + 4 half + 2 (t / 8) + t % 2) and of V's elements
//            (tile row 32 p + 8 (d % 4) + f(d % 32 / 4), f a permutation of 8).  The softmax undoes
//            the first in its masks and scales, the output the second: both are register indexes.
//            K is a tile ahead of V, so that no widening waits for the softmax before it.
//   last     cuts the CTA's run into problems, one ahead, issues the products, and says which tiles have
//            records that are far below.
// Two S, K and V tiles let a tile's first product, and the widening for it, run beside the softmax of the
// one before; up to head size 128 two CTAs share an SM.
//
// What bounds it is the roles' own instructions: at head size 128 a CTA's tile takes 2300 cycles, of
// which the tensor cores work 650.  Code size and spills count for as much as instructions (a kernel
// unrolled throughout spent 20 cycles an instruction, fetching), so what runs seldom is out of line, loops
// stay loops, and what describes a problem or a block is in shared memory.  Measured: 4 prompts of up to
// 4096 tokens behind 4096 (16 q and 8 kv heads of 128, bf16) 545 us, 743 TFLOP/s or 44 % of the measured
// rate, at the 1.5 GHz that the power cap leaves (565 in a long row of calls); 4 of 2048 tokens with head size
// 256 111.7 us (f32 rows 168.6); 5 drafts of 32 sequences on up to 16000 keys (8 q heads, 1 kv head of 256)
// 58 us (f32 84), where 30 tiles a CTA take 37 -- 88 of a tile's 128 rows are padding -- and cutting the
// line, bringing Q, the output and the merge the rest.  Four softmax warps with whole rows took a third more for
// the first, one barrier for K and V an eighth.  A second look ahead for pages and scales, and Q
// brought by the roles that wait for it, were slower by 5 and 10 %: more code.
//
// Work is the line of sx_kv8_attn.cu with problems of their own length: row group k of a sequence
// sees pos0 + 128 (k + 1) / G keys at most, so the line counts keys x G, whose sums are closed
// forms; a tile belongs to the CTA in whose run its first key lies.  Parts of cut problems meet in a
// second kernel.
#include "sx_host.h"
#include "sx_kv8.cuh"
#include "sx_launch.cuh"
#include "sx_tcgen05.cuh"

namespace sx {
namespace {

constexpr uint32_t kRows = 128;      // packed rows of a problem
constexpr int kSoft = 8;             // softmax warps
constexpr float kSlack = 8.0f, kOffset = 15.0f - kSlack;  // P is at most 2^15
constexpr float kMinScale = 1.17549435e-38f;  // a product with a masked -inf stays that

template <int D, bool SPLIT>
struct PromptShape {
  static constexpr int kCtas = D <= 128 && !(D == 128 && SPLIT) ? 2 : 1;  // per SM
  static constexpr int kTokens = 64;                                      // of a tile
  static constexpr int kStages = D == 256 && SPLIT ? 1 : 2;               // K and V tiles
  static constexpr int kS = 2;                                            // S tiles
  static constexpr int kWiden = kCtas == 2 ? 4 : 8;                       // warps that widen
  static constexpr int kThreads = (kSoft + kWiden + 1) * 32;
  static constexpr int kTerms = SPLIT ? 2 : 1;
  static constexpr float kFar = SPLIT ? 10.0f : 20.0f;                    // P of the largest is 2^-3, 2^-13 there
  static constexpr int kQTerm = (int)kRows * D * 2;
  static constexpr int kTile = kTokens * D * 2;
  static constexpr int kStaged = kTokens * D;                             // a tile's V as it comes
  static constexpr int kSmem = kTerms * kQTerm + kStages * 2 * kTile + kStaged + 1024;  // + alignment
  // tensor memory columns: S tiles (P over them), low terms of P, O
  static constexpr int kLow = kS * kTokens;
  static constexpr int kO = kLow + (SPLIT ? kS * kTokens / 2 : 0);
  static constexpr int kTotal = SPLIT && kCtas == 1 && kO + 2 * D <= 512 ? kO + D : 0;  // sums of O (fold_row), where there is room
  // Tiles after which f32 rows' O is added to a sum apart.  The tensor core cuts products off at the last bit
  // of the sum so far, always toward zero: a bias that grows with the sum's length, 9e-6 of the output on
  // 6000 keys of equal weight (head size 256) and 2.3e-5 on 31000, where the products' f32 sums err by 1.6e-6.
  // Sums of 8 tiles leave 1.7e-6 on any length, of 16 2.6e-6, of 4 (in tensor memory) 0.9e-6.  f32 prompts
  // and drafts take 10 to 13 % more time for it; bf16 rows round by 2^-9 at the end and go without.
  static constexpr uint32_t kFold = kTotal ? 4 : 8;
  static constexpr int kCols = kO + D <= 256 ? 256 : 512;
  static_assert(kO + D <= 512 && kCols * kCtas <= 512, "tensor memory");
};

// What starting and ending a problem costs, in tiles of 2400 cycles (with 3, 6, 8, 10 and 16: drafts over
// 16000 keys 74, 60, 58.5, 57.5 and 59 us; prompts of 2048 with head size 256 129, 115, 111.5, 113 and 122).
// What cutting one costs, a second start and an end that leaves a part (4 prompts of 1500 in a window of
// 300, head size 128: 48.8 us uncut, 60.4 cut).
constexpr uint32_t kPromptOver = 8, kCutTiles = 16;

// Costs on the line: keys x G of a row group, at most `cap` with a window, plus `over`.
struct GroupCost {
  uint64_t base, cap, over;  // pos0 * G; the most a group sees; what starting one costs
  uint32_t groups;
  SX_DEV uint64_t of(uint32_t k) const {
    const uint64_t c = base + (uint64_t)kRows * (k + 1);
    return (c < cap ? c : cap) + over;
  }
  SX_DEV uint64_t before(uint32_t k) const {  // of the groups below k
    uint64_t full = cap > base ? (cap - base) / kRows : 0;  // groups under the cap
    if (full > k) full = k;
    return full * base + kRows * (full * (full + 1) / 2) + (k - full) * cap + k * over;
  }
};

SX_DEV void ld_shared16(uint32_t src, uint32_t (&v)[4]) {
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];\n"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
               : "r"(src)
               : "memory");
}
SX_DEV void st_shared16(uint32_t dst, const uint32_t (&v)[4]) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(dst), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3])
               : "memory");
}

// Waits are for a phase's parity, so a waiter must be sure of the phase before and ahead of the one
// after.  Every kind of event has a barrier for even and one for odd tiles: roles and softmax warps run
// a tile ahead of one another, and S of a tile done means that all of two tiles back is.
struct PromptBars {
  uint32_t at;
  SX_DEV explicit PromptBars(uint32_t p) : at(p) {}
  SX_DEV uint32_t k_full(uint32_t t) const { return at + 8 * (t & 1); }         // K in place
  SX_DEV uint32_t v_full(uint32_t t) const { return at + 16 + 8 * (t & 1); }    // V in place
  SX_DEV uint32_t p_full(uint32_t t) const { return at + 32 + 8 * (t & 1); }    // P in place
  SX_DEV uint32_t s_done(uint32_t t) const { return at + 48 + 8 * (t & 1); }    // products done
  SX_DEV uint32_t pv_done(uint32_t t) const { return at + 64 + 8 * (t & 1); }
};

constexpr uint32_t kNoRecord = ~0u;  // (2^32 record pairs of 2 KB are past any memory)

// What stands in for a block that is not there (a branch around its loads would end in copies that
// wait for them).
__device__ uint4 g_no_block[32 * 256 / 16];

// Whether any thread of the two warps that share rows says so: one barrier for both to meet at.
SX_DEV bool pair_any(uint32_t bar, bool mine) {
  uint32_t any;
  asm volatile(
      "{\n.reg .pred p, q;\nsetp.ne.u32 p, %1, 0;\nbarrier.cta.red.or.pred q, %2, 64, p;\nselp.u32 %0, 1, 0, q;\n}\n"
      : "=r"(any)
      : "r"((uint32_t)mine), "r"(bar)
      : "memory");
  return any;
}

// This thread's row of `cols` f32 columns of tensor memory times f.  A whole warp calls it, seldom:
// out of line it stays out of the way of the loop's instructions.
__device__ __noinline__ void rescale_row(uint32_t col, int cols, float f) {
#pragma unroll 1
  for (int d = 0; d < cols; d += 16) {
    uint32_t o[16];
    tmem_ld16(col + d, o);
    tmem_wait_ld(o);
#pragma unroll
    for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
    tmem_st16(col + d, o);
  }
}

// column k of a half is token 16 (k / 4 % 2) + 8 (k / 2 % 2) + 2 (k / 8) + k % 2 of it, record k / 4 % 2
SX_DEV constexpr uint32_t key_bit(int k) { return 1u << (16 * ((k >> 2) & 1) + 8 * ((k >> 1) & 1) + 2 * (k >> 3) + (k & 1)); }

// A tile's records whose log2(v scale) is under `below`: their part of this thread's row of O, in f32 from
// the scores at s_col and the f16 tile of V, by both halves of a row in turn.  `facts`: shared memory of the
// half's two records'.  Their scores, and those of keys that `vis` lacks, are -inf afterwards.  Returns their
// part of the softmax's sum.  It takes 30 tiles' time: scales of one head that differ by over 2^10 are no
// ordinary values.  Out of line, and plain values for arguments: references to what the loop reads took 15 %
// of long prompts' time, and the call itself takes 4 % with head size 128 (bf16), 1 to 2 % elsewhere.
template <int D>
__device__ __noinline__ float add_far(uint32_t o_col, uint32_t v_tile, uint32_t s_col, uint32_t vis, uint32_t facts, float mul,
                                      float ref, float below, bool begin) {
  const uint32_t half = threadIdx.x / kRows, pair_bar = 2 + ((threadIdx.x >> 5) & 3);
  uint32_t s[32], b[2][4];
  float x[32], l = 0.0f;
  ld_shared16(facts, b[0]);
  ld_shared16(facts + 16, b[1]);
  tmem_ld32(s_col, s);
  tmem_wait_ld(s);
  const float shift = ref == -INFINITY ? 0.0f : ref - kOffset;
  auto factor = [&](int h) { return fmaxf(__uint_as_float(b[h][0]) * mul, kMinScale); };
  auto offset = [&](int h) {
    const float lv = __uint_as_float(b[h][1]);
    return lv < below && lv > (float)kKv8MinExp ? lv - shift : -INFINITY;
  };
  const float2 km = make_float2(factor(0), factor(1)), off = make_float2(offset(0), offset(1));
  const float2 unv = make_float2(__uint_as_float(b[0][2]), __uint_as_float(b[1][2]));
#pragma unroll
  for (int k = 0; k < 32; ++k) {
    const bool second = (k >> 2) & 1;
    const float add = second ? off.y : off.x;
    if (!(vis & key_bit(k))) s[k] = 0xFF800000u;
    x[k] = add != -INFINITY ? ex2(fmaf(__uint_as_float(s[k]), second ? km.y : km.x, add)) : 0.0f;
    l = fmaf(x[k], second ? unv.y : unv.x, l);
    if (add != -INFINITY) s[k] = 0xFF800000u;
  }
  tmem_st16(s_col, *reinterpret_cast<const uint32_t(*)[16]>(s));
  tmem_st16(s_col + 16, *reinterpret_cast<const uint32_t(*)[16]>(s + 16));
  if (begin) {  // zeros in O
#pragma unroll
    for (int k = 0; k < 16; ++k) s[k] = 0;
#pragma unroll 1
    for (int d = half * (D / 2); d < (int)(half + 1) * (D / 2); d += 16)
      tmem_st16(o_col + d, *reinterpret_cast<const uint32_t(*)[16]>(s));
  }
  tmem_wait_st();
#pragma unroll 1
  for (uint32_t turn = 0; turn < 2; ++turn) {
    tc_fence_before();
    pair_any(pair_bar, false);
    tc_fence_after();
    if (turn == half) {
#pragma unroll 1
      for (int d = 0; d < D; ++d) {
        float o = __uint_as_float(tmem_ld1(o_col + d));
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t v[4];
          ld_shared16(v_tile + d * 128 + (((4 * half + c) ^ (d & 7)) << 4), v);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 y = __half22float2(*reinterpret_cast<const __half2 *>(&v[k]));
            o = fmaf(x[8 * c + 2 * k], y.x, fmaf(x[8 * c + 2 * k + 1], y.y, o));
          }
        }
        tmem_st1(o_col + d, __float_as_uint(o));
      }
      tmem_wait_st();
    }
  }
  tc_fence_before();
  return l;
}

// f32 rows: this thread's half of its row of O, `cols` columns from o_col on, is added to a sum whose
// reference is in shared memory at ref_at: in tensor memory at t_col (0: there is no room), or in the
// workspace at `acc`, a row every kRows floats.  Only this thread touches it, so additions are in order; in
// the workspace they are left to L2 while the reference stays.  A whole warp calls it.
SX_DEV float ref_factor(float was, float ref) { return was == ref ? 1.0f : was == -INFINITY ? 0.0f : ex2(was - ref); }
SX_DEV float ld_shared_f32(uint32_t at) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];\n" : "=f"(v) : "r"(at) : "memory");
  return v;
}
SX_DEV void st_shared_f32(uint32_t at, float v) { asm volatile("st.shared.f32 [%0], %1;\n" ::"r"(at), "f"(v) : "memory"); }
template <bool IN_TMEM>
__device__ __noinline__ void fold_row(uint32_t o_col, uint32_t t_col, int cols, float *acc, uint32_t ref_at, float ref, bool first) {
  const float f = first ? 1.0f : ref_factor(ld_shared_f32(ref_at), ref);
  st_shared_f32(ref_at, ref);
  const bool moved = __any_sync(0xffffffffu, f != 1.0f);
#pragma unroll 1
  for (int d = 0; d < cols; d += 16, acc += 16 * kRows) {
    uint32_t o[16];
    tmem_ld16(o_col + d, o);
    if constexpr (IN_TMEM) {
      uint32_t t[16];
      tmem_ld16(t_col + d, t);
      tmem_wait_ld(o);
      tmem_wait_ld(t);
#pragma unroll
      for (int k = 0; k < 16; ++k)
        o[k] = first ? o[k] : __float_as_uint(fmaf(__uint_as_float(t[k]), f, __uint_as_float(o[k])));
      tmem_st16(t_col + d, o);
    } else if (first) {
      tmem_wait_ld(o);
#pragma unroll
      for (int k = 0; k < 16; ++k) __stcg(acc + k * kRows, __uint_as_float(o[k]));
    } else if (!moved) {
      tmem_wait_ld(o);
#pragma unroll
      for (int k = 0; k < 16; ++k) atomicAdd(acc + k * kRows, __uint_as_float(o[k]));
    } else {
      float v[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) v[k] = __ldcg(acc + k * kRows);
      tmem_wait_ld(o);
#pragma unroll
      for (int k = 0; k < 16; ++k) __stcg(acc + k * kRows, fmaf(v[k], f, __uint_as_float(o[k])));
    }
  }
  if constexpr (IN_TMEM) tmem_wait_st();
}
// and at a problem's end the sum to O
template <bool IN_TMEM>
__device__ __noinline__ void unfold_row(uint32_t o_col, uint32_t t_col, int cols, const float *acc, uint32_t ref_at, float ref) {
  const float f = ref_factor(ld_shared_f32(ref_at), ref);
#pragma unroll 2
  for (int d = 0; d < cols; d += 16, acc += 16 * kRows) {
    uint32_t o[16], v[16];
    if constexpr (IN_TMEM) {
      tmem_ld16(t_col + d, v);
    } else {
#pragma unroll
      for (int k = 0; k < 16; ++k) v[k] = __float_as_uint(__ldcg(acc + k * kRows));
    }
    tmem_ld16(o_col + d, o);
    tmem_wait_ld(o);
    if constexpr (IN_TMEM) tmem_wait_ld(v);
#pragma unroll
    for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(fmaf(__uint_as_float(v[k]), f, __uint_as_float(o[k])));
    tmem_st16(o_col + d, o);
  }
  tmem_wait_st();
}

enum Role { kSoftmax, kWidenKv, kProducts };

// 128 packed rows of one sequence and kv head, and the tiles [t0, t1) of their keys that this CTA takes.
struct Problem {
  uint32_t more;                 // 0: the run is over
  uint32_t r0, row0, rows, head; // first row of the sequence, first packed row, how many, kv head
  uint32_t seq, pos0;            // the sequence and the position of its first new row
  uint32_t first, blocks;        // first block that some row sees, how many
  uint32_t t0, t1;
  uint32_t all_lo, all_hi;       // keys that every row sees
  uint32_t slot, slot0, c0, parts;  // this part's place; that of the first part, its CTA, how many
  SX_DEV size_t row(const Kv8AttnArgs &a, uint32_t i) const { return r0 + (row0 + i) / a.gqa; }
  SX_DEV uint32_t col(const Kv8AttnArgs &a, uint32_t i) const {
    return (head * a.gqa + (row0 + i) % a.gqa) * a.c.head_dim;
  }
};

enum : uint32_t { kGone = 1, kApart = 2 };

// What the CTA's threads share.
template <int TOKENS, int WIDEN>
struct PromptShared {
  uint64_t bars[10];
  uint32_t tmem_slot, abort_flag;
  uint32_t nan_mask[2][TOKENS / 32];
  Problem problem[2];
  float row_mul[kRows];
  float row_top[2][kRows], row_sum[2][kRows];  // of the two halves of a tile's keys
  float fold_ref[2][kRows];                    // of the sum of earlier tiles' O
  // The blocks of 32 tiles: of a widening warp the record pairs (kNoRecord: nothing to read); of a pair
  // of blocks of a tile {k scale, log2(v scale), 1 / v scale, there}.
  alignas(8) uint32_t record[WIDEN][64];  // (read by twos)
  float4 facts[TOKENS / 32][64];
  // Of an even or odd tile: whether it has records that are not there or are far below (kGone, kApart), and
  // what log2(v scale) is far below.
  uint32_t odd_records[2];
  float far_below[2];
};

// A wait that runs out ends the CTA's waiting altogether: what follows runs through on whatever is
// there, and the error word says so.
__device__ __noinline__ void wait_longer(uint32_t b, uint32_t parity, volatile uint32_t *abort_flag, uint32_t *err) {
  if (*abort_flag) return;
  if (!mbar_wait_bounded(b, parity & 1)) {
    *abort_flag = 1;
    raise_error(err, kDevWaitTimeout);
  }
}

// block / blocks per page (up to 64): a product with 2^32 / blocks rounded up, at most one too much
struct PageDiv {
  uint32_t per, magic;
  SX_DEV explicit PageDiv(uint32_t page_tokens) : per(page_tokens / kKv8Block), magic(0xFFFFFFFFu / per + 1) {}
  SX_DEV uint32_t page(uint32_t x) const {
    const uint32_t q = per == 1 ? x : __umulhi(x, magic);
    return q * per > x ? q - 1 : q;
  }
};

// This CTA's run [begin, end) of the line, cut into problems: one warp, all lanes alike.
struct Schedule {
  uint64_t unit, begin, end, length, at, step;  // at: where the problem starts, step: its length
  uint32_t b, left, head, group;                // next sequence; problems left of the one before
  bool fresh;  // the first sequence: its first problems may lie before the run
  bool uncut;  // problems go whole to the CTA in whose run they start
  Kv8Rows r;
  GroupCost gc;

  SX_DEV GroupCost cost_of(const Kv8AttnArgs &a, const Kv8Rows &x) const {
    GroupCost k;
    k.base = (uint64_t)(x.len - x.n) * a.gqa;
    k.cap = a.window ? (uint64_t)a.window * a.gqa + kRows + 2 * a.gqa : ~0ull >> 1;
    k.over = kPromptOver * unit;
    k.groups = (x.n * a.gqa + kRows - 1) / kRows;
    return k;
  }
  SX_DEV uint64_t cost(const Kv8AttnArgs &a, uint32_t i, uint32_t &problems, uint64_t &longest) const {
    Kv8Rows x;
    if (!kv8_rows(a.c, a.row_start, a.kv_len, a.tokens, i, &x)) {
      if (blockIdx.x == 0) raise_error(a.err, kDevBadParams);
      return 0;
    }
    if (x.n == 0) return 0;
    const GroupCost k = cost_of(a, x);
    problems += k.groups * a.c.num_kv;
    longest = max(longest, k.of(k.groups - 1) - k.over);
    return k.before(k.groups) * a.c.num_kv;
  }
  __device__ __noinline__ void start(const Kv8AttnArgs &a, uint32_t tokens) {
    const int lane = threadIdx.x & 31;
    unit = (uint64_t)a.gqa * tokens;
    const uint32_t per = (a.c.num_seqs + 31) / 32;
    const uint32_t b0 = lane * per, b1 = min(a.c.num_seqs, b0 + per);
    uint64_t mine = 0, longest = 0;
    uint32_t problems = 0;
    for (uint32_t i = b0; i < b1; ++i) mine += cost(a, i, problems, longest);
    uint64_t incl = mine;
#pragma unroll 1
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    const uint64_t total = __shfl_sync(0xffffffffu, incl, 31);
    length = (total + gridDim.x - 1) / gridDim.x;
    length = length > a.min_run * unit ? length : a.min_run * unit;
    problems = __reduce_add_sync(0xffffffffu, problems);
#pragma unroll 1
    for (int o = 16; o > 0; o >>= 1) longest = max(longest, __shfl_xor_sync(0xffffffffu, longest, o));
    uncut = longest <= kCutTiles * unit + (problems <= gridDim.x ? length : 0);
    begin = length * blockIdx.x;
    end = begin + length < total ? begin + length : total;
    const uint32_t who = min(31, __popc(__ballot_sync(0xffffffffu, incl <= begin)));
    at = incl - mine;
    b = b0;
    if (lane == (int)who && begin < end)
      for (uint64_t n; (n = cost(a, b, problems, longest)) <= begin - at; at += n) ++b;
    at = __shfl_sync(0xffffffffu, at, who);
    b = __shfl_sync(0xffffffffu, b, who);
    if (begin >= end) at = end;  // no run for this CTA
    left = head = group = 0;
    step = 0;
    fresh = true;
  }
  // The next problem with a tile in the run.
  __device__ __noinline__ void next(const Kv8AttnArgs &a, uint32_t tile_blocks, Problem &out) {
    for (; at < end; at += step, --left) {
      if (left != 0) {
        if (++group == gc.groups) {
          group = 0;
          ++head;
        }
      }
      while (left == 0 && b < a.c.num_seqs) {  // the next sequence with rows
        const bool ok = kv8_rows(a.c, a.row_start, a.kv_len, a.tokens, b, &r);
        ++b;
        if (!ok || r.n == 0) continue;
        gc = cost_of(a, r);
        left = gc.groups * a.c.num_kv;
        head = group = 0;
        if (fresh) {
          fresh = false;
          const uint64_t per_head = gc.before(gc.groups);
          head = (uint32_t)((begin - at) / per_head);
          at += head * per_head;
          uint32_t lo = 0, hi = gc.groups - 1;  // the last group that starts at or before begin
          while (lo < hi) {
            const uint32_t mid = (lo + hi + 1) / 2;
            if (gc.before(mid) <= begin - at) lo = mid; else hi = mid - 1;
          }
          group = lo;
          at += gc.before(group);
          left -= head * gc.groups + group;
        }
      }
      if (left == 0) {  // the counts changed under the call
        at = end;
        break;
      }
      step = gc.of(group);
      Problem p;
      p.r0 = r.r0;
      p.row0 = group * kRows;
      p.rows = min(kRows, r.n * a.gqa - p.row0);
      p.head = head;
      p.seq = b - 1;
      p.pos0 = r.len - r.n;
      const uint32_t pos_lo = p.pos0 + p.row0 / a.gqa, pos_hi = p.pos0 + (p.row0 + p.rows - 1) / a.gqa;
      p.first = (a.window && pos_lo >= a.window ? pos_lo - a.window + 1 : 0) / kKv8Block;
      p.blocks = pos_hi / kKv8Block - p.first + 1;
      p.all_hi = pos_lo;
      p.all_lo = a.window && pos_hi >= a.window ? pos_hi - a.window + 1 : 0;
      const uint32_t count = (p.blocks + tile_blocks - 1) / tile_blocks;
      p.t0 = begin > at ? (uint32_t)((begin - at + unit - 1) / unit) : 0;
      const uint64_t until = (end - at + unit - 1) / unit;
      p.t1 = until < count ? (uint32_t)until : count;
      if (uncut) p.t1 = p.t0 == 0 ? count : 0;
      if (p.t0 >= p.t1) continue;  // no tile starts in the run
      // CTAs c0 .. c1 hold parts of this problem
      p.c0 = (uint32_t)(at / length);
      p.parts = (uint32_t)((at + (count - 1) * unit) / length) - p.c0 + 1;
      if (uncut) p.parts = 1;
      p.slot = 2 * blockIdx.x + (at > begin ? 1 : 0);
      p.slot0 = 2 * p.c0 + (at > length * p.c0 ? 1 : 0);
      p.more = 1;
      if ((threadIdx.x & 31) == 0) out = p;
      at += step;
      --left;
      return;
    }
    if ((threadIdx.x & 31) == 0) out.more = 0;
  }
};

// Q: power-of-two scaled f16 terms, K-major 128-byte swizzle, by all threads.
template <typename T, int D>
__device__ __noinline__ void put_q(const Kv8AttnArgs &a, const Problem &w, uint32_t q_tile, float *row_mul) {
  constexpr bool kSplit = sizeof(T) == 4;
  using P = PromptShape<D, kSplit>;
  constexpr uint32_t kLanes = D / 8, kPass = 32 / kLanes;  // lanes of a row, rows of a warp's pass
  constexpr uint32_t kStep = P::kThreads / 32 * kPass;
  constexpr int kVec = 16 / (int)sizeof(T), kBatch = kSplit ? 3 : 5;  // rows on their way
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, li = lane % kLanes;
  uint32_t i = warp * kPass + lane / kLanes;  // this lane's row; its token and q head
  uint32_t t = (w.row0 + i) / a.gqa, g = w.row0 + i - t * a.gqa;
  const uint32_t dt = kStep / a.gqa, dg = kStep - dt * a.gqa;
#pragma unroll 1
  for (uint32_t i0 = warp * kPass; i0 < kRows; i0 += kBatch * kStep) {
    uint4 raw[kBatch][8 / kVec];
#pragma unroll
    for (int n = 0; n < kBatch; ++n) {
      const T *src = static_cast<const T *>(a.q) + (size_t)(w.r0 + t) * a.q_ld + (w.head * a.gqa + g) * D + 8 * li;
#pragma unroll
      for (int k = 0; k < 8 / kVec; ++k) {
        raw[n][k] = make_uint4(0, 0, 0, 0);
        if (i + n * kStep < w.rows) raw[n][k] = *reinterpret_cast<const uint4 *>(src + kVec * k);
      }
      t += dt;
      g += dg;
      if (g >= a.gqa) {
        g -= a.gqa;
        ++t;
      }
    }
#pragma unroll
    for (int n = 0; n < kBatch; ++n, i += kStep) {
      if (i0 + n * kStep >= kRows) break;
      float x[8], m = 0.0f;
#pragma unroll
      for (int k = 0; k < 8 / kVec; ++k) {
        float v[kVec];
        load_vec<T, kVec>(reinterpret_cast<const T *>(&raw[n][k]), v);
#pragma unroll
        for (int j = 0; j < kVec; ++j) x[kVec * k + j] = v[j];
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) m = fmaxf(m, fabsf(x[k]));
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      int e = (int)(__float_as_uint(m) >> 23) - 127;
      if (m == 0.0f || e == 128) e = 0;  // nothing to scale; an infinity stays one
      e = min(max(e, -126), 126);
      const float inv = a.scale < 0.0f ? -exp2_int(-e) : exp2_int(-e);
      if (li == 0) row_mul[i] = fabsf(a.scale) * kLog2e * exp2_int(e);
      uint32_t hi[4], low[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float v0 = x[2 * k] * inv, v1 = x[2 * k + 1] * inv;
        hi[k] = pack_f16(v0, v1);
        if constexpr (kSplit) low[k] = pack_f16_rest(v0, v1, hi[k]);
      }
      const uint32_t dst = q_tile + li / 8 * (kRows * 128) + i * 128 + (((li % 8) ^ (i & 7)) << 4);
      st_shared16(dst, hi);
      if constexpr (kSplit) st_shared16(dst + P::kQTerm, low);
    }
  }
  fence_proxy_async();  // generic-proxy stores -> the tensor core's reads
}

// What a part's CTA leaves for the merge: where the problem's parts are, and which it is.
struct PromptPart {
  uint32_t parts, part, slot0, c0;  // parts 0: there is none
  uint32_t r0, row0, rows, head;
};
// The workspace: {m, l} of [2 CTAs][128 rows], [2 CTAs][128 rows][D], [2 CTAs] of the above.
SX_DEV float *part_values(const Kv8AttnArgs &a, uint32_t ctas) { return a.part + (size_t)2 * ctas * kRows * 2; }
template <int D>
SX_DEV PromptPart *part_list(const Kv8AttnArgs &a, uint32_t ctas) {
  return reinterpret_cast<PromptPart *>(part_values(a, ctas) + (size_t)2 * ctas * kRows * D);
}

// The parts of cut problems, by a second kernel (the last CTA to arrive alone would read them at 17 bytes
// a cycle, 15 us for 9 parts of 40 rows of 256): CTA j takes part j's share of its problem's rows.
// Threads: D / 4 columns x kSubs.  A sub takes a row, or with many parts every kSubs-th part of one, and
// they meet in shared memory.
constexpr int kMergeThreads = 512;
constexpr uint32_t kShareParts = 16;

struct Merged {
  float m, l;
  float4 o;
  SX_DEV void add(float mk, float lk, float4 v) {
    const float top = fmaxf(m, mk);  // a part that saw nothing has -inf and weight 0
    const float f = m == -INFINITY ? 0.0f : ex2(m - top), g = mk == -INFINITY ? 0.0f : ex2(mk - top);
    m = top;
    l = fmaf(l, f, lk * g);
    o = make_float4(fmaf(o.x, f, v.x * g), fmaf(o.y, f, v.y * g), fmaf(o.z, f, v.z * g), fmaf(o.w, f, v.w * g));
  }
};

template <typename T, int D>
__global__ void __launch_bounds__(kMergeThreads) kv8_prompt_merge_kernel(const __grid_constant__ Kv8AttnArgs a, uint32_t ctas) {
  constexpr uint32_t kItems = D / 4, kSubs = kMergeThreads / kItems, kBatch = 4;
  __shared__ Merged red[kMergeThreads];
  pdl_launch_dependents();
  pdl_wait();
  const PromptPart w = part_list<D>(a, ctas)[blockIdx.x];
  if (w.parts == 0) return;
  // (what another call's parts left here, had one run at the same time, ends as an error)
  if (w.part >= w.parts || w.c0 + w.parts > ctas || w.slot0 >= 2 * ctas || w.rows - 1 >= kRows || w.head >= a.c.num_kv ||
      w.r0 >= a.tokens || (w.row0 + w.rows - 1) / a.gqa >= a.tokens - w.r0) {
    if (threadIdx.x == 0) raise_error(a.err, kDevBadParams);
    return;
  }
  const float2 *const part_ml = reinterpret_cast<const float2 *>(a.part);
  const float *const part_o = part_values(a, ctas);
  const uint32_t item = threadIdx.x % kItems, sub = threadIdx.x / kItems;
  const bool share = w.parts > kShareParts;
  const uint32_t i0 = w.rows * w.part / w.parts, i1 = w.rows * (w.part + 1) / w.parts;
  const uint32_t first = share ? sub : 0, step = share ? kSubs : 1, rows = share ? 1 : kSubs;
#pragma unroll 1
  for (uint32_t ii = i0; ii < i1; ii += rows) {
    const uint32_t i = share ? ii : ii + sub;
    Merged sum{-INFINITY, 0.0f, make_float4(0.0f, 0.0f, 0.0f, 0.0f)};
#pragma unroll 1
    for (uint32_t k0 = first; k0 < w.parts && i < i1; k0 += kBatch * step) {
      float4 v[kBatch];
      float2 ml[kBatch];
#pragma unroll
      for (uint32_t u = 0; u < kBatch; ++u) {
        const uint32_t k = min(k0 + u * step, w.parts - 1);
        const size_t at = (size_t)(k == 0 ? w.slot0 : 2 * (w.c0 + k)) * kRows + i;
        v[u] = *reinterpret_cast<const float4 *>(part_o + at * D + 4 * item);
        ml[u] = part_ml[at];
      }
#pragma unroll
      for (uint32_t u = 0; u < kBatch; ++u)
        if (k0 + u * step < w.parts) sum.add(ml[u].x, ml[u].y, v[u]);
    }
    if (share) {
      __syncthreads();  // the row before has been added up
      red[threadIdx.x] = sum;
      __syncthreads();
      if (sub == 0)
#pragma unroll 1
        for (uint32_t u = 1; u < kSubs; ++u) {
          const Merged x = red[u * kItems + item];
          sum.add(x.m, x.l, x.o);
        }
    }
    if (i < i1 && (!share || sub == 0)) {
      const float inv = sum.l == 0.0f ? 0.0f : 1.0f / sum.l;
      const float y[4] = {sum.o.x * inv, sum.o.y * inv, sum.o.z * inv, sum.o.w * inv};
      const uint32_t pr = w.row0 + i;
      store_vec<T, 4>(static_cast<T *>(a.out) + (size_t)(w.r0 + pr / a.gqa) * a.out_ld +
                          (size_t)(w.head * a.gqa + pr % a.gqa) * D + 4 * item, y);
    }
  }
}

// One product by one thread of the warp that calls it: STEPS of 16 along K, A from shared memory
// (a_tile) or tensor memory (a_col); 32 bytes of a swizzled row per step, a panel of 64 elements every
// four.  The whole warp comes here so that descriptors are the same in all lanes.
template <int STEPS>
SX_DEV void issue_ss(uint32_t d, uint32_t a_tile, uint32_t a_panel, uint32_t b_tile, uint32_t b_panel, uint32_t idesc,
                     bool add) {
  const uint64_t x = umma_desc_sw128(a_tile), y = umma_desc_sw128(b_tile);
#pragma unroll
  for (int k = 0; k < STEPS; ++k)
    umma_f16(d, x + k / 4 * (a_panel >> 4) + 2 * (k % 4), y + k / 4 * (b_panel >> 4) + 2 * (k % 4), idesc, add || k > 0);
}
template <int STEPS>
SX_DEV void issue_ts(uint32_t d, uint32_t a_col, uint32_t b_tile, uint32_t b_panel, uint32_t idesc, bool add) {
  const uint64_t y = umma_desc_sw128(b_tile);
#pragma unroll
  for (int k = 0; k < STEPS; ++k)
    umma_f16_ts(d, a_col + 8 * k, y + k / 4 * (b_panel >> 4) + 2 * (k % 4), idesc, add || k > 0);
}

// One role's way through the CTA's problems.
template <typename T, int D, Role ROLE>
SX_DEV void prompt_role(const Kv8AttnArgs &a, uint8_t *smem_raw, PromptShared<PromptShape<D, sizeof(T) == 4>::kTokens, PromptShape<D, sizeof(T) == 4>::kWiden> &sh) {
  constexpr bool kSplit = sizeof(T) == 4;
  using P = PromptShape<D, kSplit>;
  constexpr int kTokens = P::kTokens, kS = P::kS, kWiden = P::kWiden, kTerms = P::kTerms, kStages = P::kStages;
  constexpr int kTileBlocks = kTokens / kKv8Block;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t q_tile = (smem_u32(smem_raw) + 1023) & ~1023u;  // [terms][D / 64][128 rows][128 B]
  // K and V tiles: [stages][D / 64][tokens][128 B], [stages][tokens / 64][D][128 B]
  auto k_tile = [&](uint32_t t) { return q_tile + kTerms * P::kQTerm + t % kStages * P::kTile; };
  auto v_tile = [&](uint32_t t) { return q_tile + kTerms * P::kQTerm + (kStages + t % kStages) * P::kTile; };
  const PromptBars bars(smem_u32(sh.bars));
  const uint32_t tmem = sh.tmem_slot;
  auto wait = [&](uint32_t b, uint32_t parity) {
    if (!mbar_try_wait(b, parity & 1)) wait_longer(b, parity, &sh.abort_flag, a.err);
  };
  Schedule plan;
  if constexpr (ROLE == kProducts) {
    PromptPart *const list = part_list<D>(a, gridDim.x) + 2 * blockIdx.x;
    if (lane < 2) list[lane].parts = 0;
    __syncwarp();
    plan.start(a, kTokens);
    plan.next(a, kTileBlocks, sh.problem[0]);
  }
  __syncthreads();

  uint32_t tiles = 0;  // tiles done, over all problems: every barrier's phase follows from it
#pragma unroll 1
  for (uint32_t np = 0;; ++np) {
    const Problem &pr = sh.problem[np & 1];
    if (!pr.more) break;
    const uint32_t t0 = pr.t0, t1 = pr.t1, n_tiles = t1 - t0, first = pr.first;
    // tiles whose keys some row does not see
    const uint32_t all_lo = pr.all_lo, all_hi = pr.all_hi;
    auto is_mixed = [&](uint32_t t) {
      const uint32_t key0 = (first + t * kTileBlocks) * kKv8Block;
      return key0 < all_lo || key0 + kTokens - 1 > all_hi;
    };
    if constexpr (ROLE != kWidenKv) {  // (the warps that widen ask for their first tiles before)
      put_q<T, D>(a, pr, q_tile, sh.row_mul);
      __syncthreads();
    }

    if constexpr (ROLE == kSoftmax) {
      // ================================================================ softmax: thread = half a row
      const uint32_t i = threadIdx.x % kRows, half = threadIdx.x / kRows, rows = pr.rows;
      const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16, pair_bar = 2 + (warp & 3);
      const float mul = sh.row_mul[i];
      const uint32_t pos = pr.pos0 + (pr.row0 + min(i, rows - 1)) / a.gqa;
      const uint32_t see_lo = a.window && pos >= a.window ? pos - a.window + 1 : 0, see_hi = pos + 1;
      float ref = -INFINITY, l = 0.0f;
      auto fold_at = [&] { return part_values(a, gridDim.x) + ((size_t)pr.slot * D + half * (D / 2)) * kRows + i; };
      const uint32_t fold_ref = smem_u32(&sh.fold_ref[half][i]);
      // bit = token of this thread's half of a tile: the keys that its row sees, and that are there
      auto visible = [&](uint32_t t) {
        const uint32_t k0 = (first + t * kTileBlocks) * kKv8Block + 32 * half;
        const uint32_t lo = see_lo > k0 ? see_lo - k0 : 0, hi = see_hi > k0 ? see_hi - k0 : 0;
        uint32_t vis = lo < 32 && hi > lo ? (hi < 32 ? (1u << hi) - 1 : ~0u) & (~0u << lo) : 0;
        const float4 *const block = sh.facts[half] + 2 * (t - t0) % 64;
        if (block[0].w == 0.0f) vis &= 0xFFFF0000u;
        if (block[1].w == 0.0f) vis &= 0x0000FFFFu;
        return vis;
      };
#pragma unroll 1
      for (uint32_t t = t0; t < t1; ++t) {
        const uint32_t tile = tiles + (t - t0), s_col = tmem + lanes + tile % kS * kTokens;
        const bool mixed = is_mixed(t);
        wait(bars.s_done(tile), tile / 2);
        if (mixed) wait(bars.v_full(tile), tile / 2);  // for the mask of its NaNs
        __syncwarp();
        tc_fence_after();
        uint32_t s[32];
        tmem_ld32(s_col + 32 * half, s);
        // block 2 half holds columns k with k / 4 even, block 2 half + 1 the others
        const float4 *const block = sh.facts[half] + 2 * (t - t0) % 64;
        const uint32_t odd = sh.odd_records[tile & 1];
        const float km[2] = {fmaxf(block[0].x * mul, kMinScale), fmaxf(block[1].x * mul, kMinScale)};
        tmem_wait_ld(s);
        if (mixed || (odd & kGone)) {  // some row does not see all of the tile, or a block is not there
          const uint32_t vis = visible(t);
          if (mixed && (sh.nan_mask[tile & 1][half] & vis)) l = NAN;
#pragma unroll
          for (int k = 0; k < 32; ++k)
            if (!(vis & key_bit(k))) s[k] = 0xFF800000u;
        }
        // -- the largest x + log2(v scale)
        float m[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int k = 0; k < 32; k += 4)
          m[(k >> 2) & 1] = fmaxf(fmaxf(m[(k >> 2) & 1], fmaxf(__uint_as_float(s[k]), __uint_as_float(s[k + 1]))),
                                  fmaxf(__uint_as_float(s[k + 2]), __uint_as_float(s[k + 3])));
        float top = fmaxf(fmaf(m[0], km[0], block[0].y), fmaf(m[1], km[1], block[1].y));
        // -- one that outgrew the reference: rescale the row.  The vote also says that both halves of
        // the row have been read, which P overwrites.
        auto grows = [&] { return top > ref + kSlack || (ref == -INFINITY && top > ref); };
        if (pair_any(pair_bar, grows() || (odd & kApart))) {
          sh.row_top[half][i] = top;
          pair_any(pair_bar, false);
          top = fmaxf(top, sh.row_top[half ^ 1][i]);
          const bool grow = grows();
          const float f = !grow ? 1.0f : ref == -INFINITY ? 0.0f : ex2(ref - top);
          if (grow) ref = top;
          l *= f;
          if (t > t0) {
            wait(bars.pv_done(tile - 1), (tile - 1) / 2);
            __syncwarp();
            tc_fence_after();
            rescale_row(tmem + lanes + P::kO + half * (D / 2), D / 2, f);
            tmem_wait_st();
          }
          if (odd & kApart) {
            wait(bars.v_full(tile), tile / 2);
            __syncwarp();
            l += add_far<D>(tmem + lanes + P::kO, v_tile(tile), s_col + 32 * half, visible(t), smem_u32(block), mul, ref,
                            sh.far_below[tile & 1], t == t0);
            tmem_ld32(s_col + 32 * half, s);  // (again, rather than kept over the call)
            tmem_wait_ld(s);
            pair_any(pair_bar, false);  // (both halves have, before either's P)
          }
        }
        const float shift = ref == -INFINITY ? 0.0f : ref - kOffset;
        const float off[2] = {block[0].y - shift, block[1].y - shift};
        float sum[2] = {0.0f, 0.0f};
        uint32_t hi[16];
#pragma unroll
        for (int k = 0; k < 32; k += 2) {
          const int h = (k >> 2) & 1;
          const float p0 = ex2(fmaf(__uint_as_float(s[k]), km[h], off[h]));
          const float p1 = ex2(fmaf(__uint_as_float(s[k + 1]), km[h], off[h]));
          sum[h] += p0 + p1;
          hi[k / 2] = pack_f16(p0, p1);
          if constexpr (kSplit) s[k / 2] = pack_f16_rest(p0, p1, hi[k / 2]);
        }
        tmem_st16(s_col + 16 * half, hi);  // P over S
        if constexpr (kSplit) {
#pragma unroll
          for (int k = 0; k < 16; ++k) hi[k] = s[k];
          tmem_st16(tmem + lanes + P::kLow + tile % kS * (kTokens / 2) + 16 * half, hi);
        }
        l = fmaf(sum[0], block[0].z, fmaf(sum[1], block[1].z, l));
        tmem_wait_st();
        if constexpr (kSplit) {
          if (t != t0 && (t - t0) % P::kFold == 0) {  // O of the tiles before; this tile's begins anew
            wait(bars.pv_done(tile - 1), (tile - 1) / 2);
            __syncwarp();
            tc_fence_after();
            if (32u * (warp & 3) < rows)
              fold_row<P::kTotal != 0>(tmem + lanes + P::kO + half * (D / 2), tmem + lanes + P::kTotal + half * (D / 2), D / 2, fold_at(),
                                       fold_ref, ref, t - t0 == P::kFold);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bars.p_full(tile));
      }
      // ---- the row's output, or its part: half of the columns a thread
      sh.row_sum[half][i] = l;
      pair_any(pair_bar, false);
      l = sh.row_sum[0][i] + sh.row_sum[1][i];
      wait(bars.pv_done(tiles + n_tiles - 1), (tiles + n_tiles - 1) / 2);
      __syncwarp();
      tc_fence_after();
      if (kSplit && n_tiles > P::kFold) {
        if (32u * (warp & 3) < rows)
          unfold_row<P::kTotal != 0>(tmem + lanes + P::kO + half * (D / 2), tmem + lanes + P::kTotal + half * (D / 2), D / 2, fold_at(),
                                     fold_ref, ref);
        asm volatile("bar.sync 6, %0;\n" ::"n"(kSoft * 32) : "memory");  // parts go where the sums are
      }
      const bool whole = pr.parts == 1;
      const size_t at = (size_t)pr.slot * kRows + i;
      float *const po = part_values(a, gridDim.x) + at * D;
      T *const out = static_cast<T *>(a.out) + pr.row(a, i) * a.out_ld + pr.col(a, i);
      const float inv = whole ? (l == 0.0f ? 0.0f : 1.0f / l) : 1.0f;
      // Whole rows with one CTA an SM go 64 bytes at a time through shared memory (over the K tiles, which
      // have been read), so that four lanes store them together: a lane's own row is a line of its own
      // for every 16 bytes.  (Prompts of 2048 with head size 256 128 us for 133; with two CTAs the
      // registers cost the loop more, 547 us for 534 in the long prompts.)
      constexpr bool kTogether = P::kCtas == 1;
      constexpr uint32_t kPiece = 64 / sizeof(T);
      T *dst[4];  // the rows that this lane stores then
      if constexpr (kTogether) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          dst[k] = reinterpret_cast<T *>(__shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(out), 8 * k + lane / 4)) +
                   lane % 4 * (kPiece / 4);
      }
      const uint32_t stage = k_tile(0) + warp * (32 * 80);
      if (!whole && half == 0 && i < rows) reinterpret_cast<float2 *>(a.part)[at] = make_float2(ref, l);
#pragma unroll 1
      for (int d = half * (D / 2); d < (int)(half + 1) * (D / 2) && 32u * (warp & 3) < rows; d += 32) {
        uint32_t o[32];
        tmem_ld32(tmem + lanes + P::kO + d, o);
        tmem_wait_ld(o);
        // element 4 g + i of the piece is column 8 i + f(g), f(g) = g / 2 + 4 (g % 2)
        float y[32];
#pragma unroll
        for (int k = 0; k < 32; ++k)
          y[k] = __uint_as_float(o[8 * (k & 3) + ((k >> 2) >> 1) + 4 * ((k >> 2) & 1)]) * inv;
        if (kTogether && whole) {
#pragma unroll
          for (uint32_t h = 0; h < 32; h += kPiece) {
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) {
              uint32_t w[4];
#pragma unroll
              for (uint32_t e = 0; e < 4; ++e) {
                if constexpr (kSplit) {
                  w[e] = __float_as_uint(y[h + 4 * k + e]);
                } else {
                  const __nv_bfloat162 b = __floats2bfloat162_rn(y[8 * k + 2 * e], y[8 * k + 2 * e + 1]);
                  w[e] = *reinterpret_cast<const uint32_t *>(&b);
                }
              }
              st_shared16(stage + lane * 80 + 16 * k, w);
            }
            __syncwarp();
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) {
              uint32_t w[4];
              ld_shared16(stage + (8 * k + lane / 4) * 80 + 16 * (lane % 4), w);
              if (32 * (warp & 3) + 8 * k + lane / 4 < rows)
                *reinterpret_cast<uint4 *>(dst[k] + d + h) = make_uint4(w[0], w[1], w[2], w[3]);
            }
            __syncwarp();
          }
        } else if (i < rows) {
          if (whole) {
            constexpr int kVec = 16 / (int)sizeof(T);
#pragma unroll
            for (int k = 0; k < 32; k += kVec) {
              float v[kVec];
#pragma unroll
              for (int j = 0; j < kVec; ++j) v[j] = y[k + j];
              store_vec<T, kVec>(out + d + k, v);
            }
          } else {
#pragma unroll
            for (int k = 0; k < 32; k += 4)
              *reinterpret_cast<float4 *>(po + d + k) = make_float4(y[k], y[k + 1], y[k + 2], y[k + 3]);
          }
        }
        __syncwarp();
      }
      tc_fence_before();
    } else if constexpr (ROLE == kWidenKv) {
      // ================================================================ widen K and V
      constexpr int kPairs = kTokens / 32, kShare = kWiden / kPairs;  // warps of a pair of blocks
      constexpr int kMine = D / 32 / kShare;                          // pieces of a warp
      const uint32_t g = lane >> 2, c = lane & 3;
      const uint32_t ww = warp - kSoft, pair = ww % kPairs, p0 = ww / kPairs * kMine;
      // The warp's blocks of 16 tiles, one a lane, from the problem's tile t0 + `from` on.
      uint32_t *const record = sh.record[ww];
      auto look_up = [&](uint32_t from) {
        const uint32_t n = from + lane / 2, s = (t0 + n) * kTileBlocks + 2 * pair + lane % 2;
        const uint32_t at = 2 * n % 64 + lane % 2;
        uint32_t rec = kNoRecord;
        if (t0 + n < t1 && s < pr.blocks) {
          const PageDiv div(a.c.page_tokens);
          const uint32_t x = first + s, in = div.page(x), page = a.c.table[(size_t)pr.seq * a.c.max_pages + in];
          if (page < a.c.num_pages)
            rec = (page * a.c.num_kv + pr.head) * div.per + (x - in * div.per);
          else
            raise_error(a.err, kDevBadSlot);
        }
        __syncwarp();
        record[at] = rec;
        if (p0 == 0) {
          float2 f = make_float2(0.0f, 0.0f);
          if (rec != kNoRecord) f = *reinterpret_cast<const float2 *>(a.c.scale + 2 * (size_t)rec);
          const int e = rec != kNoRecord ? kv8_scale_exponent(f.y) : kKv8MinExp;
          sh.facts[pair][at] = make_float4(f.x, (float)e, exp2_int(-e), rec != kNoRecord ? 1.0f : 0.0f);
        }
        __syncwarp();
      };
      // K: lanes with odd g take the pieces of a pair in the other order, so that a store's eight
      // lanes meet all banks.  A piece's store goes to the lane's offset with bits 5 and 6 turned by
      // which of its tokens, block and piece it is.
      const uint32_t swap = kMine >= 2 ? g & 1 : 0;
      const uint32_t k_lane = p0 / 2 * (kTokens * 128) + (32 * pair + 8 * (g / 2) + (g & 1)) * 128 +
                              ((kMine >= 2 ? swap : p0 & 1) << 6) + ((c ^ (g & 1)) << 4);
      const uint32_t fg = (g >> 1) | ((g & 1) << 2);
      const uint32_t v_lane = pair / 2 * (D * 128) + (32 * p0 + fg) * 128 + ((((pair & 1) * 4 + c) ^ fg) << 4);
      // A tile ahead: K in registers, V in shared memory (each lane reads what it had fetched).
      uint4 raw_k[2][kMine];
      const uint32_t v_stage = q_tile + kTerms * P::kQTerm + 2 * kStages * P::kTile + ww * (2 * kMine * 512) + 16 * lane;
      const uint8_t *const data = static_cast<const uint8_t *>(a.c.data), *const no_block = reinterpret_cast<const uint8_t *>(g_no_block);
      const uint32_t k_off = 512 * p0 + 16 * lane + (swap ? 512 : 0), v_off = 16 * D + 512 * p0 + 16 * lane;
      const int k_turn = swap ? -512 : 512;
      auto records = [&](uint32_t n) { return *reinterpret_cast<const uint2 *>(record + 2 * n % 64); };
      auto fetch_k = [&](uint32_t rec, int h) {
        const uint8_t *src = (rec != kNoRecord ? data + (size_t)rec * (32 * D) : no_block) + k_off;
#pragma unroll
        for (int p = 0; p < kMine; ++p) raw_k[h][p] = *reinterpret_cast<const uint4 *>(src + p / 2 * 1024 + (p & 1) * k_turn);
      };
      auto fetch_v = [&](uint32_t rec, int h) {
        const uint8_t *src = (rec != kNoRecord ? data + (size_t)rec * (32 * D) : no_block) + v_off;
#pragma unroll
        for (int p = 0; p < kMine; ++p) cp_async16(v_stage + (h * kMine + p) * 512, src + 512 * p);
      };
      look_up(0);
      {
        const uint2 rec = records(0);
        fetch_k(rec.x, 0);
        fetch_k(rec.y, 1);
        fetch_v(rec.x, 0);
        fetch_v(rec.y, 1);
        cp_async_commit();
      }
      put_q<T, D>(a, pr, q_tile, sh.row_mul);
      __syncthreads();
      // K of a tile, then V of the one before: K of the next tile waits for no softmax.
#pragma unroll 1
      for (uint32_t n = 0; n <= n_tiles; ++n) {
        if (n % 16 == 8) look_up(n + 8);
        if (n < n_tiles) {
        const uint32_t tile = tiles + n, k_at = k_tile(tile);
        if (tile >= kStages) wait(bars.s_done(tile - kStages), (tile - kStages) / 2);  // K has been read
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int p = 0; p < kMine; ++p) {
            const uint32_t at = k_at + p / 2 * (kTokens * 128) + h * 512 + (k_lane ^ (((p & 1) ^ h) << 6));
            const uint32_t at8 = k_at + p / 2 * (kTokens * 128) + h * 512 + 256 + (k_lane ^ (((p & 1) ^ h) << 6) ^ 32);
            uint32_t x[4];
            e4m3x4_f16(raw_k[h][p].x, x[0], x[1]);
            e4m3x4_f16(raw_k[h][p].y, x[2], x[3]);
            st_shared16(at, x);
            e4m3x4_f16(raw_k[h][p].z, x[0], x[1]);
            e4m3x4_f16(raw_k[h][p].w, x[2], x[3]);
            st_shared16(at8, x);
          }
        }
        fence_proxy_async();  // generic-proxy stores -> the tensor core's reads
        __syncwarp();
        if (lane == 0) mbar_arrive(bars.k_full(tile));
        const uint2 rec = records(n + 1);
        fetch_k(rec.x, 0);
        fetch_k(rec.y, 1);
        }
        if (n > 0) {
        const uint32_t tile = tiles + n - 1;
        if (tile >= kStages) wait(bars.pv_done(tile - kStages), (tile - kStages) / 2);  // V has been read
        const bool mixed = is_mixed(t0 + n - 1);
        uint32_t nan_bits = 0;
        if (mixed) {
          if (ww == 0 && lane < kPairs) sh.nan_mask[tile & 1][lane] = 0;
          asm volatile("bar.sync 1, %0;\n" ::"n"(kWiden * 32) : "memory");
        }
        cp_async_wait<0>();
        const uint32_t v_at = v_tile(tile) + v_lane;
#pragma unroll 1
        for (int p = 0; p < kMine; ++p) {
          uint32_t w[2][4];
          ld_shared16(v_stage + p * 512, w[0]);
          ld_shared16(v_stage + (kMine + p) * 512, w[1]);
          if (mixed) {
            // A NaN would reach rows that do not see its token through 0 x NaN: it is taken out, and
            // its token marked for the rows that do.
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              uint32_t &x = w[k / 4][k % 4];
              const uint32_t m = (((x & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) >> 7;
              x &= ~(m * 0xFFu);
              // bytes are tokens 2 c, 2 c + 1, 2 c + 8, 2 c + 9 of a block
              nan_bits |= ((m & 1u) | ((m >> 7) & 2u) | ((m >> 8) & 0x100u) | ((m >> 15) & 0x200u)) << (2 * c + k / 4 * 16);
            }
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {  // element 4 g + k: row 8 k + f(g) of the piece
            uint32_t x[4];
            e4m3x4_f16(w[0][k], x[0], x[1]);
            e4m3x4_f16(w[1][k], x[2], x[3]);
            st_shared16(v_at + p * 4096 + k * 1024, x);
          }
        }
        if (nan_bits) atomicOr(&sh.nan_mask[tile & 1][pair], nan_bits);
        fence_proxy_async();  // generic-proxy stores -> the tensor core's reads
        __syncwarp();
        if (lane == 0) mbar_arrive(bars.v_full(tile));
        if (n < n_tiles) {
          const uint2 rec = records(n);
          fetch_v(rec.x, 0);
          fetch_v(rec.y, 1);
          cp_async_commit();
        }
        }
      }
    } else {
      // ================================================================ the products
      // Records whose scale is far below the problem's largest so far are added apart: the softmax's
      // reference may stand for a value of that scale which is masked or has no weight, and nothing of
      // their P would be left.  (The least scale is that of zeros, or nearly: those may go.)
      int most = -128;
      auto product_s = [&](uint32_t tile) {
        wait(bars.k_full(tile), tile / 2);
        __syncwarp();
        {
          const float4 f = sh.facts[lane / 2 % 2][2 * (tile - tiles) % 64 + lane % 2];
          const bool gone = __any_sync(0xffffffffu, f.w == 0.0f);
          most = max(most, __reduce_max_sync(0xffffffffu, f.w != 0.0f ? (int)f.y : -128));
          const float below = (float)most - P::kFar;
          const bool apart = __any_sync(0xffffffffu, f.y < below && f.y > (float)kKv8MinExp);
          if (lane == 0) {
            sh.odd_records[tile & 1] = (gone ? kGone : 0) | (apart ? kApart : 0);
            sh.far_below[tile & 1] = below;
          }
          __syncwarp();
        }
        tc_fence_after();
        if (elect_one()) {
          mbar_arrive(bars.s_done(tile));  // (passes on what the widening warps wrote for the softmax)
#pragma unroll
          for (int w = kTerms - 1; w >= 0; --w)  // (the small terms first: what is cut off goes by the sum so far)
            issue_ss<D / 16>(tmem + tile % kS * kTokens, q_tile + w * P::kQTerm, kRows * 128, k_tile(tile), kTokens * 128,
                             umma_idesc_f16(kRows, kTokens), w < kTerms - 1);
          umma_commit(bars.s_done(tile));
        }
        __syncwarp();
      };
      product_s(tiles);
      const bool begun = (sh.odd_records[tiles & 1] & kApart) != 0;
      if (pr.parts > 1 && lane == 0)
        part_list<D>(a, gridDim.x)[pr.slot] =
            PromptPart{pr.parts, blockIdx.x - pr.c0, pr.slot0, pr.c0, pr.r0, pr.row0, pr.rows, pr.head};
      plan.next(a, kTileBlocks, sh.problem[(np + 1) & 1]);  // (read by all after the barrier below)
#pragma unroll 1
      for (uint32_t j = 0; j < n_tiles; ++j) {
        const uint32_t tile = tiles + j;
        if (j + 1 < n_tiles) product_s(tile + 1);  // beside this tile's softmax
        wait(bars.v_full(tile), tile / 2);
        wait(bars.p_full(tile), tile / 2);
        __syncwarp();
        tc_fence_after();
        // a sum of tiles begins with zeros, but the first where add_far has begun it
        const bool add = kSplit && j % P::kFold == 0 && j > 0 ? false : j > 0 || begun;
        if (elect_one()) {
#pragma unroll
          for (int w = 0; w < kTerms; ++w)
            issue_ts<kTokens / 16>(tmem + P::kO, tmem + (w ? P::kLow + tile % kS * (kTokens / 2) : tile % kS * kTokens),
                                   v_tile(tile), D * 128, umma_idesc_f16(kRows, D), add || w > 0);
          umma_commit(bars.pv_done(tile));
        }
        __syncwarp();
      }
    }
    tiles += n_tiles;
    __syncthreads();  // Q, the tiles and O are free, and the next problem is there
  }
}

template <typename T, int D>
__global__ void __launch_bounds__((PromptShape<D, sizeof(T) == 4>::kThreads), (PromptShape<D, sizeof(T) == 4>::kCtas))
    kv8_prompt_kernel(const __grid_constant__ Kv8AttnArgs a) {
  using P = PromptShape<D, sizeof(T) == 4>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ PromptShared<P::kTokens, P::kWiden> sh;
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    const PromptBars bars(smem_u32(sh.bars));
    for (int i = 0; i < 2; ++i) {
      mbar_init(bars.k_full(i), P::kWiden);
      mbar_init(bars.v_full(i), P::kWiden);
      mbar_init(bars.p_full(i), kSoft);
      mbar_init(bars.s_done(i), 2);
      mbar_init(bars.pv_done(i), 1);
    }
    sh.abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0) {
    tmem_alloc(smem_u32(&sh.tmem_slot), P::kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_launch_dependents();
  pdl_wait();
  if (warp < kSoft)
    prompt_role<T, D, kSoftmax>(a, smem_raw, sh);
  else if (warp < kSoft + P::kWiden)
    prompt_role<T, D, kWidenKv>(a, smem_raw, sh);
  else
    prompt_role<T, D, kProducts>(a, smem_raw, sh);
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(sh.tmem_slot, P::kCols);
  }
}

using PromptKernel = void (*)(const Kv8AttnArgs);
using PromptMerge = void (*)(const Kv8AttnArgs, uint32_t);
struct PromptVariant {
  PromptKernel fn;
  PromptMerge merge;
  uint32_t smem, ctas, threads;
};
template <typename T, int D>
PromptVariant prompt_variant() {
  using P = PromptShape<D, sizeof(T) == 4>;
  return {kv8_prompt_kernel<T, D>, kv8_prompt_merge_kernel<T, D>, (uint32_t)P::kSmem, (uint32_t)P::kCtas, (uint32_t)P::kThreads};
}
PromptVariant prompt_variant(sx_dtype t, uint32_t d) {
  if (t == SX_F32)
    return d == 64 ? prompt_variant<float, 64>() : d == 128 ? prompt_variant<float, 128>() : prompt_variant<float, 256>();
  return d == 64 ? prompt_variant<__nv_bfloat16, 64>() : d == 128 ? prompt_variant<__nv_bfloat16, 128>()
       : prompt_variant<__nv_bfloat16, 256>();
}

}  // namespace

cudaError_t prepare_kv8_prompt() {
  for (uint32_t d : {64u, 128u, 256u})
    for (sx_dtype t : {SX_F32, SX_BF16}) {
      const PromptVariant v = prompt_variant(t, d);
      const cudaError_t e = cudaFuncSetAttribute(v.fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)v.smem);
      if (e != cudaSuccess) return e;
    }
  return cudaSuccess;
}

// Two parts per CTA of 128 rows: {m, l}, and 128 (two CTAs per SM) or 256 output values a row.
size_t kv8_prompt_part_bytes(int num_sms) {
  return (size_t)2 * num_sms * (kRows * (2 * 2 + 256) * sizeof(float) + 2 * sizeof(PromptPart));
}

cudaError_t launch_kv8_prompt(Kv8AttnArgs a, sx_dtype t, int num_sms, cudaStream_t s) {
  const PromptVariant v = prompt_variant(t, a.c.head_dim);
  a.min_run = 6;  // tiles: shorter runs cost more to merge than they save
  const uint32_t ctas = num_sms * v.ctas;
  const cudaError_t e = launch_chained(v.fn, dim3(ctas), dim3(v.threads), v.smem, s, 1, a);
  if (e != cudaSuccess) return e;
  return launch_chained(v.merge, dim3(2 * ctas), dim3(kMergeThreads), 0, s, 1, a, ctas);
}

}  // namespace sx
