// kv_attention.cuh -- attention of few query rows over many keys, split along
// the keys: over the quantised paged cache (4 or 8 bits) and over dense 16-bit
// keys and values.  Instantiated by kv_attention.cu (cache, bf16),
// kv_attention_f16.cu (cache, f16) and kv_attention_dense.cu.
//
// HBM-bound: every key and value byte is read once.  A warp works on blocks
// of 16 tokens of its own: cp.async copies them into its ring of stages in
// shared memory, several blocks ahead, and mma.sync (m16n8k16, f32
// accumulators) takes them from registers.  No barrier but the warp's own
// until the end.  The tensor cores only have to keep up with memory, not to
// approach their peak, and operands in registers let the codes be unpacked on
// the way and the softmax work on the accumulators where they are; tcgen05
// would want unpacked operands back in shared memory.
//
//   S^T [tokens, rows] = K Q^T: A = 16 tokens of codes, B = 8 query rows;
//   O^T [d, rows]     += V^T P^T: A = 16 elements x 16 tokens of codes.
// The rows (the query heads that share a key head, times the queries) are the
// narrow n = 8 side, so one query head wastes idle tensor lanes, not bytes.
// S^T's accumulator layout becomes P^T's operand layout by one movmatrix per
// 8 x 8 block.
//
// Codes are used as they lie: a nibble or byte masked out of its word is the
// f16 denormal code * 2^-24 (times 16 for a high nibble), which the tensor
// core multiplies exactly; the factors 2^24 and 1/16 go into the f32 scores,
// the query operand and the output.  So unpacking costs one AND per pair (and
// a shift per four).  A group's scale and minimum never touch the codes:
//   score(t) = s_t (q . c_t) + m_t sum(q),
//   O        = sum_t (p_t s_t) c_t + sum_t p_t m_t,
// with s and m in f32 and p_t s_t rounded to f16, or to the sum of two f16
// (kTwo) where the output is f16: one rounding moves values that are small
// against s c and m, of which they are the difference, by more than the
// output's own (measured: 5.0e-4 of the result for 2.1e-4).  Over dense keys a
// bf16 weight is the sum of two (one alone has 8 bits), an f16 weight one f16.
// The running reference of the softmax is the maximum of score + log2(|s of v|),
// so p_t s_t is at most 1 whatever the scales are, and 11 bits of it are kept.
//
// The work is dealt by cost, not by sequence: every CTA gets the same number
// of units of 128 tokens (a begun segment counts two more), whatever lengths
// the sequences have, and segments that two CTAs share are joined by a second
// small kernel.
//
// Measured at 1965 MHz: 4 x 64 heads over 8, D = 128, 4 bits, 131072 tokens:
// 127 us, 4.4 TB/s of codes, scales and minima (0.68 of the measured HBM rate:
// an instruction issues in 57 % of the clocks, four warps a scheduler that wait
// for fixed latencies and the ALU); 32 sequences of 4096: 34 to 35 us for 14.5,
// 9 of them what a call over one sequence of 517 tokens takes (find the segment 1,
// first loads 2, queries 1, sums and output 2.5, the joining kernel 3).  Dense
// bf16, 16 x 32 heads over 8, 4096 of 8192 tokens: 47 us, 0.86 of the HBM rate.
// Shifting by mul.hi instead of by the ALU took 135 for then 124 us.
#pragma once

#include <atomic>

#include "attn_common.cuh"

namespace llk_b200 {
namespace split_attn {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kTok = 16;      // tokens of a block (one mma tile)
constexpr int kUnit = 8;      // blocks of a unit of work, which a CTA's warps share
constexpr int kSpan = kUnit * kTok;
// The reference of the softmax may lag the largest weight by up to this power
// of two before the sums are rescaled: weights stay below 2^8, far inside f16.
constexpr float kSlack = 8.f;
// The reference before any token: below every score, and finite, so that a
// masked score (-inf) less it is -inf.
constexpr float kNoRef = -1e38f;
// A weight carries the magnitude of its token's largest value scale, and each
// group's ratio to it follows, its sign with it: a caller's pool may hold
// negative scales, and zeros (slots never written, constant rows of another
// writer).  The magnitude counts as kLeastScale at least: far below any scale
// in use, so that a zero leaves the other tokens' weights their bits, and large
// enough that a token's own weight is not lost below 2^-126.  (The ratio costs
// a multiplication a weight also where a row is one group: 125 to 128 us at
// 131072 tokens.  A branch around it, taken by a vote on the block's scales,
// took 132.)
constexpr float kLeastScale = 0x1p-60f;

struct Params {
  AttnProblem p;
  KvPool pool;
  const int *table;
  int64_t table_width;
  int row_blocks;
  int workers;      // CTAs that share the work
  int page_shift;   // log2 of the page, or -1
  int q_vec;        // query rows start on 4 bytes
  float *part_o;    // [2 workers, 8 NT, D]: a CTA's parts of cut segments (slots as above combine_kernel)
  float2 *part_ml;  // [2 workers, 8 NT] (reference, sum)
};

constexpr int cmin(int a, int b) { return a < b ? a : b; }
constexpr int pow2_in(int n) { return n & -n; }
template <int A, int B>
constexpr int cmin_v = A < B ? A : B;

// Geometry of one (BITS, D, group): which words of a row a lane holds.
template <int BITS, int D, int G>
struct Geo {
  static constexpr int E = 32 / BITS;             // elements a word
  static constexpr int ROW = D * BITS / 32;       // words a row
  static constexpr int GROUP = D / G;
  // K: the four lanes of a token take VW neighbouring words each of a chunk
  // of 4 VW words, which lies in one group.
  static constexpr int WK = ROW / 4;
  static constexpr int VW = cmin(4, cmin(pow2_in(WK), pow2_in(BITS == 16 ? WK : GROUP / E / 4)));
  static constexpr int CHUNKS = WK / VW;
  // V: the eight lanes of a token take UB neighbouring bytes each of a unit
  // of 8 UB bytes, which lies in one group.
  static constexpr int LB = D * BITS / 64;        // bytes a lane
  static constexpr int UB = cmin(16, cmin(pow2_in(LB), pow2_in(BITS == 16 ? LB : GROUP * BITS / 64)));
  static constexpr int NU = LB / UB;
  static constexpr int UR = UB < 4 ? 1 : UB / 4;  // registers a unit
  static constexpr int TILES = D / 16;            // 16-element tiles of O^T
  static constexpr int UT = TILES / NU;           // tiles a unit
  // A warp's turn is HV blocks.  A stage of its ring, for each of them: 16
  // rows of K, of V, then each token's (scale, min) of K and of V.
  static constexpr int ROWB = D * BITS / 8, CPR = ROWB / 16;  // bytes, 16-byte chunks a row
  static constexpr int PG = BITS == 16 ? 0 : 4 * G;           // bytes of a token's parameters, of K or V
  static constexpr int HV = D * BITS <= 512 ? 2 : 1;
  static constexpr int BLOCK = kTok * (2 * ROWB + 2 * PG);
  static constexpr int STAGE = HV * BLOCK;
  static constexpr int STAGES = STAGE <= 2560 ? 4 : 3;
};

// Row t of an mma tile's 16 slots holds token slot_token(t): the four lanes'
// value tokens (slots 2c, 2c + 1) are of both parities then, which spreads
// rows of 64 bytes over all banks.
__host__ __device__ constexpr int slot_token(int t) { return t ^ ((t >> 1) & 1); }
// Chunks of row (token) t are stored permuted, chunk ^ swizzle(t), so that the
// key reads (two tokens' neighbouring chunks a quarter warp) and the value
// reads (four tokens' two chunks) both meet all banks once.
template <int CPR>
__device__ __forceinline__ int swizzle(int t) {
  if constexpr (CPR >= 8 && (CPR & (CPR - 1)) == 0) return ((t & 6) ^ ((t & 1) << 2));
  if constexpr (CPR == 4) return (t >> 1) & 2;
  return 0;
}

// N bytes from global to shared memory; without `in` zeros (nothing is read).
template <int N>
__device__ __forceinline__ void cp_async(uint32_t dst, const void *src) {
  if constexpr (N == 16) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  } else {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(N) : "memory");
  }
}
__device__ __forceinline__ void cp_async16_if(uint32_t dst, const void *src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}

template <int WORDS>
__device__ __forceinline__ void lds(const uint8_t *a, uint32_t *w) {
  if constexpr (WORDS == 4) {
    const uint4 x = *reinterpret_cast<const uint4 *>(a);
    w[0] = x.x;
    w[1] = x.y;
    w[2] = x.z;
    w[3] = x.w;
  } else if constexpr (WORDS == 2) {
    const uint2 x = *reinterpret_cast<const uint2 *>(a);
    w[0] = x.x;
    w[1] = x.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t *>(a);
  }
}

template <bool kBf16>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  if constexpr (kBf16) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}

// The same onto zeros.
template <bool kBf16>
__device__ __forceinline__ void mma16816_zero(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  if constexpr (kBf16) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
  } else {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
  }
}

__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

template <bool kBf16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (kBf16) {
    asm("cvt.rn.bf16x2.f32 %0, %2, %1;" : "=r"(r) : "f"(lo), "f"(hi));
  } else {
    asm("cvt.rn.f16x2.f32 %0, %2, %1;" : "=r"(r) : "f"(lo), "f"(hi));
  }
  return r;
}

template <bool kBf16>
__device__ __forceinline__ float2 unpack2(uint32_t r) {
  if constexpr (kBf16) {
    return make_float2(__uint_as_float(r << 16), __uint_as_float(r & 0xffff0000u));
  } else {
    return __half22float2(*reinterpret_cast<const __half2 *>(&r));
  }
}

__device__ __forceinline__ void store_o(void *o, int64_t at, int dtype, float v) {
  if (dtype == LLK_DTYPE_FP16) {
    static_cast<__half *>(o)[at] = __float2half_rn(v);
  } else {
    static_cast<__nv_bfloat16 *>(o)[at] = __float2bfloat16_rn(v);
  }
}

// The 16-token blocks that any query of a sequence sees: nsb blocks of
// sinks, then from the window's first block.
struct Range {
  int n, m;            // keys, queries
  int p_first, p_last; // positions of the first and the last query
  int lo, s_end;       // keys seen: [0, s_end) and [lo, n)
  int nsb, wb0, blocks;
  int full0, full1;    // blocks of which every query sees every token
};

__device__ __forceinline__ Range make_range(const AttnMask &mk, int n, int m) {
  Range r;
  r.n = n;
  r.m = m;
  r.p_first = r.n - r.m;
  r.p_last = r.n - 1;
  r.lo = window_lo(mk, r.p_first);
  r.s_end = mk.sinks < r.lo ? mk.sinks : r.lo;
  r.nsb = (r.s_end + kTok - 1) / kTok;
  r.wb0 = r.lo / kTok;
  if (r.nsb > r.wb0) r.nsb = r.wb0;  // the sinks reach into the window's first block
  const int end = (r.n + kTok - 1) / kTok;
  r.blocks = r.m > 0 && end > r.wb0 ? r.nsb + end - r.wb0 : 0;
  // (of the window's blocks; the sinks' are looked at token by token)
  const int last_lo = window_lo(mk, r.p_last);
  r.full0 = r.nsb + (last_lo + kTok - 1) / kTok - r.wb0;
  r.full1 = r.nsb + (r.p_first + 1 > 0 ? (r.p_first + 1) / kTok : 0) - r.wb0;
  return r;
}

// ---- The work and its split.  A segment is a (sequence, key head, block of
// query rows); its units are kSpan tokens each, at least one (a segment
// without tokens still writes its zeros), and it costs kStart more: the time
// before a segment's first tokens are there and behind its last, in units
// (measured: 2.5 us where a unit takes 1.2).  The cost of all segments in the
// order (sequence, key head, row block), each segment's start in front of its
// units, is dealt to the workers in runs of equal length (or one more),
// whatever the sequences' lengths are.  A segment whose units fall to one
// worker is written by it; of one that is cut, the first of its workers leaves
// its part in slot 2 w + 1 and each further one (whose run begins with it) in
// slot 2 w, and combine_kernel joins them in order.  (split_supported keeps
// all counts below 2^31.)
constexpr int kStart = 2;
__device__ __forceinline__ int seq_units(const AttnMask &mk, int b) {
  int n, m;
  seq_lens(mk, b, n, m);
  const int blocks = make_range(mk, n, m).blocks;
  return blocks > kUnit ? (blocks + kUnit - 1) / kUnit : 1;
}

// Cost of the sequences before b0 (*before) and of all (returned), of one
// segment each, by one warp.
__device__ __forceinline__ int count_cost(const AttnMask &mk, int B, int b0, int *before) {
  int all = 0, pre = 0;
  for (int b = threadIdx.x & 31; b < B; b += 32) {
    const int u = kStart + seq_units(mk, b);
    all += u;
    pre += b < b0 ? u : 0;
  }
  *before = __reduce_add_sync(0xffffffffu, pre);
  return __reduce_add_sync(0xffffffffu, all);
}

// The sequence that holds the place `at`, counting one segment a sequence:
// *first = cost before that sequence.  By one warp.
__device__ __forceinline__ int find_seq(const AttnMask &mk, int B, int at, int *first) {
  int base = 0;
  for (int b0 = 0; b0 < B; b0 += 32) {
    const int b = b0 + (threadIdx.x & 31);
    const int u = b < B ? kStart + seq_units(mk, b) : 0;
    int inc = u;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, off);
      if ((threadIdx.x & 31) >= off) inc += v;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, base + inc > at);
    if (hit) {
      const int l = __ffs(hit) - 1;
      *first = base + __shfl_sync(0xffffffffu, inc - u, l);
      return b0 + l;
    }
    base += __shfl_sync(0xffffffffu, inc, 31);
  }
  *first = base;
  return B;
}

// The runs: of a cost of `total`, worker w has each = total / workers, the
// first `more` workers one more.
struct Runs {
  int each, more, workers;
  __device__ __forceinline__ Runs(int total, int all) {
    workers = total < all ? total : all;
    each = total / workers;
    more = total - each * workers;
  }
  __device__ __forceinline__ int begin(int w) const { return w * each + (w < more ? w : more); }
  __device__ __forceinline__ int worker_of(int u) const {
    const int edge = more * (each + 1);
    return u < edge ? u / (each + 1) : more + (u - edge) / each;
  }
};

// Row R of a (sequence, key head): query R / g, head hk g + R % g.
__device__ __forceinline__ int64_t row_at(const View4 &v, int b, int hk, int g, int R) {
  return b * v.sb + static_cast<int64_t>(hk * g + R % g) * v.sh + static_cast<int64_t>(R / g) * v.sl;
}

__device__ __forceinline__ float lg2_approx(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A block that does not exist, or whose page is not in the pool.
constexpr uint32_t kNoBlock = 0xffffffffu;

template <int BITS, int D, int G, bool kBf16, bool kTwo, int NT, int CTAS>
__global__ void __launch_bounds__(kThreads, CTAS) split_kernel(const __grid_constant__ Params A) {
  using X = Geo<BITS, D, G>;
  constexpr int E = X::E, WK = X::WK, VW = X::VW, NU = X::NU, UR = X::UR, UT = X::UT;
  constexpr bool kQuant = BITS < 16;
  constexpr int KS = D / 16;  // k16 steps of a score
  constexpr int kLd = D + 2;
  // the warps' rings, and at a segment's end [kWarps][8 NT][kLd] sums in their place
  extern __shared__ __align__(128) uint8_t smem[];
  float *buf = reinterpret_cast<float *>(smem);
  __shared__ float2 ml[kWarps][8 * NT];
  __shared__ __align__(16) uint16_t qs[8 * NT][4 * KS * 4];  // the query operand, by row and lane c
  __shared__ float qfac[8 * NT], qsum[8 * NT][kQuant ? G : 1];

  const AttnProblem &P = A.p;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, c = lane & 3;
  const int g = P.H / P.Hkv, per_seq = P.Hkv * A.row_blocks;
  pdl_wait();
  pdl_launch_dependents();  // (after the wait: the next kernel may read the lengths before its own)
  int before;
  const int total = count_cost(P.mask, P.B, 0, &before) * per_seq;
  const Runs runs(total, A.workers);
  if (static_cast<int>(blockIdx.x) >= runs.workers) return;
  const int run1 = runs.begin(blockIdx.x + 1);
  int at = runs.begin(blockIdx.x), seq0;
  int b = find_seq(P.mask, P.B, at / per_seq, &seq0);
  seq0 *= per_seq;
  constexpr int HV = X::HV, kTurns = 32 / HV, kStep = kWarps * HV;
  auto token0 = [&](const Range &rg, int blk) { return (blk < rg.nsb ? blk : rg.wb0 + blk - rg.nsb) * kTok; };
  // row of a block's first token among the rows of the pool (dense: of the head)
  auto look = [&](const Range &rg, int b_at, int hk, int blk, int end) -> uint32_t {
    if (blk >= end) return kNoBlock;
    const int t0 = token0(rg, blk);
    if constexpr (kQuant) {
      const int page = A.page_shift >= 0 ? t0 >> A.page_shift : t0 / A.pool.page;
      const int entry = A.table[b_at * A.table_width + page];
      if (entry < 0 || entry >= A.pool.num_pages) return kNoBlock;
      return (static_cast<uint32_t>(entry) * P.Hkv + hk) * A.pool.page + (t0 - page * A.pool.page);
    } else {
      return t0;
    }
  };
  // the first rows of the next segment, when this one's last are under way
  uint32_t rows_after = kNoBlock;
  bool looked = false;

  // ---- segment by segment
  while (at < run1) {
    int n, m;
    seq_lens(P.mask, b, n, m);
    const Range rg = make_range(P.mask, n, m);
    const int units = rg.blocks > kUnit ? (rg.blocks + kUnit - 1) / kUnit : 1;
    const int seg = (at - seq0) / (kStart + units), seg0 = seq0 + seg * (kStart + units);
    const int hk = seg / A.row_blocks, rb = seg - hk * A.row_blocks;
    const int v0 = at - seg0 - kStart, v1 = run1 - seg0 - kStart;
    const int u0 = v0 > 0 ? v0 : 0, u1 = v1 < units ? v1 : units;
    const int rows = g * rg.m, row0 = rb * 8 * NT;
    at = seg0 + kStart + u1;
    const int b_now = b;
    if (seg + 1 == per_seq && u1 == units) {
      seq0 = at;
      ++b;
    }
    const bool had = looked;
    looked = false;
    if (u1 <= u0) break;            // the run ends before the segment's first unit
    if (row0 >= rows) continue;     // rows behind the sequence's queries: nothing is written

    // ---- the queries' elements, on their way while the first blocks are sent for: warp w has rows w, w + 4, ..
    constexpr int kPairs = (D + 63) / 64, kRows = 8 * NT / kWarps;
    uint32_t qraw[kRows][kPairs];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int R = row0 + warp + kWarps * i;
      const uint16_t *q = static_cast<const uint16_t *>(P.q.p) + (R < rows ? row_at(P.q, b_now, hk, g, R) : 0);
#pragma unroll
      for (int k = 0; k < kPairs; ++k) {
        const int e = 2 * (lane + 32 * k);
        qraw[i][k] = 0;
        if (R < rows && e < D)
          qraw[i][k] = A.q_vec ? *reinterpret_cast<const uint32_t *>(q + e)
                               : q[e] | static_cast<uint32_t>(q[e + 1]) << 16;
      }
    }

    // ---- this warp's blocks of the segment's units [u0, u1); lane i looks at the i-th of the next 32
    const int beg = u0 * kUnit, end = u1 * kUnit < rg.blocks ? u1 * kUnit : rg.blocks;
    const int first = beg + warp * HV;
    auto look_ahead = [&](int turn) {
      return look(rg, b_now, hk, first + (turn + lane / HV) * kStep + lane % HV, end);
    };
    uint32_t rows_now = had ? rows_after : look_ahead(0);
    uint32_t rows_next = end - first > kTurns * kStep ? look_ahead(kTurns) : kNoBlock;

    const char *kbase, *vbase;
    int64_t k_sl, v_sl;  // bytes between tokens
    if constexpr (kQuant) {
      kbase = static_cast<const char *>(A.pool.k_codes);
      vbase = static_cast<const char *>(A.pool.v_codes);
      k_sl = v_sl = X::ROWB;
    } else {
      kbase = static_cast<const char *>(P.k.p) + 2 * (b_now * P.k.sb + hk * P.k.sh);
      vbase = static_cast<const char *>(P.v.p) + 2 * (b_now * P.v.sb + hk * P.v.sh);
      k_sl = 2 * P.k.sl;
      v_sl = 2 * P.v.sl;
    }
    // a token that no query of the sequence sees is not read: what lies there may be anything
    auto seen = [&](int t) { return t < rg.n && (t >= rg.lo || t < rg.s_end); };
    const uint32_t ring = warp * X::STAGES * X::STAGE, smem_at = smem_u32(smem);  // (offsets in smem)
    constexpr int kPer = kTok * X::CPR / 32;  // chunks of K (of V) a lane
    static_assert(kTok * X::CPR % 32 == 0, "whole chunks a lane");
    // chunk i of this lane: token (lane + 32 i) / CPR, its place in the stage
    uint32_t put[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = lane + 32 * i, t = e / X::CPR;
      put[i] = t * X::ROWB + (((e % X::CPR) ^ swizzle<X::CPR>(t)) << 4);
    }
    const char *psrc = static_cast<const char *>(lane < 16 ? A.pool.k_params : A.pool.v_params) + (lane & 15) * X::PG;
    const uint32_t pput = 2 * kTok * X::ROWB + (lane & 15) * 2 * X::PG + (lane >> 4) * X::PG;
    // a block into its place of a stage; tokens that are not read become zeros
    // (of kNoBlock nothing is used: codes are finite whatever lies in the stage)
    auto load = [&](uint32_t dst, int blk, uint32_t row) {
      if (row == kNoBlock) return;
      if (blk >= rg.full0 && blk < rg.full1) {
        if constexpr (kQuant) {
          const int64_t o = static_cast<int64_t>(row) * X::ROWB + lane * 16;
          const char *ks = kbase + o, *vs = vbase + o;
#pragma unroll
          for (int i = 0; i < kPer; ++i) {
            cp_async<16>(dst + put[i], ks + 512 * i);
            cp_async<16>(dst + put[i] + kTok * X::ROWB, vs + 512 * i);
          }
        } else {
#pragma unroll
          for (int i = 0; i < kPer; ++i) {
            const int64_t t = row + (lane + 32 * i) / X::CPR;
            const int ch = (lane + 32 * i) % X::CPR;
            cp_async<16>(dst + put[i], kbase + t * k_sl + 16 * ch);
            cp_async<16>(dst + put[i] + kTok * X::ROWB, vbase + t * v_sl + 16 * ch);
          }
        }
      } else {
        const int t0 = token0(rg, blk);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const int e = lane + 32 * i, t = e / X::CPR, ch = e % X::CPR;
          const bool in = seen(t0 + t);
          const int64_t at_row = static_cast<int64_t>(row) + t;
          cp_async16_if(dst + put[i], in ? kbase + at_row * k_sl + 16 * ch : kbase, in);
          cp_async16_if(dst + put[i] + kTok * X::ROWB, in ? vbase + at_row * v_sl + 16 * ch : vbase, in);
        }
      }
      if constexpr (kQuant) {
        // (a page is in the pool whole; what is not seen is masked when it is used)
        const char *src = psrc + static_cast<int64_t>(row) * X::PG;
#pragma unroll
        for (int i = 0; i < X::PG; i += 16) cp_async<cmin_v<X::PG, 16>>(dst + pput + i, src + i);
      }
    };

    const int tr = slot_token(r), tv = slot_token(2 * c);
    // where this lane reads in a block: key chunks of row tr, value units of rows tv and tv ^ 1, parameters of row tr
    uint32_t k_at[X::CHUNKS], v_at[2][NU];
#pragma unroll
    for (int u = 0; u < X::CHUNKS; ++u)
      k_at[u] = tr * X::ROWB + ((u * 16 * VW + c * 4 * VW) ^ (swizzle<X::CPR>(tr) << 4));
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int u = 0; u < NU; ++u)
        v_at[i][u] = (kTok + (tv ^ i)) * X::ROWB + ((u * 8 * X::UB + r * X::UB) ^ (swizzle<X::CPR>(tv ^ i) << 4));
    const uint32_t p_at = 2 * kTok * X::ROWB + tr * 2 * X::PG;
    uint32_t none = 0;  // blocks in the ring that do not exist, HV bits a turn, the latest lowest
    auto load_turn = [&](uint32_t dst, int blk, int turn) {
#pragma unroll
      for (int hv = 0; hv < HV; ++hv) {
        const int at_lane = turn * HV + hv;
        const uint32_t row = __shfl_sync(0xffffffffu, at_lane < 32 ? rows_now : rows_next, at_lane & 31);
        load(dst + hv * X::BLOCK, blk + hv, row);
        none = none << 1 | (row == kNoBlock ? 1u : 0u);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < X::STAGES - 1; ++i) load_turn(smem_at + ring + i * X::STAGE, first + i * kStep, i);

    // ---- the query operand: each row into shared memory in the order the lanes read it
#pragma unroll 1
    for (int i = 0; i < kRows; ++i) {
      const int row = warp + kWarps * i;
      float x[kPairs][2];
      int k2 = 0;
#pragma unroll
      for (int k = 0; k < kPairs; ++k) {
        uint32_t w = qraw[0][k];
#pragma unroll
        for (int j = 1; j < kRows; ++j) w = i == j ? qraw[j][k] : w;
        if constexpr (kQuant) {
          const float2 y = P.dtype == LLK_DTYPE_FP16 ? unpack2<false>(w) : unpack2<true>(w);
          x[k][0] = y.x;
          x[k][1] = y.y;
        } else {
          x[k][0] = __uint_as_float(w);  // (as it is)
        }
      }
      if constexpr (kQuant) {
        // q times a power of two into f16: exact down to 2^-24 of the row's
        // largest element, and 2^-35 of that below
        float top = 0.f;
#pragma unroll
        for (int k = 0; k < kPairs; ++k) top = fmaxf(top, fmaxf(fabsf(x[k][0]), fabsf(x[k][1])));
        top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
        const int ex = static_cast<int>(__float_as_uint(top) >> 23) - 127;  // floor(log2 top)
        k2 = top > 0.f && ex < 128 ? 9 - ex : 0;  // -118 at least
        k2 = k2 > 126 ? 126 : k2;
        const float up = __uint_as_float(static_cast<uint32_t>(127 + k2) << 23);
#pragma unroll
        for (int k = 0; k < kPairs; ++k) {
          x[k][0] *= up;
          x[k][1] *= up;
        }
        // each group's sum in the units of the tensor core's scores, 2^-24 up
#pragma unroll
        for (int gi = 0; gi < G; ++gi) {
          float sum = 0.f;
#pragma unroll
          for (int k = 0; k < kPairs; ++k)
            if (2 * (lane + 32 * k) / X::GROUP == gi) sum += x[k][0] + x[k][1];
#pragma unroll
          for (int off = 16; off >= 1; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
          if (lane == 0) qsum[row][gi] = sum * 0x1p-24f;
        }
      }
      if constexpr (kQuant) {
        // (the largest bf16 queries, from 2^113 on: a factor that is finite still tells their scores apart)
        const float f = scalbnf(P.scale * kLog2e, 24 - k2);
        if (lane == 0) qfac[row] = fminf(fmaxf(f, -0x1.fffffep127f), 0x1.fffffep127f);
      } else if (lane == 0) {
        qfac[row] = P.scale * kLog2e;
      }
#pragma unroll
      for (int k = 0; k < kPairs; ++k) {
        const int e = 2 * (lane + 32 * k);  // even, so e and e + 1 lie in one word
        if (e < D) {
          const int word = e / E, in = e % E, lc = word / VW % 4, w = word / (4 * VW) * VW + word % VW;
          if constexpr (BITS == 4) {
            // word w's elements (i, i + 4): operand registers 0 (i = 0), 1 (1, held 16 times), 2 (2), 3 (3, 16 times)
            uint16_t *to = &qs[row][(lc * KS + 2 * w + ((in & 2) >> 1)) * 4 + (in >> 2)];
            to[0] = __half_as_ushort(__float2half_rn(x[k][0]));
            to[2] = __half_as_ushort(__float2half_rn(x[k][1] * 0.0625f));
          } else if constexpr (BITS == 8) {
            // (0, 2) and (1, 3)
            uint16_t *to = &qs[row][(lc * KS + w) * 4 + (in >> 1)];
            to[0] = __half_as_ushort(__float2half_rn(x[k][0]));
            to[2] = __half_as_ushort(__float2half_rn(x[k][1]));
          } else {
            *reinterpret_cast<uint32_t *>(&qs[row][(lc * KS + w / 2) * 4 + 2 * (w % 2)]) = __float_as_uint(x[k][0]);
          }
        }
      }
    }
    __syncthreads();
    uint32_t qf[NT][KS][2];
    float fcol[NT][2], mq[NT][kQuant ? G : 1][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        const uint2 w = *reinterpret_cast<const uint2 *>(&qs[8 * nt + r][(c * KS + k) * 4]);
        qf[nt][k][0] = w.x;
        qf[nt][k][1] = w.y;
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        fcol[nt][j] = qfac[8 * nt + 2 * c + j];
#pragma unroll
        for (int gi = 0; gi < (kQuant ? G : 1); ++gi) mq[nt][gi][j] = kQuant ? qsum[8 * nt + 2 * c + j][gi] : 0.f;
      }
    }
    if (kQuant && u1 == units && at < run1) {
      // the run goes on: look at the next segment's first blocks now (kStep at a time, like this one's)
      int n2, m2;
      seq_lens(P.mask, b, n2, m2);
      const Range r2 = make_range(P.mask, n2, m2);
      const int units2 = r2.blocks > kUnit ? (r2.blocks + kUnit - 1) / kUnit : 1;
      const int v2 = run1 - at - kStart, e2 = v2 < units2 ? v2 * kUnit : r2.blocks;
      const int seg2 = b != b_now ? 0 : seg + 1;
      rows_after = look(r2, b, seg2 / A.row_blocks, (warp + lane / HV * kWarps) * HV + lane % HV,
                        e2 < r2.blocks ? e2 : r2.blocks);
      looked = true;
    }
    float acc[X::TILES][NT][4], mrun[NT][2], l[NT][2], pm[NT][kQuant ? G : 1][2];
#pragma unroll
    for (int t = 0; t < X::TILES; ++t)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][nt][i] = 0.f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        mrun[nt][j] = kNoRef;
        l[nt][j] = 0.f;
#pragma unroll
        for (int i = 0; i < (kQuant ? G : 1); ++i) pm[nt][i][j] = 0.f;
      }

    uint32_t at_use = ring, at_load = ring + (X::STAGES - 1) * X::STAGE;
    const uint32_t ring_end = ring + X::STAGES * X::STAGE;
    int turn = 0;  // of the 32 rows in rows_now
    for (int blk = first; blk < end; blk += kStep) {
      // the turn STAGES - 1 ahead goes where the last one was (all lanes have read it); then this one is waited for
      __syncwarp();
      load_turn(smem_at + at_load, blk + (X::STAGES - 1) * kStep, turn + X::STAGES - 1);
      at_load = at_load + X::STAGE == ring_end ? ring : at_load + X::STAGE;
      asm volatile("cp.async.wait_group %0;" ::"n"(X::STAGES - 1) : "memory");
      __syncwarp();
      if (++turn == kTurns) {
        turn = 0;
        rows_now = rows_next;
        rows_next = look_ahead((blk - first) / kStep + 1 + kTurns);
      }
      if (kQuant && looked && blk == first) {
        // the next segment's first turns into L2
#pragma unroll
        for (int i = 0; i < (X::STAGES - 1) * HV; ++i) {
          const uint32_t row = __shfl_sync(0xffffffffu, rows_after, i);
          constexpr int kLines = kTok * X::ROWB / 128;
          if (row != kNoBlock && (lane & 15) < kLines) {
            const char *at_l2 = (lane < 16 ? kbase : vbase) + static_cast<int64_t>(row) * X::ROWB + (lane & 15) * 128;
            asm volatile("prefetch.global.L2 [%0];" ::"l"(at_l2));
          }
        }
      }
      const uint32_t absent = none >> ((X::STAGES - 1) * HV);
      const bool full = blk >= rg.full0 && blk + HV <= rg.full1 && (absent & ((1u << HV) - 1)) == 0;
      float z[HV][NT][4], sr[HV][2][kQuant ? G : 1], mr[HV][2][kQuant ? G : 1], rs[HV][2];
#pragma unroll
      for (int hv = 0; hv < HV; ++hv) {
        const uint32_t stage = at_use + hv * X::BLOCK;
        uint32_t kw[2][WK], par[2][kQuant ? 2 * G : 1];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
          for (int u = 0; u < X::CHUNKS; ++u)
            lds<VW>(smem + (stage + k_at[u]) + 8 * i * X::ROWB, &kw[i][u * VW]);
          if constexpr (kQuant) {
#pragma unroll
            for (int w = 0; w < 2 * G; w += cmin_v<2 * G, 4>)
              lds<cmin_v<2 * G, 4>>(smem + (stage + p_at) + 8 * i * 2 * X::PG + 4 * w, &par[i][w]);
          }
        }
        if constexpr (kQuant) {
          if (!full) {
            // parameters of tokens that no query sees may be anything: here scale 1, min 0
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const bool in = !(absent >> (HV - 1 - hv) & 1) && seen(token0(rg, blk + hv) + tr + 8 * i);
#pragma unroll
              for (int w = 0; w < 2 * G; ++w) par[i][w] = in ? par[i][w] : 0x3f80u;
            }
          }
        }
        // ---- scores of this lane's tokens (slots r, r + 8) and its two columns, in the tensor core's units
        float s2[NT][4], cg[NT][4];
        constexpr int kWordsAStep = BITS == 16 ? 2 : 1;
#pragma unroll
        for (int w = 0; w < WK; w += kWordsAStep) {
          const uint32_t x = kw[0][w], y = kw[1][w];
          const int gi = kQuant ? (w / VW) * 4 * VW * E / X::GROUP : 0;
          // the first and the last word of a group
          const bool starts = w == 0 || (kQuant && ((w - 1) / VW) * 4 * VW * E / X::GROUP != gi);
          const bool ends = kQuant && (w + 1 == WK || ((w + 1) / VW) * 4 * VW * E / X::GROUP != gi);
          if constexpr (BITS == 4) {
            const uint32_t xs = (x >> 8), ys = (y >> 8);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              if (starts) {
                mma16816_zero<false>(cg[nt], x & 0x000f000fu, y & 0x000f000fu, x & 0x00f000f0u, y & 0x00f000f0u,
                                     qf[nt][2 * w][0], qf[nt][2 * w][1]);
              } else {
                mma16816<false>(cg[nt], x & 0x000f000fu, y & 0x000f000fu, x & 0x00f000f0u, y & 0x00f000f0u,
                                qf[nt][2 * w][0], qf[nt][2 * w][1]);
              }
              mma16816<false>(cg[nt], xs & 0x000f000fu, ys & 0x000f000fu, xs & 0x00f000f0u, ys & 0x00f000f0u,
                              qf[nt][2 * w + 1][0], qf[nt][2 * w + 1][1]);
            }
          } else if constexpr (BITS == 8) {
            const uint32_t a0 = x & 0x00ff00ffu, a1 = y & 0x00ff00ffu, a2 = (x >> 8) & 0x00ff00ffu,
                           a3 = (y >> 8) & 0x00ff00ffu;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              if (starts) {
                mma16816_zero<false>(cg[nt], a0, a1, a2, a3, qf[nt][w][0], qf[nt][w][1]);
              } else {
                mma16816<false>(cg[nt], a0, a1, a2, a3, qf[nt][w][0], qf[nt][w][1]);
              }
            }
          } else {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              if (starts) {
                mma16816_zero<kBf16>(cg[nt], x, y, kw[0][w + 1], kw[1][w + 1], qf[nt][w / 2][0], qf[nt][w / 2][1]);
              } else {
                mma16816<kBf16>(cg[nt], x, y, kw[0][w + 1], kw[1][w + 1], qf[nt][w / 2][0], qf[nt][w / 2][1]);
              }
            }
          }
          if (ends) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t pw = par[i >> 1][gi];
              const float sc = __uint_as_float(pw << 16), mn = __uint_as_float(pw & 0xffff0000u);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                const float um = gi == 0 ? mn * mq[nt][gi][i & 1] : fmaf(mn, mq[nt][gi][i & 1], s2[nt][i]);
                s2[nt][i] = fmaf(sc, cg[nt][i], um);
              }
            }
          }
        }
        if constexpr (!kQuant) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) s2[nt][i] = cg[nt][i];
        }
        // ---- z = log2 of the weight p s_v; a token's p, its p min_v and its p s_v of a group follow from the weight by
        // factors of the token
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float lg = 0.f;
          rs[hv][i] = 1.f;
          if constexpr (kQuant) {
            float mx = kLeastScale;
#pragma unroll
            for (int gi = 0; gi < G; ++gi) {
              sr[hv][i][gi] = __uint_as_float(par[i][G + gi] << 16);
              mx = fmaxf(mx, fabsf(sr[hv][i][gi]));
            }
            lg = lg2_approx(mx);
            rs[hv][i] = rcp_approx(mx);
#pragma unroll
            for (int gi = 0; gi < G; ++gi) {
              sr[hv][i][gi] *= rs[hv][i];
              mr[hv][i][gi] = __uint_as_float(par[i][G + gi] & 0xffff0000u) * rs[hv][i];
            }
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j) z[hv][nt][2 * i + j] = fmaf(s2[nt][2 * i + j], fcol[nt][j], lg);
        }
        // masks: only turns at an edge of some row's range compare token by token
        if (!full) {
          const int t0 = token0(rg, blk + hv);
          const bool gone = absent >> (HV - 1 - hv) & 1;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int R = row0 + 8 * nt + 2 * c + (i & 1), p = R < rows ? rg.p_first + R / g : -1;
              if (gone || !key_visible(t0 + tr + 8 * (i >> 1), p, window_lo(P.mask, p), P.mask.sinks))
                z[hv][nt][i] = -INFINITY;
            }
        }
      }
      // ---- the reference, when some weight is far above it
      bool grew = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float mx = fmaxf(z[0][nt][j], z[0][nt][2 + j]);
          if constexpr (HV == 2) mx = fmaxf(mx, fmaxf(z[HV - 1][nt][j], z[HV - 1][nt][2 + j]));
          grew |= mx > mrun[nt][j] + kSlack;
        }
      if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float mx = mrun[nt][j];
#pragma unroll
            for (int hv = 0; hv < HV; ++hv) mx = fmaxf(mx, fmaxf(z[hv][nt][j], z[hv][nt][2 + j]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            const float corr = exp2_approx(mrun[nt][j] - mx);
            mrun[nt][j] = mx;
            l[nt][j] *= corr;
#pragma unroll
            for (int gi = 0; gi < (kQuant ? G : 1); ++gi) pm[nt][gi][j] *= corr;
#pragma unroll
            for (int t = 0; t < X::TILES; ++t) {
              acc[t][nt][j] *= corr;
              acc[t][nt][2 + j] *= corr;
            }
          }
      }
      // ---- weights and values
#pragma unroll
      for (int hv = 0; hv < HV; ++hv) {
        const uint32_t stage = at_use + hv * X::BLOCK;
        uint32_t vw[4][NU * UR];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
          for (int u = 0; u < NU; ++u) {
            const uint8_t *a = smem + (stage + v_at[i & 1][u]) + 8 * (i >> 1) * X::ROWB;
            if constexpr (X::UB == 2) {
              vw[i][u] = *reinterpret_cast<const uint16_t *>(a);
            } else {
              lds<UR>(a, &vw[i][u * UR]);
            }
          }
        }
        constexpr int kLo = kTwo ? 2 : 1;  // weights as a sum of two, so that their rounding does not show
        uint32_t bw[kQuant ? G : 1][NT][2][kLo];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float wt[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              wt[j] = exp2_approx(z[hv][nt][2 * i + j] - mrun[nt][j]);
              l[nt][j] = kQuant ? fmaf(wt[j], rs[hv][i], l[nt][j]) : l[nt][j] + wt[j];
            }
#pragma unroll
            for (int gi = 0; gi < (kQuant ? G : 1); ++gi) {
              float w0 = wt[0], w1 = wt[1];
              if constexpr (kQuant) {
#pragma unroll
                for (int j = 0; j < 2; ++j) pm[nt][gi][j] = fmaf(wt[j], mr[hv][i][gi], pm[nt][gi][j]);
                w0 *= sr[hv][i][gi];
                w1 *= sr[hv][i][gi];
              }
              const uint32_t hi = pack2<kBf16>(w0, w1);
              bw[gi][nt][i][0] = movmatrix_trans(hi);
              if constexpr (kTwo) {
                const float2 back = unpack2<kBf16>(hi);
                bw[gi][nt][i][1] = movmatrix_trans(pack2<kBf16>(w0 - back.x, w1 - back.y));
              }
            }
          }
#pragma unroll
        for (int u = 0; u < NU; ++u) {
          const int gi = kQuant ? u * 8 * X::UB * 8 / BITS / X::GROUP : 0;
#pragma unroll
          for (int w = 0; w < UR; ++w) {
            // halves of the word: the tokens of slots (2c, 2c + 1) and (2c + 8, 2c + 9)
            const uint32_t x0 = vw[0][u * UR + w], x1 = vw[1][u * UR + w], x2 = vw[2][u * UR + w],
                           x3 = vw[3][u * UR + w];
            const uint32_t lo01 = __byte_perm(x0, x1, 0x5410), lo23 = __byte_perm(x2, x3, 0x5410);
            const uint32_t hi01 = X::UB == 2 ? 0u : __byte_perm(x0, x1, 0x7632);
            const uint32_t hi23 = X::UB == 2 ? 0u : __byte_perm(x2, x3, 0x7632);
            if constexpr (BITS == 16) {
              const int tile = u * UT + w;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int q = 0; q < kLo; ++q)
                  mma16816<kBf16>(acc[tile][nt], lo01, hi01, lo23, hi23, bw[0][nt][0][q], bw[0][nt][1][q]);
            } else {
#pragma unroll
              for (int hf = 0; hf < (X::UB == 2 ? 1 : 2); ++hf) {
                const uint32_t a = hf ? hi01 : lo01, d = hf ? hi23 : lo23;
                if constexpr (BITS == 8) {
                  const int tile = u * UT + 2 * w + hf;
#pragma unroll
                  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int q = 0; q < kLo; ++q)
                      mma16816<false>(acc[tile][nt], a & 0x00ff00ffu, (a >> 8) & 0x00ff00ffu, d & 0x00ff00ffu,
                                      (d >> 8) & 0x00ff00ffu, bw[gi][nt][0][q], bw[gi][nt][1][q]);
                } else {
#pragma unroll
                  for (int k = 0; k < 2; ++k) {
                    const uint32_t as = k ? (a >> 8) : a, ds = k ? (d >> 8) : d;
                    const int tile = u * UT + 4 * w + 2 * hf + k;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                      for (int q = 0; q < kLo; ++q)
                        mma16816<false>(acc[tile][nt], as & 0x000f000fu, as & 0x00f000f0u, ds & 0x000f000fu,
                                        ds & 0x00f000f0u, bw[gi][nt][0][q], bw[gi][nt][1][q]);
                  }
                }
              }
            }
          }
        }
      }
      at_use = at_use + X::STAGE == ring_end ? ring : at_use + X::STAGE;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();  // every warp has left its ring: the sums go there

    // ---- join the warps: each leaves its sums in shared memory, relative to its own reference
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int col = 8 * nt + 2 * c + j;
#pragma unroll
        for (int off = 4; off <= 16; off <<= 1) {
          l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], off);
          if constexpr (kQuant) {
#pragma unroll
            for (int gi = 0; gi < G; ++gi) pm[nt][gi][j] += __shfl_xor_sync(0xffffffffu, pm[nt][gi][j], off);
          }
        }
        if (r == 0) ml[warp][col] = make_float2(mrun[nt][j], l[nt][j]);
        float *dst = buf + (warp * 8 * NT + col) * kLd;
#pragma unroll
        for (int t = 0; t < X::TILES; ++t) {
          const int u = t / UT, in_u = t % UT;
          const int d = BITS == 16 ? (u * 8 + r) * X::UB / 2 + 2 * in_u : (u * 8 + r) * X::UB * 8 / BITS + 2 * in_u;
          const int gi = kQuant ? u * 8 * X::UB * 8 / BITS / X::GROUP : 0;
          const float up = kQuant ? 0x1p24f : 1.f, up1 = BITS == 4 ? 0x1p20f : up;
          *reinterpret_cast<float2 *>(dst + d) =
              make_float2(fmaf(acc[t][nt][j], up, pm[nt][gi][j]), fmaf(acc[t][nt][2 + j], up1, pm[nt][gi][j]));
        }
      }
    __syncthreads();
    // ---- out: the row's result, or this worker's part of it
    const bool whole = u0 == 0 && u1 == units;
    const int64_t slot = 2 * blockIdx.x + (u0 == 0 ? 1 : 0);
    for (int col = warp; col < 8 * NT; col += kWarps) {
      const int R = row0 + col;
      if (R >= rows) break;
      float ref = -INFINITY, sum = 0.f, f[kWarps];
#pragma unroll
      for (int v = 0; v < kWarps; ++v) ref = fmaxf(ref, ml[v][col].x);
#pragma unroll
      for (int v = 0; v < kWarps; ++v) {
        f[v] = exp2_approx(ml[v][col].x - ref);
        sum = fmaf(ml[v][col].y, f[v], sum);
      }
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      const int64_t o_at = row_at(P.o, b_now, hk, g, R);
      bool bad = false, nan = false;
      for (int d = lane; d < D; d += 32) {
        float x = 0.f;
#pragma unroll
        for (int v = 0; v < kWarps; ++v) x = fmaf(buf[(v * 8 * NT + col) * kLd + d], f[v], x);
        if (whole) {
          x *= inv;
          bad |= !isfinite(x);
          nan |= x != x;
          if constexpr (!kQuant && !kBf16) x = within_f16(x);
          store_o(P.o.p, o_at + d, P.dtype, x);
        } else {
          A.part_o[(slot * 8 * NT + col) * D + d] = x;
        }
      }
      if (!whole && lane == 0) A.part_ml[slot * 8 * NT + col] = make_float2(ref, sum);
      if constexpr (!kQuant) {
        // a value that the row does not see may be the cause (its own scores are not: see the sum)
        if (sum == sum && __any_sync(0xffffffffu, bad)) {
          using T = typename std::conditional<kBf16, __nv_bfloat16, __half>::type;
          const int pos = rg.p_first + R / g, lo = window_lo(P.mask, pos);
          const T *v = reinterpret_cast<const T *>(vbase);
          if (redo_row<T, true>(v, P.v.sl, P.mask, D, rg.n, rg.m, pos, lo, __any_sync(0xffffffffu, nan))) {
            __syncwarp();
            attention_row<T>(static_cast<const T *>(P.q.p) + row_at(P.q, b_now, hk, g, R),
                             reinterpret_cast<const T *>(kbase), v, static_cast<T *>(P.o.p) + o_at, P.k.sl, P.v.sl, D,
                             pos, lo, P.mask.sinks, P.scale * kLog2e);
          }
        }
      }
    }
    __syncthreads();  // buf and ml are free for the next segment
  }
}

// Joins the parts of the rows whose segment was cut: one warp a row, the
// workers in order.
template <int D, bool kBf16, bool kDense>
__global__ void __launch_bounds__(kThreads) combine_kernel(const __grid_constant__ Params A, int nrows) {
  const AttnProblem &P = A.p;
  const int lane = threadIdx.x & 31, g = P.H / P.Hkv;
  const int rows_all = g * P.mask.Lq, per_seq = P.Hkv * A.row_blocks;
  const unsigned id = blockIdx.x * kWarps + (threadIdx.x >> 5);  // ((b Hkv) + hk) rows_all + R
  const unsigned bh = id / rows_all;
  const int R = id - bh * rows_all, b = bh / P.Hkv, hk = bh - b * P.Hkv;
  if (b >= P.B) return;
  // Where the parts are, before the wait: the split kernel starts this one
  // when it has waited for the kernels before it, so the lengths are there.
  int n, m, before;
  seq_lens(P.mask, b, n, m);
  const int total = count_cost(P.mask, P.B, b, &before) * per_seq;
  const Runs runs(total, A.workers);
  const int units = seq_units(P.mask, b);
  const int first = before * per_seq + (hk * A.row_blocks + R / nrows) * (kStart + units) + kStart;
  const int w0 = runs.worker_of(first), w1 = runs.worker_of(first + units - 1);
  // whole: its worker writes it; rows behind the queries: nobody
  const bool cut = w0 != w1 && R < g * m;
  const int col = R % nrows;
  auto slot = [&](int w) { return static_cast<int64_t>(2 * w + (w == w0 ? 1 : 0)) * nrows + col; };
  pdl_launch_dependents();
  pdl_wait();
  if (!cut) return;
  constexpr int kPer = (D + 31) / 32, kAt = 4;  // parts in flight
  float ref = kNoRef, acc[kPer], sum = 0.f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) acc[i] = 0.f;
  for (int w = w0; w <= w1; w += kAt) {
    float2 t[kAt];
    float x[kAt][kPer];
#pragma unroll
    for (int k = 0; k < kAt; ++k) {
      t[k] = make_float2(kNoRef, 0.f);
      if (w + k <= w1) t[k] = A.part_ml[slot(w + k)];
#pragma unroll
      for (int i = 0; i < kPer; ++i)
        x[k][i] = w + k <= w1 && lane + 32 * i < D ? A.part_o[slot(w + k) * D + lane + 32 * i] : 0.f;
    }
    float top = ref;
#pragma unroll
    for (int k = 0; k < kAt; ++k) top = fmaxf(top, t[k].x);
    const float corr = exp2_approx(ref - top);
    sum *= corr;
#pragma unroll
    for (int i = 0; i < kPer; ++i) acc[i] *= corr;
    ref = top;
#pragma unroll
    for (int k = 0; k < kAt; ++k) {
      const float f = exp2_approx(t[k].x - ref);
      sum = fmaf(t[k].y, f, sum);
#pragma unroll
      for (int i = 0; i < kPer; ++i) acc[i] = fmaf(x[k][i], f, acc[i]);
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int64_t at = row_at(P.o, b, hk, g, R);
  bool bad = false, nan = false;
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (lane + 32 * i < D) {
      float x = acc[i] * inv;
      bad |= !isfinite(x);
      nan |= x != x;
      if constexpr (kDense && !kBf16) x = within_f16(x);
      store_o(P.o.p, at + lane + 32 * i, P.dtype, x);
    }
  if constexpr (kDense) {
    if (sum == sum && __any_sync(0xffffffffu, bad)) {
      using T = typename std::conditional<kBf16, __nv_bfloat16, __half>::type;
      const int pos = n - m + R / g, lo = window_lo(P.mask, pos);
      const T *v = static_cast<const T *>(P.v.p) + b * P.v.sb + hk * P.v.sh;
      if (redo_row<T, true>(v, P.v.sl, P.mask, D, n, m, pos, lo, __any_sync(0xffffffffu, nan))) {
        __syncwarp();
        attention_row<T>(static_cast<const T *>(P.q.p) + row_at(P.q, b, hk, g, R),
                         static_cast<const T *>(P.k.p) + b * P.k.sb + hk * P.k.sh, v, static_cast<T *>(P.o.p) + at,
                         P.k.sl, P.v.sl, D, pos, lo, P.mask.sinks, P.scale * kLog2e);
      }
    }
  }
}

// Dynamic shared memory of a CTA: the rings, or the warps' sums.
constexpr int split_smem(int bits, int D, int G, int NT) {
  const int rowb = D * bits / 8, block = kTok * (2 * rowb + (bits == 16 ? 0 : 8 * G));
  const int stage = block * (D * bits <= 512 ? 2 : 1), rings = kWarps * (stage <= 2560 ? 4 : 3) * stage;
  const int sums = kWarps * 8 * NT * (D + 2) * 4;
  return rings > sums ? rings : sums;
}

// CTAs of 128 threads an SM holds: what the registers (accumulators, query
// operand, a block's codes) and 228 KB of shared memory leave.  Not to the
// last KB: CTAs that come and go one by one leave gaps (measured: 6 of 148
// SMs then held one less, and their work waited for a whole CTA's time).
// With weights of two parts no more than without: llk_kv_cache_attention_scratch
// does not know the type.
constexpr int ctas_per_sm(int bits, int D, int G, int NT, bool two) {
  const int by_regs = bits < 16 && two && D < 256 ? (NT == 2 ? 2 : D == 64 && G == 1 ? 4 : 3) : D == 256    ? (bits == 16 ? 1 : 2)
                      : NT == 2   ? (D == 64 ? 3 : 2)
                      : bits == 16 ? (D == 128 ? 2 : 3)
                                   : (D == 128 && (bits == 8 || G > 1) ? 3 : 4);
  const int fixed = 8 * NT * (2 * D + 8 + 4 * G + 4) + kWarps * 64 * NT + 1024;
  const int by_smem = 224 * 1024 / (split_smem(bits, D, G, NT) + fixed);
  return by_regs < by_smem ? by_regs : by_smem;
}

template <int BITS, int D, int G, bool kBf16, bool kTwo, int NT>
cudaError_t launch_split(const Params &a, cudaStream_t stream) {
  using X = Geo<BITS, D, G>;
  constexpr int CTAS = ctas_per_sm(BITS, D, G, NT, kTwo), smem = split_smem(BITS, D, G, NT);
  static_assert(smem >= kWarps * X::STAGES * X::STAGE, "the rings' place");
  auto kern = split_kernel<BITS, D, G, kBf16, kTwo, NT, CTAS>;
  auto join = combine_kernel<D, kBf16, BITS == 16>;
  // Once a device.  Both kernels ask for the largest shared memory: while one
  // drains and the next one's CTAs move in, an SM cannot change its split of
  // shared memory and L1, and would hold fewer of them.
  static std::atomic<uint64_t> ready{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (e == cudaSuccess && !(ready.load(std::memory_order_acquire) & bit)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, 100);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(join, cudaFuncAttributePreferredSharedMemoryCarveout, 100);
    if (e == cudaSuccess) ready.fetch_or(bit, std::memory_order_release);
  }
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(a.workers));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kern, a);
  if (e == cudaSuccess && a.part_ml) {
    const int64_t rows = static_cast<int64_t>(a.p.B) * a.p.H * a.p.mask.Lq;
    cfg.gridDim = dim3(static_cast<unsigned>((rows + kWarps - 1) / kWarps));
    cfg.dynamicSmemBytes = 0;
    e = cudaLaunchKernelEx(&cfg, join, a, 8 * NT);
  }
  return e != cudaSuccess ? e : cudaGetLastError();
}

// Query rows of a block: one n = 8 tile, or two where a key head has more
// rows than that and the accumulators leave registers for it.
constexpr int row_tiles(int rows, int D) { return rows > 8 && D <= 128 ? 2 : 1; }

template <int BITS, int D, int G, bool kTwo>
cudaError_t launch_cache_nt(const Params &a, cudaStream_t stream) {
  if constexpr (row_tiles(16, D) == 2)
    if (row_tiles(a.p.H / a.p.Hkv * a.p.mask.Lq, D) == 2) return launch_split<BITS, D, G, false, kTwo, 2>(a, stream);
  return launch_split<BITS, D, G, false, kTwo, 1>(a, stream);
}

template <int BITS, bool kTwo>
cudaError_t launch_bits(const Params &a, cudaStream_t stream) {
  const int groups = a.p.D / a.pool.group;
  if (a.p.D == 64) return groups == 1 ? launch_cache_nt<BITS, 64, 1, kTwo>(a, stream) : launch_cache_nt<BITS, 64, 2, kTwo>(a, stream);
  if (a.p.D == 128)
    return groups == 1   ? launch_cache_nt<BITS, 128, 1, kTwo>(a, stream)
           : groups == 2 ? launch_cache_nt<BITS, 128, 2, kTwo>(a, stream)
                         : launch_cache_nt<BITS, 128, 4, kTwo>(a, stream);
  return groups == 2   ? launch_cache_nt<BITS, 256, 2, kTwo>(a, stream)
         : groups == 4 ? launch_cache_nt<BITS, 256, 4, kTwo>(a, stream)
                       : launch_cache_nt<BITS, 256, 8, kTwo>(a, stream);
}

cudaError_t launch_dense(const Params &a, cudaStream_t stream);      // kv_attention_dense.cu
cudaError_t launch_cache_f16(const Params &a, cudaStream_t stream);  // kv_attention_f16.cu

}  // namespace split_attn
}  // namespace llk_b200
