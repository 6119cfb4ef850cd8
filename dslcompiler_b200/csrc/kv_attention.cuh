// kv_attention.cuh -- attention of few query rows over many keys, split along
// the keys: over the quantised paged cache (4 or 8 bits) and over dense 16-bit
// keys and values.  Instantiated by kv_attention.cu and kv_attention_dense.cu.
//
// HBM-bound: every key and value byte is read once, from global memory
// straight into the registers that feed mma.sync (m16n8k16, f32
// accumulators).  The tensor cores only have to keep up with memory, not to
// approach their peak, and registers as operands cost no shared-memory round
// trip and no TMEM round trip for the softmax; so not tcgen05, whose operands
// come from shared memory.
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
// with s and m in f32 and p_t s_t rounded to f16.  The running reference of
// the softmax is the maximum of score + log2(s of v), so p_t s_t is at most 1
// whatever the scales are, and 11 bits of it are kept.
#pragma once

#include "attn_common.cuh"

namespace llk_b200 {
namespace split_attn {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kTok = 16;  // tokens of a block (one mma tile)

struct Params {
  AttnProblem p;
  KvPool pool;
  const int *table;
  int64_t table_width;
  int splits, row_blocks;
  float *part_o;   // [B, Hkv, row_blocks, splits, 8 NT, D]
  float2 *part_ml; // [B, Hkv, row_blocks, splits, 8 NT] (reference, sum)
};

constexpr int cmin(int a, int b) { return a < b ? a : b; }
constexpr int pow2_in(int n) { return n & -n; }

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
};

template <int WORDS>
__device__ __forceinline__ void ld_stream(const void *p, uint32_t *w) {
  if constexpr (WORDS == 4) {
    asm volatile("ld.global.nc.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];"
        : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
        : "l"(p));
  } else if constexpr (WORDS == 2) {
    asm volatile("ld.global.nc.L1::no_allocate.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
  } else {
    asm volatile("ld.global.nc.L1::no_allocate.b32 %0, [%1];" : "=r"(w[0]) : "l"(p));
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

// One query element (q is bf16 or f16 in every instance).
__device__ __forceinline__ float load_q(const void *q, int64_t at, int dtype) {
  return dtype == LLK_DTYPE_FP16 ? __half2float(static_cast<const __half *>(q)[at])
                                 : __bfloat162float(static_cast<const __nv_bfloat16 *>(q)[at]);
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
};

__device__ __forceinline__ Range seq_range(const AttnMask &mk, int b) {
  Range r;
  seq_lens(mk, b, r.n, r.m);
  r.p_first = r.n - r.m;
  r.p_last = r.n - 1;
  r.lo = window_lo(mk, r.p_first);
  r.s_end = mk.sinks < r.lo ? mk.sinks : r.lo;
  r.nsb = (r.s_end + kTok - 1) / kTok;
  r.wb0 = r.lo / kTok;
  if (r.nsb > r.wb0) r.nsb = r.wb0;  // the sinks reach into the window's first block
  const int end = (r.n + kTok - 1) / kTok;
  r.blocks = r.m > 0 && end > r.wb0 ? r.nsb + end - r.wb0 : 0;
  return r;
}

// Row R of a (sequence, key head): query R / g, head hk g + R % g.
__device__ __forceinline__ int64_t row_at(const View4 &v, int b, int hk, int g, int R) {
  return b * v.sb + static_cast<int64_t>(hk * g + R % g) * v.sh + static_cast<int64_t>(R / g) * v.sl;
}

template <int BITS, int D, int G, bool kBf16, int NT, int SUB>
__global__ void __launch_bounds__(kThreads) split_kernel(const Params A) {
  using X = Geo<BITS, D, G>;
  constexpr int E = X::E, WK = X::WK, VW = X::VW, NU = X::NU, UR = X::UR, UT = X::UT;
  constexpr bool kQuant = BITS < 16;
  constexpr int KS = D / 16;  // k16 steps of a score
  constexpr int kLd = D + 4;
  __shared__ float buf[8 * NT][kLd];
  __shared__ float2 ml[kWarps][8 * NT];

  const AttnProblem &P = A.p;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, r = lane >> 2, c = lane & 3;
  const int b = blockIdx.z, hk = blockIdx.y / A.row_blocks, rb = blockIdx.y % A.row_blocks, split = blockIdx.x;
  const int g = P.H / P.Hkv;
  pdl_launch_dependents();
  pdl_wait();
  const Range rg = seq_range(P.mask, b);
  const int rows = g * rg.m, row0 = rb * 8 * NT;
  if (row0 >= rows) return;  // no query here: nothing is written, nothing is combined

  // ---- queries: B operands, per-column factors and sums
  uint32_t qf[NT][KS][2];
  float fcol[NT][2], mq[NT][kQuant ? G : 1][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int R = row0 + 8 * nt + r;
    const bool in = R < rows;
    const int64_t at = in ? row_at(P.q, b, hk, g, R) : 0;
    auto elem = [&](int e) { return in ? load_q(P.q.p, at + e, P.dtype) : 0.f; };
    float up = 1.f;
    if constexpr (kQuant) {
      // q times a power of two into f16: exact down to 2^-24 of the row's
      // largest element, and 2^-35 of that below
      float top = 0.f;
#pragma unroll
      for (int w = 0; w < WK; ++w)
#pragma unroll
        for (int e = 0; e < E; ++e) top = fmaxf(top, fabsf(elem(E * ((w / VW) * 4 * VW + c * VW + w % VW) + e)));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int ex = static_cast<int>(__float_as_uint(top) >> 23) - 127;  // floor(log2 top)
      const int k = top > 0.f && ex < 128 ? 9 - ex : 0;
      up = k > 126 ? 0x1p126f : __uint_as_float(static_cast<uint32_t>(127 + (k < -126 ? -126 : k)) << 23);
      float sum[G];
#pragma unroll
      for (int i = 0; i < G; ++i) sum[i] = 0.f;
#pragma unroll
      for (int w = 0; w < WK; ++w) {
        const int word = (w / VW) * 4 * VW + c * VW + w % VW;
        float x[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
          x[e] = elem(E * word + e);
          sum[(w / VW) * 4 * VW * E / X::GROUP] += x[e];
          x[e] *= up;
        }
        if constexpr (BITS == 4) {
          qf[nt][2 * w][0] = pack2<false>(x[0], x[4]);
          qf[nt][2 * w][1] = pack2<false>(x[1] * 0.0625f, x[5] * 0.0625f);
          qf[nt][2 * w + 1][0] = pack2<false>(x[2], x[6]);
          qf[nt][2 * w + 1][1] = pack2<false>(x[3] * 0.0625f, x[7] * 0.0625f);
        } else {
          qf[nt][w][0] = pack2<false>(x[0], x[2]);
          qf[nt][w][1] = pack2<false>(x[1], x[3]);
        }
      }
#pragma unroll
      for (int i = 0; i < G; ++i) {
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
        sum[i] *= P.scale * kLog2e;
#pragma unroll
        for (int j = 0; j < 2; ++j) mq[nt][i][j] = __shfl_sync(0xffffffffu, sum[i], 4 * (2 * c + j));
      }
    } else {
#pragma unroll
      for (int w = 0; w < WK; ++w) {
        const int word = (w / VW) * 4 * VW + c * VW + w % VW;
        qf[nt][w / 2][w % 2] = pack2<kBf16>(elem(2 * word), elem(2 * word + 1));
      }
      mq[nt][0][0] = mq[nt][0][1] = 0.f;
    }
    const float f = P.scale * kLog2e * (kQuant ? 0x1p24f / up : 1.f);
#pragma unroll
    for (int j = 0; j < 2; ++j) fcol[nt][j] = __shfl_sync(0xffffffffu, f, 4 * (2 * c + j));
  }
  // the two columns of this lane in a score tile: rows row0 + 8 nt + 2 c + j
  int pcol[NT][2], wlo[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int R = row0 + 8 * nt + 2 * c + j;
      pcol[nt][j] = R < rows ? rg.p_first + R / g : -1;
      wlo[nt][j] = window_lo(P.mask, pcol[nt][j]);
    }

  // ---- this warp's blocks of the split's [beg, end)
  const int beg = static_cast<int>(static_cast<int64_t>(rg.blocks) * split / A.splits);
  const int end = static_cast<int>(static_cast<int64_t>(rg.blocks) * (split + 1) / A.splits);
  auto token0 = [&](int blk) { return (blk < rg.nsb ? blk : rg.wb0 + blk - rg.nsb) * kTok; };
  // row of the block's first token (in rows of a head), or -1: no such block, or a page that is not in the pool
  auto block_row = [&](int blk) -> int64_t {
    if (blk >= end) return -1;
    const int t0 = token0(blk);
    if constexpr (kQuant) {
      const int page = t0 / A.pool.page;
      const int entry = A.table[b * A.table_width + page];
      if (entry < 0 || entry >= A.pool.num_pages) return -1;
      return (static_cast<int64_t>(entry) * P.Hkv + hk) * A.pool.page + (t0 - page * A.pool.page);
    } else {
      return t0;
    }
  };
  const char *kbase, *vbase;
  int64_t k_sl, v_sl;  // bytes between tokens
  if constexpr (kQuant) {
    kbase = static_cast<const char *>(A.pool.k_codes);
    vbase = static_cast<const char *>(A.pool.v_codes);
    k_sl = v_sl = D * BITS / 8;
  } else {
    kbase = static_cast<const char *>(P.k.p) + 2 * (b * P.k.sb + hk * P.k.sh);
    vbase = static_cast<const char *>(P.v.p) + 2 * (b * P.v.sb + hk * P.v.sh);
    k_sl = 2 * P.k.sl;
    v_sl = 2 * P.v.sl;
  }
  // a token that no query of the sequence sees is not read: what lies there may be anything
  auto seen = [&](int t) { return t < rg.n && (t >= rg.lo || t < rg.s_end); };

  uint32_t kw[SUB][2][WK], vw[SUB][4][NU * UR], kp[SUB][2][kQuant ? G : 1], vp[SUB][2][kQuant ? G : 1];
  auto load_params = [&](const void *params, int64_t row, bool ok, uint32_t (&w)[kQuant ? G : 1]) {
    if constexpr (kQuant) {
#pragma unroll
      for (int i = 0; i < G; ++i) w[i] = 0;
      if (ok) {
        const uint32_t *src = static_cast<const uint32_t *>(params) + row * G;
        if constexpr (G >= 4) {
#pragma unroll
          for (int i = 0; i < G; i += 4) ld_stream<4>(src + i, w + i);
        } else {
          ld_stream<G>(src, w);
        }
      }
    }
  };
  auto load_k = [&](int s, int t0, int64_t row) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int t = r + 8 * i;
      const bool ok = row >= 0 && seen(t0 + t);
      const char *src = kbase + (row + t) * k_sl;
#pragma unroll
      for (int u = 0; u < X::CHUNKS; ++u) {
#pragma unroll
        for (int w = 0; w < VW; ++w) kw[s][i][u * VW + w] = 0;
        if (ok) ld_stream<VW>(src + 4 * (u * 4 * VW + c * VW), &kw[s][i][u * VW]);
      }
      load_params(A.pool.k_params, row + t, ok, kp[s][i]);
    }
  };
  auto load_v = [&](int s, int t0, int64_t row) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = 2 * c + (i & 1) + 8 * (i >> 1);
      const bool ok = row >= 0 && seen(t0 + t);
      const char *src = vbase + (row + t) * v_sl;
#pragma unroll
      for (int u = 0; u < NU; ++u) {
#pragma unroll
        for (int w = 0; w < UR; ++w) vw[s][i][u * UR + w] = 0;
        if (ok) {
          if constexpr (X::UB == 2) {
            unsigned short x;
            asm volatile("ld.global.nc.L1::no_allocate.u16 %0, [%1];" : "=h"(x) : "l"(src + (u * 8 + r) * 2));
            vw[s][i][u] = x;
          } else {
            ld_stream<UR>(src + (u * 8 + r) * X::UB, &vw[s][i][u * UR]);
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
      load_params(A.pool.v_params, row + r + 8 * i, row >= 0 && seen(t0 + r + 8 * i), vp[s][i]);
  };

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
      mrun[nt][j] = -INFINITY;
      l[nt][j] = 0.f;
#pragma unroll
      for (int i = 0; i < (kQuant ? G : 1); ++i) pm[nt][i][j] = 0.f;
    }

  int blk = beg + warp * SUB;
  int64_t row_now[SUB], row_next[SUB];
#pragma unroll
  for (int s = 0; s < SUB; ++s) {
    row_now[s] = block_row(blk + s);
    load_k(s, token0(blk + s), row_now[s]);
    load_v(s, token0(blk + s), row_now[s]);
    row_next[s] = block_row(blk + kWarps * SUB + s);
  }
  for (; blk < end; blk += kWarps * SUB) {
    const int nxt = blk + kWarps * SUB;
    // ---- scores (times log2 e) of this lane's tokens r, r + 8 and its two columns
    float s2[SUB][NT][4], sv[SUB][2][kQuant ? G : 1], mv[SUB][2][kQuant ? G : 1];
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      float t[NT][4], um[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) t[nt][i] = um[nt][i] = 0.f;
      float cg[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) cg[nt][i] = 0.f;
      constexpr int kWordsAStep = BITS == 16 ? 2 : 1;
#pragma unroll
      for (int w = 0; w < WK; w += kWordsAStep) {
        const uint32_t x = kw[s][0][w], y = kw[s][1][w];
        if constexpr (BITS == 4) {
          const uint32_t xs = x >> 8, ys = y >> 8;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma16816<false>(cg[nt], x & 0x000f000fu, y & 0x000f000fu, x & 0x00f000f0u, y & 0x00f000f0u,
                            qf[nt][2 * w][0], qf[nt][2 * w][1]);
            mma16816<false>(cg[nt], xs & 0x000f000fu, ys & 0x000f000fu, xs & 0x00f000f0u, ys & 0x00f000f0u,
                            qf[nt][2 * w + 1][0], qf[nt][2 * w + 1][1]);
          }
        } else if constexpr (BITS == 8) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            mma16816<false>(cg[nt], x & 0x00ff00ffu, y & 0x00ff00ffu, (x >> 8) & 0x00ff00ffu, (y >> 8) & 0x00ff00ffu,
                            qf[nt][w][0], qf[nt][w][1]);
        } else {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            mma16816<kBf16>(cg[nt], x, y, kw[s][0][w + 1], kw[s][1][w + 1], qf[nt][w / 2][0], qf[nt][w / 2][1]);
        }
        if constexpr (kQuant) {
          // the group's last word: fold its sum in
          const int gi = (w / VW) * 4 * VW * E / X::GROUP;
          const bool ends = w + 1 == WK || ((w + 1) / VW) * 4 * VW * E / X::GROUP != gi;
          if (ends) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint32_t pw = kp[s][i >> 1][gi];
              const float sc = __uint_as_float(pw << 16), mn = __uint_as_float(pw & 0xffff0000u);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                t[nt][i] = fmaf(sc, cg[nt][i], t[nt][i]);
                um[nt][i] = fmaf(mn, mq[nt][gi][i & 1], um[nt][i]);
                cg[nt][i] = 0.f;
              }
            }
          }
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          s2[s][nt][i] = kQuant ? fmaf(t[nt][i], fcol[nt][i & 1], um[nt][i]) : cg[nt][i] * fcol[nt][i & 1];
      // masks: only blocks at an edge of some row's range compare token by token
      const int t0 = token0(blk + s), t1 = t0 + kTok - 1;
      const bool none = row_now[s] < 0;
      const bool full = !none && t1 <= rg.p_first && t1 < rg.n &&
                        (P.mask.window == 0 || t0 >= window_lo(P.mask, rg.p_last) || t1 < P.mask.sinks);
      if (!full) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (none || !key_visible(t0 + r + 8 * (i >> 1), pcol[nt][i & 1], wlo[nt][i & 1], P.mask.sinks))
              s2[s][nt][i] = -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int gi = 0; gi < (kQuant ? G : 1); ++gi) {
          sv[s][i][gi] = kQuant ? __uint_as_float(vp[s][i][gi] << 16) : 1.f;
          mv[s][i][gi] = kQuant ? __uint_as_float(vp[s][i][gi] & 0xffff0000u) : 0.f;
        }
    }
    // the K registers are free: the next blocks' keys load while this one's softmax and values run
#pragma unroll
    for (int s = 0; s < SUB; ++s) load_k(s, token0(nxt + s), row_next[s]);

    // ---- softmax: reference = max (score + log2 of the values' scale)
    float lg[SUB][2];
#pragma unroll
    for (int s = 0; s < SUB; ++s)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        lg[s][i] = 0.f;
        if constexpr (kQuant) {
          float mx = sv[s][i][0];
#pragma unroll
          for (int gi = 1; gi < G; ++gi) mx = fmaxf(mx, sv[s][i][gi]);
          lg[s][i] = __log2f(mx);
        }
      }
    bool grew = false;
    float mnew[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float mx = -INFINITY;
#pragma unroll
        for (int s = 0; s < SUB; ++s) {
#pragma unroll
          for (int i = 0; i < 2; ++i) mx = fmaxf(mx, s2[s][nt][2 * i + j] + lg[s][i]);
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        mnew[nt][j] = fmaxf(mrun[nt][j], mx);
        grew |= mnew[nt][j] > mrun[nt][j];
      }
    if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float corr = mrun[nt][j] == -INFINITY ? 0.f : exp2_approx(mrun[nt][j] - mnew[nt][j]);
          mrun[nt][j] = mnew[nt][j];
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
    for (int s = 0; s < SUB; ++s) {
      constexpr int kLo = kBf16 ? 2 : 1;  // bf16 weights as a sum of two, so that their rounding does not show
      uint32_t bw[kQuant ? G : 1][NT][2][kLo];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float p[2];
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float x = s2[s][nt][2 * i + j];
            p[j] = x == -INFINITY ? 0.f : exp2_approx(x - mrun[nt][j]);
            l[nt][j] += p[j];
          }
#pragma unroll
          for (int gi = 0; gi < (kQuant ? G : 1); ++gi) {
            if constexpr (kQuant) {
#pragma unroll
              for (int j = 0; j < 2; ++j) pm[nt][gi][j] = fmaf(p[j], mv[s][i][gi], pm[nt][gi][j]);
            }
            const float w0 = p[0] * sv[s][i][gi], w1 = p[1] * sv[s][i][gi];
            const uint32_t hi = pack2<kBf16>(w0, w1);
            bw[gi][nt][i][0] = movmatrix_trans(hi);
            if constexpr (kBf16) {
              const float2 back = unpack2<true>(hi);
              bw[gi][nt][i][1] = movmatrix_trans(pack2<true>(w0 - back.x, w1 - back.y));
            }
          }
        }
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        const int gi = kQuant ? u * 8 * X::UB * 8 / BITS / X::GROUP : 0;
#pragma unroll
        for (int w = 0; w < UR; ++w) {
          // halves of the word: lanes' tokens (2c, 2c + 1) and (2c + 8, 2c + 9)
          const uint32_t x0 = vw[s][0][u * UR + w], x1 = vw[s][1][u * UR + w], x2 = vw[s][2][u * UR + w],
                         x3 = vw[s][3][u * UR + w];
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
                  mma16816<false>(acc[tile][nt], a & 0x00ff00ffu, (a >> 8) & 0x00ff00ffu, d & 0x00ff00ffu,
                                  (d >> 8) & 0x00ff00ffu, bw[gi][nt][0][0], bw[gi][nt][1][0]);
              } else {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                  const uint32_t as = k ? a >> 8 : a, ds = k ? d >> 8 : d;
                  const int tile = u * UT + 4 * w + 2 * hf + k;
#pragma unroll
                  for (int nt = 0; nt < NT; ++nt)
                    mma16816<false>(acc[tile][nt], as & 0x000f000fu, as & 0x00f000f0u, ds & 0x000f000fu,
                                    ds & 0x00f000f0u, bw[gi][nt][0][0], bw[gi][nt][1][0]);
                }
              }
            }
          }
        }
      }
    }
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      load_v(s, token0(nxt + s), row_next[s]);
      row_now[s] = row_next[s];
      row_next[s] = block_row(nxt + kWarps * SUB + s);
    }
  }

  // ---- join the warps: sums over the lanes of a column, then the warps in order
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int off = 4; off <= 16; off <<= 1) {
        l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], off);
        if constexpr (kQuant) {
#pragma unroll
          for (int gi = 0; gi < G; ++gi) pm[nt][gi][j] += __shfl_xor_sync(0xffffffffu, pm[nt][gi][j], off);
        }
      }
      if (r == 0) ml[warp][8 * nt + 2 * c + j] = make_float2(mrun[nt][j], l[nt][j]);
    }
  __syncthreads();
  for (int w = 0; w < kWarps; ++w) {
    if (warp == w) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int col = 8 * nt + 2 * c + j;
          float ref = -INFINITY;
#pragma unroll
          for (int v = 0; v < kWarps; ++v) ref = fmaxf(ref, ml[v][col].x);
          const float f = mrun[nt][j] == -INFINITY ? 0.f : exp2_approx(mrun[nt][j] - ref);
#pragma unroll
          for (int t = 0; t < X::TILES; ++t) {
            const int u = t / UT, in_u = t % UT;
            const int d = BITS == 16 ? (u * 8 + r) * X::UB / 2 + 2 * in_u : (u * 8 + r) * X::UB * 8 / BITS + 2 * in_u;
            const int gi = kQuant ? u * 8 * X::UB * 8 / BITS / X::GROUP : 0;
            const float up = kQuant ? 0x1p24f : 1.f, up1 = BITS == 4 ? 0x1p20f : up;
            const float x = fmaf(acc[t][nt][j], up, pm[nt][gi][j]) * f;
            const float y = fmaf(acc[t][nt][2 + j], up1, pm[nt][gi][j]) * f;
            if (w == 0) {
              buf[col][d] = x;
              buf[col][d + 1] = y;
            } else {
              buf[col][d] += x;
              buf[col][d + 1] += y;
            }
          }
        }
    }
    __syncthreads();
  }
  // ---- out: the row's result, or this split's part of it
  const int64_t part = ((static_cast<int64_t>(b) * P.Hkv + hk) * A.row_blocks + rb) * A.splits + split;
  for (int col = warp; col < 8 * NT; col += kWarps) {
    const int R = row0 + col;
    if (R >= rows) break;
    float ref = -INFINITY, sum = 0.f;
#pragma unroll
    for (int v = 0; v < kWarps; ++v) ref = fmaxf(ref, ml[v][col].x);
#pragma unroll
    for (int v = 0; v < kWarps; ++v)
      sum += ml[v][col].x == -INFINITY ? ml[v][col].y * 0.f : ml[v][col].y * exp2_approx(ml[v][col].x - ref);
    if (A.splits == 1) {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      const int64_t at = row_at(P.o, b, hk, g, R);
      bool bad = false;
      for (int d = lane; d < D; d += 32) {
        const float x = buf[col][d] * inv;
        bad |= !isfinite(x);
        store_o(P.o.p, at + d, P.dtype, x);
      }
      if constexpr (!kQuant) {
        // several queries: a value row of another query's range may hold an infinity or NaN
        if (rg.m > 1 && __any_sync(0xffffffffu, bad)) {
          using T = typename std::conditional<kBf16, __nv_bfloat16, __half>::type;
          const int pos = rg.p_first + R / g;
          __syncwarp();
          attention_row<T>(static_cast<const T *>(P.q.p) + row_at(P.q, b, hk, g, R), reinterpret_cast<const T *>(kbase),
                           reinterpret_cast<const T *>(vbase), static_cast<T *>(P.o.p) + at, P.k.sl, P.v.sl, D, pos,
                           window_lo(P.mask, pos), P.mask.sinks, P.scale * kLog2e);
        }
      }
    } else {
      for (int d = lane; d < D; d += 32) A.part_o[(part * 8 * NT + col) * D + d] = buf[col][d];
      if (lane == 0) A.part_ml[part * 8 * NT + col] = make_float2(ref, sum);
    }
  }
}

// Joins the splits of a row: one warp a row, splits in order.
template <int D, bool kBf16, bool kDense>
__global__ void __launch_bounds__(kThreads) combine_kernel(const Params A, int nrows) {
  const AttnProblem &P = A.p;
  const int lane = threadIdx.x & 31, g = P.H / P.Hkv;
  const int rows_all = g * P.mask.Lq;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  pdl_launch_dependents();
  pdl_wait();
  const int R = static_cast<int>(id % rows_all);
  const int64_t bh = id / rows_all;
  const int hk = static_cast<int>(bh % P.Hkv);
  if (bh / P.Hkv >= P.B) return;
  const int b = static_cast<int>(bh / P.Hkv);
  int n, m;
  seq_lens(P.mask, b, n, m);
  if (R >= g * m) return;
  const int64_t part0 = (bh * A.row_blocks + R / nrows) * A.splits;
  const int col = R % nrows;
  float ref = -INFINITY;
  for (int s = lane; s < A.splits; s += 32) ref = fmaxf(ref, A.part_ml[(part0 + s) * nrows + col].x);
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) ref = fmaxf(ref, __shfl_xor_sync(0xffffffffu, ref, off));
  constexpr int kPer = (D + 31) / 32;
  float acc[kPer], sum = 0.f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) acc[i] = 0.f;
  for (int s = 0; s < A.splits; ++s) {
    const float2 t = A.part_ml[(part0 + s) * nrows + col];
    if (t.x == -INFINITY && t.y == 0.f) continue;  // an empty split
    const float f = t.x == -INFINITY ? 0.f : exp2_approx(t.x - ref);
    sum = fmaf(t.y, f, sum);
    const float *src = A.part_o + ((part0 + s) * nrows + col) * D;
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (lane + 32 * i < D) acc[i] = fmaf(src[lane + 32 * i], f, acc[i]);
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int64_t at = row_at(P.o, b, hk, g, R);
  bool bad = false;
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (lane + 32 * i < D) {
      const float x = acc[i] * inv;
      bad |= !isfinite(x);
      store_o(P.o.p, at + lane + 32 * i, P.dtype, x);
    }
  if constexpr (kDense) {
    if (m > 1 && __any_sync(0xffffffffu, bad)) {
      using T = typename std::conditional<kBf16, __nv_bfloat16, __half>::type;
      const int pos = n - m + R / g;
      __syncwarp();
      attention_row<T>(static_cast<const T *>(P.q.p) + row_at(P.q, b, hk, g, R),
                       static_cast<const T *>(P.k.p) + b * P.k.sb + hk * P.k.sh,
                       static_cast<const T *>(P.v.p) + b * P.v.sb + hk * P.v.sh, static_cast<T *>(P.o.p) + at, P.k.sl,
                       P.v.sl, D, pos, window_lo(P.mask, pos), P.mask.sinks, P.scale * kLog2e);
    }
  }
}

template <int BITS, int D, int G, bool kBf16, int NT>
cudaError_t launch_split(const Params &a, cudaStream_t stream) {
  // blocks in flight a warp: about 4 KB of codes
  constexpr int SUB = D * BITS <= 512 ? 2 : 1;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(a.splits), static_cast<unsigned>(a.p.Hkv * a.row_blocks),
                     static_cast<unsigned>(a.p.B));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, split_kernel<BITS, D, G, kBf16, NT, SUB>, a);
  if (e == cudaSuccess && a.splits > 1) {
    const int64_t rows = static_cast<int64_t>(a.p.B) * a.p.H * a.p.mask.Lq;
    cfg.gridDim = dim3(static_cast<unsigned>((rows + kWarps - 1) / kWarps));
    e = cudaLaunchKernelEx(&cfg, combine_kernel<D, kBf16, BITS == 16>, a, 8 * NT);
  }
  return e != cudaSuccess ? e : cudaGetLastError();
}

// Query rows of a block: one n = 8 tile, or two where a key head has more
// rows than that and the accumulators leave registers for it.
constexpr int row_tiles(int rows, int D) { return rows > 8 && D <= 128 ? 2 : 1; }

cudaError_t launch_dense(const Params &a, cudaStream_t stream);  // kv_attention_dense.cu

}  // namespace split_attn
}  // namespace llk_b200
