// attn_common.cuh -- device helpers the serving attention kernels share: the
// element types, a sequence's visible key ranges, and the row-by-row form of
// the operator that a kernel falls back on for a row whose result a value that
// it does not see may have made non-finite.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <type_traits>

#include "kv_kernels.h"
#include "llk_b200.h"
#include "sm100_ptx.cuh"

namespace llk_b200 {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// 2^x, 2 ulp (MUFU); exp2_approx(-inf) = 0.
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A mean of finite f16 values by weights that were rounded to 16 bits: not past
// the largest f16, which rounding would make an infinity.
__device__ __forceinline__ float within_f16(float x) {
  return fabsf(x) < INFINITY ? fminf(fmaxf(x, -65504.f), 65504.f) : x;
}

// Keys n and queries m of sequence b, clamped to the tensors.
__device__ __forceinline__ void seq_lens(const AttnMask &mk, int b, int &n, int &m) {
  n = mk.kv_lens ? mk.kv_lens[b] : mk.Lk;
  m = mk.q_lens ? mk.q_lens[b] : mk.Lq;
  n = n < 0 ? 0 : (n > mk.Lk ? mk.Lk : n);
  m = m < 0 ? 0 : (m > mk.Lq ? mk.Lq : m);
}

// First key of the window of a query at position p (0 without a window).
__device__ __forceinline__ int window_lo(const AttnMask &mk, int p) {
  return mk.window > 0 && p >= mk.window ? p - mk.window + 1 : 0;
}

__device__ __forceinline__ bool key_visible(int j, int p, int lo, int sinks) {
  return j <= p && (j >= lo || j < sinks);
}

// ---- Rows whose result is not finite.  The tiled kernels multiply a masked
// weight 0 with the value row of its tile, which is wrong where that row holds
// an infinity or NaN.  They find it by the non-finite result; but a row that
// sees such a value itself, or has a NaN among its own scores, is not finite by
// right, and there can be as many of those as there are queries.  So a row is
// redone (attention_row) only where one of the keys that it does not see and
// its tiles hold has a value that is not finite: those keys lie behind its
// position or in front of its window, and there are no more of them than a tile
// has queries (and keys).

template <typename T>
__device__ __forceinline__ bool not_finite(T x, bool inf) {  // inf: only infinities
  const float f = fabsf(to_f32(x));
  return inf ? f == INFINITY : !(f < INFINITY);
}

// The first of the rows from, from + step, .. (count of them, step 1 or -1) of
// v that holds a value that is not finite (inf: an infinity), or -1.  By one warp.
template <typename T>
__device__ __noinline__ int bad_row(const T *v, int64_t v_sl, int D, int from, int count, int step, bool inf) {
  constexpr int kAt = 8, kVec = 16 / sizeof(T), kNone = 0x7fffffff;
  const int lane = threadIdx.x & 31;
  // pieces of a row, 16 bytes where rows start there, and rows of a round of kAt pieces a lane
  const bool vec = ((reinterpret_cast<uintptr_t>(v) | v_sl * sizeof(T) | D * sizeof(T)) & 15) == 0;
  const int pieces = vec ? D / kVec : D, rows = 32 * kAt / pieces;  // (D <= 256: a row at least)
  int row[kAt];
  const T *at[kAt];
#pragma unroll
  for (int u = 0; u < kAt; ++u) {
    const int c = lane + 32 * u;
    row[u] = c / pieces < rows ? c / pieces : kNone;
    at[u] = v + static_cast<int64_t>(from + (row[u] < rows ? row[u] : 0) * step) * v_sl + c % pieces * (vec ? kVec : 1);
  }
  for (int j = 0; j < count; j += rows) {
    int found = kNone;
    uint4 x[kAt];
#pragma unroll
    for (int u = 0; u < kAt; ++u) {
      x[u] = make_uint4(0, 0, 0, 0);
      if (row[u] < count - j) {
        if (vec) {
          x[u] = *reinterpret_cast<const uint4 *>(at[u]);
        } else {
          *reinterpret_cast<T *>(&x[u]) = *at[u];
        }
      }
      at[u] += static_cast<int64_t>(rows) * step * v_sl;
    }
#pragma unroll
    for (int u = 0; u < kAt; ++u) {
      const T *e = reinterpret_cast<const T *>(&x[u]);
      bool bad = false;
#pragma unroll
      for (int i = 0; i < kVec; ++i) bad |= not_finite(e[i], inf);
      if (bad && j + row[u] < found) found = j + row[u];
    }
    found = __reduce_min_sync(0xffffffffu, found);
    if (found != kNone) return from + found * step;
  }
  return -1;
}

// What of the values hidden from a warp's rows is not finite: the last of the
// keys behind the first row's position p0 (before hi), and the first of those
// from `from` to before the last row's window, last_lo; -1 for none.
struct HiddenBad {
  int late, early;
  // whether a row at position p with its window from lo may have met one
  __device__ __forceinline__ bool meets(int p, int lo) const {
    return (late >= 0 && late > p) || (early >= 0 && early < lo);
  }
};
template <typename T>
__device__ __forceinline__ HiddenBad hidden_bad(const T *v, int64_t v_sl, int D, int p0, int hi, int from,
                                                int last_lo) {
  const int first = p0 + 1 > 0 ? p0 + 1 : 0;
  HiddenBad b;
  b.late = hi > first ? bad_row(v, v_sl, D, hi - 1, hi - first, -1, false) : -1;
  b.early = last_lo > from ? bad_row(v, v_sl, D, from, last_lo - from, 1, false) : -1;
  return b;
}

// The same for one row at position p of a sequence of n keys and m queries whose
// window begins at lo: whether it is to be redone.  k16: the tiles' weights were
// one f16 or a sum of two numbers, and one that is 0 there (or a sum of either
// sign) times an infinity that the row does see is NaN, not so by the
// definition.
template <typename T, bool k16>
__device__ __forceinline__ bool redo_row(const T *v, int64_t v_sl, const AttnMask &mk, int D, int n, int m, int p,
                                         int lo, bool nan) {
  const int first = window_lo(mk, n - m);
  if (hidden_bad<T>(v, v_sl, D, p, n, first > mk.sinks ? first : mk.sinks, lo).meets(p, lo)) return true;
  if (!k16 || !nan) return false;
  const int s_end = mk.sinks < lo ? mk.sinks : lo, end = p + 1 > 0 ? p + 1 : 0;
  return bad_row<T>(v, v_sl, D, 0, s_end < end ? s_end : end, 1, true) >= 0 ||
         bad_row<T>(v, v_sl, D, lo, end - lo, 1, true) >= 0;
}

// A 16-byte piece as f32.
template <typename T>
__device__ __forceinline__ float piece_at(const uint4 &x, int i) {
  return to_f32(reinterpret_cast<const T *>(&x)[i]);
}

// One query row, one warp, straight from the definition; keys that the row
// does not see are not touched.  D <= 256.  o holds the tiles' result: where all
// of it that is not finite is NaN by the row's own token, it stands (values that
// are NaN throughout would have every row redone).
//
// 32 keys at a time: a lane has the score of one, then a 16-byte piece of every
// (32 / pieces)-th value row; what rows are not made of such pieces goes element
// by element.  Latency is all there is to it (a warp alone, many loads ahead).
template <typename T>
__device__ __noinline__ void attention_row(const T *q, const T *k, const T *v, T *o, int64_t k_sl, int64_t v_sl, int D,
                                           int p, int lo, int sinks, float scale_log2) {
  constexpr int kVec = 16 / sizeof(T), kAt = 8;
  const int lane = threadIdx.x & 31;
  bool needed = p < 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = lane + 32 * i;
    if (p >= 0 && d < D && not_finite(o[d], false)) needed |= !isnan(to_f32(v[p * v_sl + d]));
  }
  if (!__any_sync(0xffffffffu, needed)) return;
  const int pieces = D / kVec;
  const bool vec = ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
                     k_sl * sizeof(T) | v_sl * sizeof(T) | D * sizeof(T)) & 15) == 0 && pieces <= 32;
  // a lane's piece, and its first row of the rows that the warp reads at once
  const int at_once = vec ? 32 / pieces : 1, mine = vec ? lane % pieces : 0, row0 = vec ? lane / pieces : 0;
  float acc[8], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.f;
  // the keys 0 .. min(sinks, lo) - 1, then lo .. p, in chunks of 32
  const int s_end = sinks < lo ? sinks : lo;
  for (int part = 0; part < 2; ++part) {
    const int first = part == 0 ? 0 : lo, end = part == 0 ? (s_end < p + 1 ? s_end : p + 1) : p + 1;
    for (int j0 = first; j0 < end; j0 += 32) {
      const int j = j0 + lane, cnt = end - j0 < 32 ? end - j0 : 32;
      auto value_rows = [&](int t0, uint4 (&x)[kAt]) {  // kAt of this lane's value rows, from the t0-th on
#pragma unroll
        for (int u = 0; u < kAt; ++u) {
          const int t = (t0 + u) * at_once + row0;
          x[u] = make_uint4(0, 0, 0, 0);
          if (row0 < at_once && t < cnt)
            x[u] = *reinterpret_cast<const uint4 *>(v + static_cast<int64_t>(j0 + t) * v_sl + mine * kVec);
        }
      };
      uint4 vx[kAt];
      if (vec) value_rows(0, vx);
      float s = -INFINITY;
      if (j < end) {
        const T *kr = k + static_cast<int64_t>(j) * k_sl;
        s = 0.f;
        if (vec) {
          for (int c0 = 0; c0 < pieces; c0 += kAt) {
            uint4 x[kAt], y[kAt];
#pragma unroll
            for (int u = 0; u < kAt; ++u) {
              const int c = c0 + u < pieces ? c0 + u : c0;
              x[u] = *reinterpret_cast<const uint4 *>(q + c * kVec);
              y[u] = *reinterpret_cast<const uint4 *>(kr + c * kVec);
            }
#pragma unroll
            for (int u = 0; u < kAt; ++u)
              if (c0 + u < pieces)
#pragma unroll
                for (int i = 0; i < kVec; ++i) s = fmaf(piece_at<T>(x[u], i), piece_at<T>(y[u], i), s);
          }
        } else {
          for (int d = 0; d < D; ++d) s = fmaf(to_f32(q[d]), to_f32(kr[d]), s);
        }
        s *= scale_log2;
      }
      float mx = s;
#pragma unroll
      for (int off = 16; off >= 1; off >>= 1) {
        const float t = __shfl_xor_sync(0xffffffffu, mx, off);
        mx = (mx != mx || t != t) ? NAN : fmaxf(mx, t);
      }
      const float m_new = (mx != mx || m != m) ? NAN : fmaxf(m, mx);
      const float corr = m == -INFINITY ? 0.f : exp2f(m - m_new);
      const float pj = s == -INFINITY ? 0.f : exp2f(s - m_new);
      l = fmaf(l, corr, pj);  // of this lane's keys
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] *= corr;
      if (vec) {
        for (int t0 = 0; t0 * at_once < cnt; t0 += kAt) {
          if (t0 > 0) value_rows(t0, vx);
#pragma unroll
          for (int u = 0; u < kAt; ++u) {
            const int t = (t0 + u) * at_once + row0;
            const float pt = __shfl_sync(0xffffffffu, pj, t & 31);
            if (row0 < at_once && t < cnt)
#pragma unroll
              for (int i = 0; i < kVec; ++i) acc[i] = fmaf(pt, piece_at<T>(vx[u], i), acc[i]);
          }
        }
      } else {
        for (int t = 0; t < cnt; ++t) {
          const float pt = __shfl_sync(0xffffffffu, pj, t);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int d = lane + 32 * i;
            if (d < D) acc[i] = fmaf(pt, to_f32(v[static_cast<int64_t>(j0 + t) * v_sl + d]), acc[i]);
          }
        }
      }
      m = m_new;
    }
  }
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
  if (vec) {
    // the lanes that share a piece, in order of their rows
    for (int r = 1; r < at_once; ++r)
#pragma unroll
      for (int i = 0; i < kVec; ++i) {
        const float x = __shfl_sync(0xffffffffu, acc[i], (mine + r * pieces) & 31);
        if (row0 == 0) acc[i] += x;
      }
    if (row0 == 0)
#pragma unroll
      for (int i = 0; i < kVec; ++i) o[mine * kVec + i] = from_f32<T>(l == 0.f ? 0.f : acc[i] / l);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int d = lane + 32 * i;
      if (d < D) o[d] = from_f32<T>(l == 0.f ? 0.f : acc[i] / l);
    }
  }
}

}  // namespace llk_b200
