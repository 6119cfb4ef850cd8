// attn_common.cuh -- device helpers the serving attention kernels share: the
// element types, a sequence's visible key ranges, and the row-by-row form of
// the operator that a kernel falls back on for a row whose result is not
// finite.
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

// One query row, one warp, straight from the definition; keys that the row
// does not see are not touched.  The tiled kernels multiply a masked weight 0
// with the value row of its tile, which is wrong only where that row holds an
// infinity or NaN: they find it by the non-finite result and redo the row
// here.  D <= 256.
template <typename T>
__device__ __noinline__ void attention_row(const T *q, const T *k, const T *v, T *o, int64_t k_sl, int64_t v_sl, int D,
                                           int p, int lo, int sinks, float scale_log2) {
  const int lane = threadIdx.x & 31;
  float acc[8], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.f;
  // the keys 0 .. min(sinks, lo) - 1, then lo .. p, in chunks of 32
  const int s_end = sinks < lo ? sinks : lo;
  for (int part = 0; part < 2; ++part) {
    const int first = part == 0 ? 0 : lo, end = part == 0 ? (s_end < p + 1 ? s_end : p + 1) : p + 1;
    for (int j0 = first; j0 < end; j0 += 32) {
      const int j = j0 + lane;
      float s = -INFINITY;
      if (j < end) {
        s = 0.f;
        for (int d = 0; d < D; ++d) s = fmaf(to_f32(q[d]), to_f32(k[j * k_sl + d]), s);
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
      l = l * corr;
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] *= corr;
      const int cnt = end - j0 < 32 ? end - j0 : 32;
      for (int t = 0; t < cnt; ++t) {
        const float pt = __shfl_sync(0xffffffffu, pj, t);
        l += pt;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int d = lane + 32 * i;
          if (d < D) acc[i] = fmaf(pt, to_f32(v[(j0 + t) * v_sl + d]), acc[i]);
        }
      }
      m = m_new;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = lane + 32 * i;
    if (d < D) o[d] = from_f32<T>(l == 0.f ? 0.f : acc[i] / l);
  }
}

}  // namespace llk_b200
