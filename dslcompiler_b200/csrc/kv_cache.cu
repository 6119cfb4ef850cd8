// kv_cache.cu -- the quantised paged KV cache's writer and reader.
//
// A token's key or value of one head, x [D], is held in groups of `group`
// elements.  With x saturated to +-65504 and NaN counted as 0, per group
//   m = bf16(min x),   s = bf16(f32(max((max x - m) / (2^bits - 1), 2^-30))),
//   code = clamp(rint((x - m) / s), 0, 2^bits - 1)  (ties to even),
// both quotients as in 64 bits; the group stands for s * code + m.  With 4
// bits the elements 2j and 2j + 1 share byte j (2j in the low nibble).
//
// HBM-bound both ways; what there is to save is instructions.  A thread owns
// 16 elements of a row, a row is D / 16 neighbouring lanes.  A CTA first works
// out where its tokens lie, once for all heads.  Writing: the group's minimum
// and maximum are packed 16-bit operations and shuffles of the pair (min, -max);
// the quotient (x - m) / s is a product with 1 / s and one correction by its remainder, which makes it
// exact wherever the quotient is a tie between two codes (the remainder is
// exact, and so is the corrected quotient when it is representable), so
// rounding to even by adding 1.5 * 2^23 settles the ties of 16-bit inputs;
// quotients nearer to a tie than the f32 error without surely being one go by the
// sign of x - m - (k + 1/2) s.  Codes are put together as f32 sums (exact below
// 2^24), two chains at a time in packed f32 operations.  Reading: a nibble is
// masked into the mantissa of 2^23 where it lies, so that a subtraction makes
// it code * 16^i, and one fused multiply-add with scale / 16^i the value.
//
// Measured at 1965 MHz, 4 x 8191 bf16 tokens of 8 heads, D = 128, 4 bits: write
// 78 us (7 of them the look for repeated slots), read 34 us, each 170 MB, 26 us
// at the measured HBM rate.  The write issues an instruction in 70 % of the
// clocks: 420 of them a warp for 16 elements a lane.  32 tokens: 3.2 and 2.2 us,
// a launch.  2000 f32 tokens of 32 heads, D = 64, 8 bits: 16 and 8 us.
#include <cuda.h>
#include <cuda_runtime.h>

#include "attn_common.cuh"

namespace llk_b200 {

namespace {

constexpr int kThreads = 256;
constexpr int kCtas = 4;              // resident on an SM: 64 registers
constexpr int kMaxTokens = 64;        // tokens of a writer's CTA
// Tokens of a writer's launch: the look for repeated slots is 7 of 78 us there
// (8 heads of 128), what splitting further would save goes into more launches.
constexpr int64_t kMaxLaunch = 32768;
constexpr int kBitmapWords = 1024;    // 32768 bits over the low bits of the CTA's slots, as many over a hash
constexpr float kLargest = 65504.f;
constexpr double kLeastScale = 0x1p-30;

__device__ __forceinline__ uint64_t f32x2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 split2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

// A thread's elements of a row, as they lie.
constexpr int kN = 16;
template <typename T>
struct Piece {
  uint32_t w[kN * sizeof(T) / 4];
};

template <typename T>
__device__ __forceinline__ void load_piece(const T *src, bool vec, Piece<T> &x) {
  if (vec) {
#pragma unroll
    for (int i = 0; i < kN * static_cast<int>(sizeof(T)) / 16; ++i) {
      const uint4 v = __ldcs(reinterpret_cast<const uint4 *>(src) + i);
      x.w[4 * i] = v.x;
      x.w[4 * i + 1] = v.y;
      x.w[4 * i + 2] = v.z;
      x.w[4 * i + 3] = v.w;
    }
  } else if constexpr (sizeof(T) == 2) {
    const uint16_t *e = reinterpret_cast<const uint16_t *>(src);
#pragma unroll
    for (int i = 0; i < kN / 2; ++i) x.w[i] = e[2 * i] | static_cast<uint32_t>(e[2 * i + 1]) << 16;
  } else {
#pragma unroll
    for (int i = 0; i < kN; ++i) x.w[i] = __float_as_uint(src[i]);
  }
}

template <typename T>
__device__ __forceinline__ float element(const Piece<T> &x, int i) {
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(x.w[i]);
  } else if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = *reinterpret_cast<const __half2 *>(&x.w[i / 2]);
    return i % 2 ? __high2float(h) : __low2float(h);
  } else {
    return __uint_as_float(i % 2 ? x.w[i / 2] & 0xffff0000u : x.w[i / 2] << 16);
  }
}

// 8 values to 8 elements.
template <typename T>
__device__ __forceinline__ void store8(T *dst, bool vec, const float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    if (vec) {
      reinterpret_cast<float4 *>(dst)[0] = make_float4(x[0], x[1], x[2], x[3]);
      reinterpret_cast<float4 *>(dst)[1] = make_float4(x[4], x[5], x[6], x[7]);
      return;
    }
  } else if (vec) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __half>::value) {
        asm("cvt.rn.f16x2.f32 %0, %2, %1;" : "=r"(w[i]) : "f"(x[2 * i]), "f"(x[2 * i + 1]));
      } else {
        asm("cvt.rn.bf16x2.f32 %0, %2, %1;" : "=r"(w[i]) : "f"(x[2 * i]), "f"(x[2 * i + 1]));
      }
    }
    *reinterpret_cast<uint4 *>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) dst[i] = from_f32<T>(x[i]);
}

__device__ __forceinline__ float saturate(float v) { return v != v ? 0.f : fminf(fmaxf(v, -kLargest), kLargest); }

// Smallest and largest of a group over the gl lanes that share it; NaN if it
// holds one.
template <typename T>
__device__ __forceinline__ float2 group_range(const Piece<T> &x, int gl) {
  if constexpr (sizeof(T) == 2) {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    const T2 *p = reinterpret_cast<const T2 *>(x.w);
    T2 mn = p[0], mx = p[0];
#pragma unroll
    for (int i = 1; i < kN / 2; ++i) {
      mn = __hmin2_nan(mn, p[i]);
      mx = __hmax2_nan(mx, p[i]);
    }
    // both halves' minima with both halves' negated maxima
    mx = __hneg2(mx);
    const uint32_t a = *reinterpret_cast<const uint32_t *>(&mn), b = *reinterpret_cast<const uint32_t *>(&mx);
    const uint32_t lo = __byte_perm(a, b, 0x5410), hi = __byte_perm(a, b, 0x7632);
    T2 r = __hmin2_nan(*reinterpret_cast<const T2 *>(&lo), *reinterpret_cast<const T2 *>(&hi));
#pragma unroll
    for (int off = 1; off < 8; off <<= 1) {
      const uint32_t o = __shfl_xor_sync(0xffffffffu, *reinterpret_cast<const uint32_t *>(&r), off);
      const T2 both = __hmin2_nan(r, *reinterpret_cast<const T2 *>(&o));
      if (off < gl) r = both;
    }
    return make_float2(to_f32(r.x), -to_f32(r.y));
  } else {
    float mn = INFINITY, mx = -INFINITY;
    bool nan = false;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const float f = __uint_as_float(x.w[i]);
      mn = fminf(mn, f);
      mx = fmaxf(mx, f);
      nan |= f != f;
    }
    if (nan) mn = NAN;
#pragma unroll
    for (int off = 1; off < 8; off <<= 1) {
      const float a = __shfl_xor_sync(0xffffffffu, mn, off), c = __shfl_xor_sync(0xffffffffu, mx, off);
      if (off < gl) {
        mn = a != a || mn != mn ? NAN : fminf(mn, a);
        mx = fmaxf(mx, c);
      }
    }
    return make_float2(mn, mx);
  }
}

// Whether x - m is exact for every x of the piece, 16-bit: 8 bits (f16: 11)
// and m's 8 no more than 24 bits apart, or one of them 0.  Magnitudes compare
// as their bits do; less one, a 0 becomes the largest.
template <typename T>
__device__ __forceinline__ bool exact_differences(const Piece<T> &x, float m, float largest) {
  constexpr float kApart = std::is_same<T, __half>::value ? 0x1p-11f : 0x1p-14f;
  uint32_t least = 0xffffffffu;
#pragma unroll
  for (int i = 0; i < kN / 2; ++i) least = __viaddmin_u16x2(x.w[i] & 0x7fff7fffu, 0xffffffffu, least);
  // of both halves, and one back (all zero: 0xffff + 1 has no 16 bits, and is larger than any)
  const uint32_t bits = min(least & 0xffffu, least >> 16) + 1;
  const float am = fabsf(m);
  if (bits > 0xffffu || am == 0.f) return true;
  const unsigned short us = static_cast<unsigned short>(bits);
  const float small = to_f32(*reinterpret_cast<const T *>(&us));
  return small >= am * kApart && am >= largest * kApart;
}

// scale = bf16(f32(max((mx - m) / top, 2^-30))), the quotient as in 64 bits: in
// f32 first, in f64 where that lies next to the middle of two bf16.
template <int BITS>
__device__ __forceinline__ __nv_bfloat16 scale_of(float mx, float m) {
  constexpr float kTop = static_cast<float>((1 << BITS) - 1);
  const float q = (mx - m) * (1.f / kTop);
  if (q > 0x1p-29f && abs(static_cast<int>(__float_as_uint(q) & 0xffffu) - 0x8000) > 8) return __float2bfloat16_rn(q);
  const double d = (static_cast<double>(mx) - static_cast<double>(m)) / static_cast<double>(kTop);
  return __float2bfloat16_rn(static_cast<float>(d < kLeastScale ? kLeastScale : d));
}

// Codes of a thread's elements (packed: words of the row) and its group's
// (scale, min), from the group's (smallest, largest).  kWild: some element of
// the warp is not finite or too large, and each saturates.
template <typename T, int BITS, bool kWild>
__device__ __forceinline__ void quantise_in(const Piece<T> &raw, float2 range, uint32_t (&words)[kN * BITS / 32],
                                            uint32_t *param) {
  constexpr float kTop = static_cast<float>((1 << BITS) - 1);
  constexpr float kRound = 12582912.f;  // 1.5 * 2^23
  auto x = [&](int i) {
    const float v = element(raw, i);
    return kWild ? saturate(v) : v;
  };
  const __nv_bfloat16 mb = __float2bfloat16_rn(range.x);
  const float m = __bfloat162float(mb);
  const __nv_bfloat16 sb = scale_of<BITS>(range.y, m);
  const float s = __bfloat162float(sb);
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
  *param = static_cast<uint32_t>(__bfloat16_as_ushort(sb)) | (static_cast<uint32_t>(__bfloat16_as_ushort(mb)) << 16);
  const uint64_t m2 = f32x2(-m, -m), inv2 = f32x2(inv, inv), s2 = f32x2(-s, -s), round2 = f32x2(kRound, kRound),
                 unround2 = f32x2(-kRound, -kRound), one2 = f32x2(-1.f, -1.f);
  // error of the corrected quotient: an ulp or two of at most 2^BITS + 1 (and of x - m, 2^-24 of it)
  constexpr float kNear = static_cast<float>(1 << BITS) * 0x1p-22f, kLo = (0.5f - kNear) * (0.5f - kNear);
  // the squared distance to the code: (kLo, 1/4) iff within kHalf of kMid (with a margin, so that 1/4 itself is not)
  constexpr float kMid = (kLo + 0.25f) / 2, kHalf = (0.25f - kLo) * 0.49f;
  const uint64_t mid2 = f32x2(-kMid, -kMid);
  uint64_t k[kN / 2];  // codes of the elements 8 h + i and 8 h + i + 4 in k[4 h + i]
  bool near = false;
#pragma unroll
  for (int p = 0; p < kN / 2; ++p) {
    const int e = p / 4 * 8 + p % 4;
    const uint64_t d = add2(f32x2(x(e), x(e + 4)), m2);
    uint64_t q = mul2(d, inv2);
    q = fma2(fma2(q, s2, d), inv2, q);
    // (a lower bound only where m may lie above the smallest element: bf16
    // elements are their own bf16 minimum, but a saturated one, 65504, is not a
    // bf16; an upper one only where the scale's rounding can push the largest
    // past the top)
    constexpr bool kLow = kWild || !std::is_same<T, __nv_bfloat16>::value, kHigh = BITS == 8;
    if constexpr (kLow || kHigh) {
      float2 c = split2(q);
      if constexpr (kLow) c = make_float2(fmaxf(c.x, 0.f), fmaxf(c.y, 0.f));
      if constexpr (kHigh) c = make_float2(fminf(c.x, kTop), fminf(c.y, kTop));
      q = f32x2(c.x, c.y);
    }
    k[p] = add2(add2(q, round2), unround2);
    const uint64_t r = fma2(k[p], one2, q);
    if constexpr (sizeof(T) == 2) {
      // a tie (1/4) is settled where x - m is exact, see below
      const float2 v = split2(fma2(r, r, mid2));
      near |= fabsf(v.x) < kHalf || fabsf(v.y) < kHalf;
    } else {
      const float2 v = split2(mul2(r, r));
      near |= v.x > kLo || v.y > kLo;
    }
  }
  if constexpr (sizeof(T) == 2) near |= !exact_differences(raw, m, fmaxf(fabsf(range.y), fabsf(m)));
  if (near) {
#pragma unroll
    for (int p = 0; p < kN / 2; ++p) {
      float c[2];
      const float2 kk = split2(k[p]);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        // x - m = d + e exactly; against the border on the quotient's side of k
        const float xi = x(p / 4 * 8 + p % 4 + 4 * j), d = xi - m, t = d - xi, e = (xi - (d - t)) - (m + t);
        const float k0 = j ? kk.y : kk.x, q = d * inv;
        const float lo = q < k0 ? k0 - 1.f : k0;  // the border between lo and lo + 1
        const float side = fmaf(-(lo + 0.5f), s, d) + e;
        c[j] = side > 0.f || (side == 0.f && (static_cast<int>(lo) & 1)) ? lo + 1.f : lo;
        c[j] = fminf(fmaxf(c[j], 0.f), kTop);
      }
      k[p] = f32x2(c[0], c[1]);
    }
  }
  const uint64_t base2 = f32x2(0x1p23f, 0x1p23f);
#pragma unroll
  for (int h = 0; h < kN / 8; ++h) {
    const uint64_t *kh = k + 4 * h;
    if constexpr (BITS == 4) {
      const uint64_t by16 = f32x2(16.f, 16.f);
      const uint64_t c = add2(fma2(fma2(fma2(kh[3], by16, kh[2]), by16, kh[1]), by16, kh[0]), base2);
      words[h] = __byte_perm(static_cast<uint32_t>(c), static_cast<uint32_t>(c >> 32), 0x5410);
    } else {
      const uint64_t by256 = f32x2(256.f, 256.f);
      const uint64_t c0 = add2(fma2(kh[1], by256, kh[0]), base2), c1 = add2(fma2(kh[3], by256, kh[2]), base2);
      words[2 * h] = __byte_perm(static_cast<uint32_t>(c0), static_cast<uint32_t>(c1), 0x5410);
      words[2 * h + 1] = __byte_perm(static_cast<uint32_t>(c0 >> 32), static_cast<uint32_t>(c1 >> 32), 0x5410);
    }
  }
}

template <typename T, int BITS>
__device__ __forceinline__ void quantise(const Piece<T> &raw, int gl, uint32_t (&words)[kN * BITS / 32],
                                         uint32_t *param) {
  float2 range = group_range(raw, gl);
  if (!__any_sync(0xffffffffu, !(range.x >= -kLargest && range.y <= kLargest))) {
    quantise_in<T, BITS, false>(raw, range, words, param);
    return;
  }
  float mn = INFINITY, mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < kN; ++i) {
    const float v = saturate(element(raw, i));
    mn = fminf(mn, v);
    mx = fmaxf(mx, v);
  }
#pragma unroll
  for (int off = 1; off < 8; off <<= 1) {
    const float a = __shfl_xor_sync(0xffffffffu, mn, off), c = __shfl_xor_sync(0xffffffffu, mx, off);
    if (off < gl) {
      mn = fminf(mn, a);
      mx = fmaxf(mx, c);
    }
  }
  quantise_in<T, BITS, true>(raw, make_float2(mn, mx), words, param);
}

// 8 values from their codes; si[i] = (scale / 2^(BITS i)) twice, m2 = min twice.
template <int BITS>
__device__ __forceinline__ void values8(const uint32_t *words, const uint64_t *si, uint64_t m2, float (&x)[8]) {
  const uint64_t base2 = f32x2(-0x1p23f, -0x1p23f);
  constexpr int kIn = 16 / BITS;  // codes of a 16-bit half word
#pragma unroll
  for (int h = 0; h < BITS / 4; ++h) {
    const uint32_t w = words[h], v = w >> 16;
#pragma unroll
    for (int i = 0; i < kIn; ++i) {
      const uint32_t mask = ((1u << BITS) - 1) << (BITS * i);
      const uint64_t c = add2(f32x2(__uint_as_float((w & mask) | 0x4b000000u), __uint_as_float((v & mask) | 0x4b000000u)),
                              base2);
      const float2 y = split2(fma2(c, si[i], m2));
      x[2 * h * kIn + i] = y.x;
      x[(2 * h + 1) * kIn + i] = y.y;
    }
  }
}

struct Move {
  KvPool pool;
  View4 k, v;
  const int64_t *slots;
  uint32_t first, n_tokens, L;  // the launch's tokens [first, n_tokens) of the call's B L; L
  int tokens;            // of a CTA
  int pairs;             // (tensor, head) pairs of a CTA
  int step_pairs, step_tokens;  // rows of a round of the CTA: whole pairs and what is left
  int page_shift;        // log2 of the page, or -1
  int vec;
};

// A slot's bit of the second bitmap: the 15 upper bits of a product with 2^32
// over the golden ratio.
__device__ __forceinline__ uint32_t slot_hash(uint32_t s) { return s * 0x9e3779b1u >> 17; }

// Where a CTA's tokens lie: rows of the dense tensors (element offsets at head
// 0) and of the pool (at head 0; -1: nowhere).
struct Place {
  int64_t k, v, row;
};

__device__ __forceinline__ int64_t pool_row(const Move &A, int64_t s) {
  if (s < 0 || s >= A.pool.num_pages * A.pool.page) return -1;
  const int64_t page = A.page_shift >= 0 ? s >> A.page_shift : s / A.pool.page;
  return page * A.pool.Hkv * A.pool.page + (s - page * A.pool.page);
}

__device__ __forceinline__ Place place(const Move &A, uint32_t n) {
  const uint32_t b = n / A.L, l = n - b * A.L;
  return {b * A.k.sb + l * A.k.sl, b * A.v.sb + l * A.v.sl, pool_row(A, A.slots[n])};
}

// Writer.  CTA: `tokens` tokens (blockIdx.x) of `pairs` pairs (blockIdx.y);
// row = pair * tokens + token.  The same slot twice in a call: the CTA looks
// through all later tokens' slots (two bitmaps over its own slots rule nearly
// all of them out: one alone lets a token through for each of the CTA's when
// the call has 2^15, and each costs a loop over the CTA's slots) and leaves out its tokens that a later one overwrites, so a
// slot holds its last token whatever order the CTAs run in.  That look grows
// with the square of the tokens, so a launch takes kMaxLaunch of them at most,
// and the launches of a longer call follow one another: a later one overwrites.
template <typename T, int BITS>
__global__ void __launch_bounds__(kThreads, kCtas) kv_write_kernel(const __grid_constant__ Move A) {
  __shared__ Place at[kMaxTokens];
  __shared__ int64_t slot[kMaxTokens];
  __shared__ uint32_t bitmap[2 * kBitmapWords];
  const KvPool &P = A.pool;
  const uint32_t n0 = A.first + blockIdx.x * A.tokens, n_tokens = A.n_tokens;
  const bool several = n_tokens - A.first > 1;
  const int cnt = n_tokens - n0 < static_cast<uint32_t>(A.tokens) ? static_cast<int>(n_tokens - n0) : A.tokens;
  if (several)
    for (int i = threadIdx.x; i < 2 * kBitmapWords; i += kThreads) bitmap[i] = 0;
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();
  if (threadIdx.x < cnt) {
    const Place p = place(A, n0 + threadIdx.x);
    const int64_t s = p.row >= 0 ? A.slots[n0 + threadIdx.x] : -1;
    at[threadIdx.x] = p;
    slot[threadIdx.x] = s;
    if (s >= 0 && several) {
      const uint32_t hash = slot_hash(static_cast<uint32_t>(s));
      atomicOr(&bitmap[(s >> 5) & (kBitmapWords - 1)], 1u << (s & 31));
      atomicOr(&bitmap[kBitmapWords + (hash >> 5)], 1u << (hash & 31));
    }
  }
  __syncthreads();
  if (several) {
    // A slot's low word decides for nearly all.
    auto look = [&](uint32_t n, uint32_t s) {
      if (!(bitmap[(s >> 5) & (kBitmapWords - 1)] >> (s & 31) & 1)) return;
      const uint32_t hash = slot_hash(s);
      if (!(bitmap[kBitmapWords + (hash >> 5)] >> (hash & 31) & 1)) return;
      const int64_t full = A.slots[n];
      const int before = n - n0 < static_cast<uint32_t>(cnt) ? static_cast<int>(n - n0) : cnt;
      for (int t = 0; t < before; ++t)
        if (slot[t] == full) at[t].row = -1;  // (whoever finds it writes the same)
    };
    // two a load, from a 16-byte boundary (token n0 itself does no harm), and
    // several loads ahead: it is L2's latency that counts
    constexpr int kAhead = 4;
    const uint32_t i0 = n0 + 1 - static_cast<uint32_t>(reinterpret_cast<uintptr_t>(A.slots + n0 + 1) >> 3 & 1);
    const uint4 *two = reinterpret_cast<const uint4 *>(A.slots + i0);
    const uint32_t twos = (n_tokens - i0) / 2;
    for (uint32_t p = threadIdx.x; p < twos; p += kAhead * kThreads) {
      uint4 v[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (p + u * kThreads < twos) v[u] = two[p + u * kThreads];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const uint32_t at2 = p + u * kThreads;
        if (at2 >= twos) break;
        look(i0 + 2 * at2, v[u].x);
        look(i0 + 2 * at2 + 1, v[u].z);
      }
    }
    if (threadIdx.x == 0 && (n_tokens - i0) % 2) look(n_tokens - 1, static_cast<uint32_t>(A.slots[n_tokens - 1]));
    __syncthreads();
  }

  const int lpr = P.D / kN, l = threadIdx.x & (lpr - 1);  // lanes a row
  const int rows = A.tokens * A.pairs;
  const int gl = P.group / kN, groups = P.D / P.group;
  const int step = kThreads / lpr, mine = threadIdx.x / lpr;
  // every lane runs every round (the group's shuffles take the whole warp);
  // the next round's row loads while this one's is worked on
  Piece<T> x, ahead;
  int64_t row, row_ahead;
  bool is_v, is_v_ahead;
  const int end_pair = (blockIdx.y + 1) * A.pairs;
  int next_pair = blockIdx.y * A.pairs + mine / A.tokens, next_t = mine % A.tokens;
  auto load = [&]() {
    const int t = next_t, pair = next_pair;
    is_v_ahead = pair >= P.Hkv;
    const int h = is_v_ahead ? pair - P.Hkv : pair;
    row_ahead = pair < end_pair && t < cnt ? at[t].row : -1;
#pragma unroll
    for (int i = 0; i < static_cast<int>(kN * sizeof(T) / 4); ++i) ahead.w[i] = 0;
    if (row_ahead >= 0) {
      const View4 &src = is_v_ahead ? A.v : A.k;
      load_piece(static_cast<const T *>(src.p) + (is_v_ahead ? at[t].v : at[t].k) + h * src.sh + kN * l, A.vec, ahead);
      row_ahead += static_cast<int64_t>(h) * P.page;
    }
    next_pair += A.step_pairs;  // the thread's row of the next round
    next_t += A.step_tokens;
    if (next_t >= A.tokens) {
      next_t -= A.tokens;
      ++next_pair;
    }
  };
  load();
  for (int r0 = 0; r0 < rows; r0 += step) {
    x = ahead;
    row = row_ahead;
    is_v = is_v_ahead;
    if (r0 + step < rows) load();
    uint32_t param, words[kN * BITS / 32];
    quantise<T, BITS>(x, gl, words, &param);
    if (row < 0) continue;
    uint8_t *dst = static_cast<uint8_t *>(is_v ? P.v_codes : P.k_codes) + row * (P.D * BITS / 8) + kN * BITS / 8 * l;
    if constexpr (BITS == 4) {
      *reinterpret_cast<uint2 *>(dst) = make_uint2(words[0], words[1]);
    } else {
      *reinterpret_cast<uint4 *>(dst) = make_uint4(words[0], words[1], words[2], words[3]);
    }
    if ((l & (gl - 1)) == 0)
      static_cast<uint32_t *>(is_v ? P.v_params : P.k_params)[row * groups + l / gl] = param;
  }
}

// Reader.  CTAs as the writer's.
template <typename T, int BITS>
__global__ void __launch_bounds__(kThreads, kCtas) kv_read_kernel(const __grid_constant__ Move A) {
  __shared__ Place at[kMaxTokens];
  const KvPool &P = A.pool;
  const uint32_t n0 = blockIdx.x * A.tokens;
  const int cnt = A.n_tokens - n0 < static_cast<uint32_t>(A.tokens) ? static_cast<int>(A.n_tokens - n0) : A.tokens;
  pdl_wait();
  pdl_launch_dependents();
  if (threadIdx.x < cnt) at[threadIdx.x] = place(A, n0 + threadIdx.x);
  __syncthreads();
  const int lpr = P.D / kN, l = threadIdx.x & (lpr - 1);
  const int rows = A.tokens * A.pairs;
  const int gl = P.group / kN, groups = P.D / P.group;
  constexpr int kU = 2, kW = kN * BITS / 32;
  const int step = kThreads / lpr, mine = threadIdx.x / lpr;
  uint32_t words[kU][kW], param[kU], words_ahead[kU][kW], param_ahead[kU];
  T *dst[kU], *dst_ahead[kU];
  const int end_pair = (blockIdx.y + 1) * A.pairs;
  int next_pair = blockIdx.y * A.pairs + mine / A.tokens, next_t = mine % A.tokens;
  auto next_row = [&]() {  // the thread's row of the next round
    next_pair += A.step_pairs;
    next_t += A.step_tokens;
    if (next_t >= A.tokens) {
      next_t -= A.tokens;
      ++next_pair;
    }
  };
  auto load = [&]() {
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int t = next_t, pair = next_pair;
      const bool is_v = pair >= P.Hkv;
      const int h = is_v ? pair - P.Hkv : pair;
      dst_ahead[u] = nullptr;
      param_ahead[u] = 0;  // a slot outside the cache reads as zeros
#pragma unroll
      for (int i = 0; i < kW; ++i) words_ahead[u][i] = 0;
      next_row();
      if (pair >= end_pair || t >= cnt) continue;
      const View4 &out = is_v ? A.v : A.k;
      dst_ahead[u] = static_cast<T *>(out.p) + (is_v ? at[t].v : at[t].k) + h * out.sh + kN * l;
      if (at[t].row < 0) continue;
      const int64_t row = at[t].row + static_cast<int64_t>(h) * P.page;
      const uint8_t *src = static_cast<const uint8_t *>(is_v ? P.v_codes : P.k_codes) + row * (P.D * BITS / 8) +
                           kN * BITS / 8 * l;
      if constexpr (BITS == 4) {
        const uint2 w = *reinterpret_cast<const uint2 *>(src);
        words_ahead[u][0] = w.x;
        words_ahead[u][1] = w.y;
      } else {
        const uint4 w = *reinterpret_cast<const uint4 *>(src);
        words_ahead[u][0] = w.x;
        words_ahead[u][1] = w.y;
        words_ahead[u][2] = w.z;
        words_ahead[u][3] = w.w;
      }
      param_ahead[u] = static_cast<const uint32_t *>(is_v ? P.v_params : P.k_params)[row * groups + l / gl];
    }
  };
  load();
  for (int r0 = 0; r0 < rows; r0 += kU * step) {
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      dst[u] = dst_ahead[u];
      param[u] = param_ahead[u];
#pragma unroll
      for (int i = 0; i < kW; ++i) words[u][i] = words_ahead[u][i];
    }
    if (r0 + kU * step < rows) load();
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      if (!dst[u]) continue;
      const float s = __uint_as_float(param[u] << 16), m = __uint_as_float(param[u] & 0xffff0000u);
      uint64_t si[16 / BITS];
#pragma unroll
      for (int i = 0; i < 16 / BITS; ++i) {
        const float f = s * (1.f / static_cast<float>(1 << (BITS * i)));
        si[i] = f32x2(f, f);
      }
#pragma unroll
      for (int g = 0; g < kN / 8; ++g) {
        float x[8];
        values8<BITS>(&words[u][g * BITS / 4], si, f32x2(m, m), x);
        store8(dst[u] + 8 * g, A.vec, x);
      }
    }
  }
}

bool rows_on_16_bytes(const View4 &v, int64_t el) {
  return (reinterpret_cast<uintptr_t>(v.p) & 15) == 0 && v.sb * el % 16 == 0 && v.sh * el % 16 == 0 &&
         v.sl * el % 16 == 0;
}

template <typename T>
cudaError_t move_t(bool write, const KvPool &p, const View4 &k, const View4 &v, int64_t B, int64_t L,
                   const int64_t *slots, int sm_count, cudaStream_t stream) {
  Move a = {};
  a.pool = p;
  a.k = k;
  a.v = v;
  a.slots = slots;
  a.L = static_cast<uint32_t>(L);
  a.vec = rows_on_16_bytes(k, sizeof(T)) && rows_on_16_bytes(v, sizeof(T));
  a.page_shift = -1;
  for (int i = 4; i < 17; ++i)
    if (p.page == 1 << i) a.page_shift = i;
  // CTAs: tokens x a share of the heads.  A writer's CTA looks through all
  // later slots, so it should have many rows; but the SM with the most CTAs is
  // the last to finish, and one CTA alone leaves it idle for a third of the
  // time.  The least of an SM's CTAs x a CTA's cost, in the units of an
  // instruction of all its warps, as measured: 500 for a round of 16 elements
  // a lane, 0.1 for a slot looked through, 600 to begin with.
  const int64_t all = B * L, launches = write ? (all + kMaxLaunch - 1) / kMaxLaunch : 1;
  const int64_t n = (all + launches - 1) / launches;  // tokens of a launch
  const int lpr = p.D / kN;
  int ysplit = 1;
  double least = 0;
  for (int y = 1; 2 * p.Hkv % y == 0; y *= 2)
    for (int most = 1; most <= 3 * kCtas; ++most) {  // CTAs of an SM
      int64_t tokens = (n * y + most * static_cast<int64_t>(sm_count) - 1) / (most * static_cast<int64_t>(sm_count));
      if (tokens > kMaxTokens) tokens = kMaxTokens;
      const int64_t ctas = (n + tokens - 1) / tokens * y;
      const int64_t rounds = (tokens * (2 * p.Hkv / y) * lpr + kThreads - 1) / kThreads;
      const double of_sm = static_cast<double>((ctas + sm_count - 1) / sm_count);
      const double cost = (of_sm < 1.6 ? 1.6 : of_sm) *
                          (600 + 500 * static_cast<double>(rounds) + (write ? 0.1 * static_cast<double>(n) / 2 : 0));
      if (least == 0 || cost < least) {
        least = cost;
        a.tokens = static_cast<int>(tokens);
        ysplit = y;
      }
    }
  a.pairs = 2 * p.Hkv / ysplit;
  a.step_pairs = kThreads / lpr / a.tokens;
  a.step_tokens = kThreads / lpr % a.tokens;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim.y = static_cast<unsigned>(ysplit);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  for (int64_t first = 0; first < all; first += n) {
    a.first = static_cast<uint32_t>(first);
    a.n_tokens = static_cast<uint32_t>(first + n < all ? first + n : all);
    cfg.gridDim.x = (a.n_tokens - a.first + a.tokens - 1) / a.tokens;
    const cudaError_t e =
        write ? cudaLaunchKernelEx(&cfg, p.bits == 4 ? kv_write_kernel<T, 4> : kv_write_kernel<T, 8>, a)
              : cudaLaunchKernelEx(&cfg, p.bits == 4 ? kv_read_kernel<T, 4> : kv_read_kernel<T, 8>, a);
    if (e != cudaSuccess) return e;
  }
  return cudaGetLastError();
}

cudaError_t move(bool write, const KvPool &p, const View4 &k, const View4 &v, int dtype, int64_t B, int64_t L,
                 const int64_t *slots, int sm_count, cudaStream_t stream) {
  if (B * L == 0) return cudaSuccess;
  if (dtype == LLK_DTYPE_FP32) return move_t<float>(write, p, k, v, B, L, slots, sm_count, stream);
  if (dtype == LLK_DTYPE_FP16) return move_t<__half>(write, p, k, v, B, L, slots, sm_count, stream);
  return move_t<__nv_bfloat16>(write, p, k, v, B, L, slots, sm_count, stream);
}

}  // namespace

bool kv_pool_supported(const KvPool &p) {
  return (p.D == 64 || p.D == 128 || p.D == 256) && (p.bits == 4 || p.bits == 8) &&
         (p.group == 32 || p.group == 64 || p.group == 128) && p.D % p.group == 0 && p.page >= 16 &&
         p.page % 16 == 0 && p.page <= 65536 && p.Hkv >= 1 && p.Hkv <= 4096 && p.num_pages >= 0 &&
         p.num_pages <= (int64_t(1) << 31) - 1;
}

cudaError_t kv_write_launch(const KvPool &p, const View4 &k, const View4 &v, int dtype, int64_t B, int64_t L,
                            const int64_t *slots, int sm_count, cudaStream_t stream) {
  return move(true, p, k, v, dtype, B, L, slots, sm_count, stream);
}

cudaError_t kv_read_launch(const KvPool &p, const View4 &k, const View4 &v, int dtype, int64_t B, int64_t L,
                           const int64_t *slots, int sm_count, cudaStream_t stream) {
  return move(false, p, k, v, dtype, B, L, slots, sm_count, stream);
}

}  // namespace llk_b200
