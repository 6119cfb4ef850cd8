// kv_cache.cu -- the quantised paged KV cache's writer and reader.
//
// A token's key or value of one head, x [D], is held in groups of `group`
// elements.  With x saturated to +-65504 and NaN counted as 0, per group
//   m = bf16(min x),   s = bf16(f32(max((max x - m) / (2^bits - 1), 2^-30))),
//   code = clamp(rint((x - m) / s), 0, 2^bits - 1)  (ties to even),
// both quotients as in 64 bits; the group stands for s * code + m.  With 4
// bits the elements 2j and 2j + 1 share byte j (2j in the low nibble).
//
// HBM-bound both ways: a thread owns 8 elements of a row (one 16-byte load
// for 16-bit types), a row is D / 8 neighbouring lanes, the group's minimum
// and maximum are shuffles.  Codes next to a border between two (|q - k -
// 1/2| below the f32 quotient's error, the exact ties of 16-bit inputs among
// them) are decided by the sign of x - m - (k + 1/2) s in f64, so the codes do
// not depend on how the quotient was rounded.
#include <cuda.h>
#include <cuda_runtime.h>

#include "attn_common.cuh"

namespace llk_b200 {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 64;        // tokens of a writer's CTA
constexpr int kBitmapWords = 1024;    // 32768 bits over the low bits of the CTA's slots
constexpr float kLargest = 65504.f;
constexpr double kLeastScale = 0x1p-30;

template <typename T>
__device__ __forceinline__ void load_elems(const T *src, bool vec, float (&x)[8]) {
  if (vec) {
    constexpr int kPieces = sizeof(T) * 8 / 16;
    uint4 w[kPieces];
#pragma unroll
    for (int i = 0; i < kPieces; ++i) w[i] = __ldcs(reinterpret_cast<const uint4 *>(src) + i);
    const T *e = reinterpret_cast<const T *>(w);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32(src[i]);
  }
}

template <typename T>
__device__ __forceinline__ void store_elems(T *dst, bool vec, const float (&x)[8]) {
  T e[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(x[i]);
  if (vec) {
    constexpr int kPieces = sizeof(T) * 8 / 16;
    uint4 w[kPieces];
    memcpy(w, e, sizeof(w));
#pragma unroll
    for (int i = 0; i < kPieces; ++i) reinterpret_cast<uint4 *>(dst)[i] = w[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) dst[i] = e[i];
  }
}

// Codes of one lane's 8 elements (packed, BITS bytes) and its group's
// (scale, min); gl lanes share a group.
template <int BITS>
__device__ __forceinline__ uint64_t quantise8(float (&x)[8], int gl, uint32_t *param) {
  constexpr float kTop = static_cast<float>((1 << BITS) - 1);
  float mn = INFINITY, mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[i] = x[i] != x[i] ? 0.f : fminf(fmaxf(x[i], -kLargest), kLargest);
    mn = fminf(mn, x[i]);
    mx = fmaxf(mx, x[i]);
  }
#pragma unroll
  for (int off = 1; off < 16; off <<= 1) {
    const float a = __shfl_xor_sync(0xffffffffu, mn, off), c = __shfl_xor_sync(0xffffffffu, mx, off);
    if (off < gl) {
      mn = fminf(mn, a);
      mx = fmaxf(mx, c);
    }
  }
  const __nv_bfloat16 mb = __float2bfloat16_rn(mn);
  const float m = __bfloat162float(mb);
  const double q = (static_cast<double>(mx) - static_cast<double>(m)) / static_cast<double>((1 << BITS) - 1);
  const __nv_bfloat16 sb = __float2bfloat16_rn(static_cast<float>(q < kLeastScale ? kLeastScale : q));
  const float s = __bfloat162float(sb), inv = 1.f / s;
  *param = static_cast<uint32_t>(__bfloat16_as_ushort(sb)) | (static_cast<uint32_t>(__bfloat16_as_ushort(mb)) << 16);
  uint64_t codes = 0;
  // error of the f32 quotient: three roundings of 2^-24 on at most 2^BITS
  constexpr float kNear = static_cast<float>(1 << BITS) * 0x1p-21f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float v = (x[i] - m) * inv;
    const float k = floorf(v), f = v - k;
    float c = f > 0.5f ? k + 1.f : k;
    if (fabsf(f - 0.5f) < kNear) {
      const double d = (static_cast<double>(x[i]) - static_cast<double>(m)) -
                       (static_cast<double>(k) + 0.5) * static_cast<double>(s);
      c = d > 0.0 || (d == 0.0 && (static_cast<int>(k) & 1)) ? k + 1.f : k;
    }
    c = fminf(fmaxf(c, 0.f), kTop);
    codes |= static_cast<uint64_t>(static_cast<uint32_t>(c)) << (BITS * i);
  }
  return codes;
}

// Writer.  CTA: `tokens` tokens (blockIdx.x) of `pairs` (tensor, head) pairs
// (blockIdx.y); row = pair * tokens + token.  The same slot twice in a call:
// the CTA looks through all later tokens' slots (a bitmap over its own slots
// rules nearly all of them out) and leaves out its tokens that a later one
// overwrites, so a slot holds its last token whatever order the CTAs run in.
template <typename T, int BITS>
__global__ void __launch_bounds__(kThreads) kv_write_kernel(const KvPool P, const View4 K, const View4 V,
                                                            const int64_t *__restrict__ slots, uint32_t n_tokens,
                                                            uint32_t L, int tokens, int pairs, int vec) {
  __shared__ int64_t slot[kMaxTokens];
  __shared__ uint32_t bitmap[kBitmapWords];
  const uint32_t n0 = blockIdx.x * tokens;
  const int cnt = n_tokens - n0 < static_cast<uint32_t>(tokens) ? static_cast<int>(n_tokens - n0) : tokens;
  const int64_t n_slots = P.num_pages * P.page;
  if (n_tokens > 1)
    for (int i = threadIdx.x; i < kBitmapWords; i += kThreads) bitmap[i] = 0;
  __syncthreads();
  pdl_launch_dependents();
  pdl_wait();
  if (threadIdx.x < cnt) {
    const int64_t s = slots[n0 + threadIdx.x];
    const bool ok = s >= 0 && s < n_slots;
    slot[threadIdx.x] = ok ? s : -1;
    if (ok && n_tokens > 1) atomicOr(&bitmap[(s >> 5) & (kBitmapWords - 1)], 1u << (s & 31));
  }
  __syncthreads();
  for (uint32_t n = n0 + 1 + threadIdx.x; n < n_tokens; n += kThreads) {
    const int64_t s = slots[n];
    if (s < 0 || s >= n_slots || !(bitmap[(s >> 5) & (kBitmapWords - 1)] >> (s & 31) & 1)) continue;
    const int before = n - n0 < static_cast<uint32_t>(cnt) ? static_cast<int>(n - n0) : cnt;
    for (int t = 0; t < before; ++t)
      if (slot[t] == s) slot[t] = -1;  // only ever set to -1 here: threads agree, and a later equal token remains
  }
  __syncthreads();

  const int lpr = P.D / 8;  // lanes a row
  const int rows = cnt * pairs, l = threadIdx.x % lpr;
  const int gl = P.group / 8, groups = P.D / P.group;
  const int64_t row_bytes = P.D * BITS / 8;
  constexpr int kU = 4;  // rows in flight a thread
  const int step = kThreads / lpr;
  // every lane runs every round (the group's shuffles take the whole warp)
  for (int r0 = 0; r0 < rows; r0 += kU * step) {
    float x[kU][8];
    int64_t at[kU];
    int which[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int r = r0 + u * step + threadIdx.x / lpr;
      at[u] = -1;
      which[u] = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) x[u][i] = 0.f;
      if (r < rows) {
        const int pair = blockIdx.y * pairs + r / cnt, t = r % cnt;
        const int64_t s = slot[t];
        which[u] = pair >= P.Hkv;
        const int h = which[u] ? pair - P.Hkv : pair;
        if (s >= 0) {
          const View4 &src = which[u] ? V : K;
          const uint32_t n = n0 + t, b = n / L;
          load_elems(static_cast<const T *>(src.p) + b * src.sb + h * src.sh + (n - b * L) * src.sl + 8 * l, vec,
                     x[u]);
          at[u] = (s / P.page * P.Hkv + h) * P.page + s % P.page;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      uint32_t param;
      const uint64_t codes = quantise8<BITS>(x[u], gl, &param);
      if (at[u] < 0) continue;
      uint8_t *dst = static_cast<uint8_t *>(which[u] ? P.v_codes : P.k_codes) + at[u] * row_bytes + BITS * l;
      if constexpr (BITS == 4) {
        *reinterpret_cast<uint32_t *>(dst) = static_cast<uint32_t>(codes);
      } else {
        *reinterpret_cast<uint64_t *>(dst) = codes;
      }
      if (l % gl == 0) static_cast<uint32_t *>(which[u] ? P.v_params : P.k_params)[at[u] * groups + l / gl] = param;
    }
  }
}

// Reader.  A thread turns the codes of 8 elements into values, one fused
// multiply-add each (s * code is exact in f32); rows in the order of the
// output, kU of them in flight a thread.
template <typename T, int BITS>
__global__ void __launch_bounds__(kThreads) kv_read_kernel(const KvPool P, const View4 K, const View4 V,
                                                           const int64_t *__restrict__ slots, uint32_t n_rows,
                                                           uint32_t B, uint32_t L, int vec) {
  const int64_t n_slots = P.num_pages * P.page;
  const int lpr = P.D / 8, l = threadIdx.x % lpr, gl = P.group / 8, groups = P.D / P.group;
  const int64_t row_bytes = P.D * BITS / 8;
  constexpr int kU = 4;
  const uint32_t step = kThreads / lpr;
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t r0 = blockIdx.x * (kU * step) + threadIdx.x / lpr;
  uint64_t codes[kU];
  uint32_t param[kU];
  int64_t dst[kU];
#pragma unroll
  for (int u = 0; u < kU; ++u) {
    const uint32_t r = r0 + u * step;
    codes[u] = 0;
    param[u] = 0;
    dst[u] = -1;
    if (r >= n_rows) continue;
    // r = ((which * B + b) * Hkv + h) * L + t
    const uint32_t t = r % L, wbh = r / L, h = wbh % P.Hkv, wb = wbh / P.Hkv;
    const bool isv = wb >= B;
    const uint32_t b = isv ? wb - B : wb;
    const View4 &out = isv ? V : K;
    dst[u] = b * out.sb + h * out.sh + t * out.sl + 8 * l;
    const int64_t s = slots[static_cast<int64_t>(b) * L + t];
    if (s < 0 || s >= n_slots) continue;  // reads as zeros
    const int64_t at = (s / P.page * P.Hkv + h) * P.page + s % P.page;
    const uint8_t *src = static_cast<const uint8_t *>(isv ? P.v_codes : P.k_codes) + at * row_bytes + BITS * l;
    codes[u] = BITS == 4 ? *reinterpret_cast<const uint32_t *>(src) : *reinterpret_cast<const uint64_t *>(src);
    param[u] = static_cast<const uint32_t *>(isv ? P.v_params : P.k_params)[at * groups + l / gl];
  }
#pragma unroll
  for (int u = 0; u < kU; ++u) {
    const uint32_t r = r0 + u * step;
    if (r >= n_rows) continue;
    const bool isv = r / L / P.Hkv >= B;
    const float s = __uint_as_float(param[u] << 16), m = __uint_as_float(param[u] & 0xffff0000u);
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      x[i] = fmaf(s, static_cast<float>(static_cast<uint32_t>(codes[u] >> (BITS * i)) & ((1u << BITS) - 1)), m);
    store_elems(static_cast<T *>(isv ? V.p : K.p) + dst[u], vec, x);
  }
}

bool rows_on_16_bytes(const View4 &v, int64_t el) {
  return (reinterpret_cast<uintptr_t>(v.p) & 15) == 0 && v.sb * el % 16 == 0 && v.sh * el % 16 == 0 &&
         v.sl * el % 16 == 0;
}

template <typename... Args>
cudaError_t launch(void (*kern)(Args...), dim3 grid, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
  return e != cudaSuccess ? e : cudaGetLastError();
}

template <typename T>
cudaError_t write_t(const KvPool &p, const View4 &k, const View4 &v, int64_t B, int64_t L, const int64_t *slots,
                    int sm_count, cudaStream_t stream) {
  const int vec = rows_on_16_bytes(k, sizeof(T)) && rows_on_16_bytes(v, sizeof(T));
  const int64_t n = B * L;
  // Few CTAs look through the slots (each reads all later ones) and fill the
  // GPU twice: shrink a CTA's tokens, then its heads, until they do.
  int tokens = kMaxTokens, ysplit = 1;
  const int total = 2 * p.Hkv;
  auto ctas = [&] { return (n + tokens - 1) / tokens * ysplit; };
  while (ctas() < 2 * sm_count && tokens > 16) tokens /= 2;
  while (ctas() < 2 * sm_count && total % (2 * ysplit) == 0) ysplit *= 2;
  while (ctas() < 2 * sm_count && tokens > 1) tokens /= 2;
  const dim3 grid(static_cast<unsigned>((n + tokens - 1) / tokens), static_cast<unsigned>(ysplit));
  return launch(p.bits == 4 ? kv_write_kernel<T, 4> : kv_write_kernel<T, 8>, grid, stream, p, k, v, slots,
                static_cast<uint32_t>(n), static_cast<uint32_t>(L), tokens, total / ysplit, vec);
}

template <typename T>
cudaError_t read_t(const KvPool &p, const View4 &k, const View4 &v, int64_t B, int64_t L, const int64_t *slots,
                   cudaStream_t stream) {
  const int vec = rows_on_16_bytes(k, sizeof(T)) && rows_on_16_bytes(v, sizeof(T));
  const uint32_t rows = static_cast<uint32_t>(2 * B * p.Hkv * L), per = 4 * (kThreads / (p.D / 8));
  return launch(p.bits == 4 ? kv_read_kernel<T, 4> : kv_read_kernel<T, 8>, dim3((rows + per - 1) / per), stream, p, k,
                v, slots, rows, static_cast<uint32_t>(B), static_cast<uint32_t>(L), vec);
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
  if (B * L == 0) return cudaSuccess;
  if (dtype == LLK_DTYPE_FP32) return write_t<float>(p, k, v, B, L, slots, sm_count, stream);
  if (dtype == LLK_DTYPE_FP16) return write_t<__half>(p, k, v, B, L, slots, sm_count, stream);
  return write_t<__nv_bfloat16>(p, k, v, B, L, slots, sm_count, stream);
}

cudaError_t kv_read_launch(const KvPool &p, const View4 &k, const View4 &v, int dtype, int64_t B, int64_t L,
                           const int64_t *slots, int sm_count, cudaStream_t stream) {
  if (B * L == 0) return cudaSuccess;
  if (dtype == LLK_DTYPE_FP32) return read_t<float>(p, k, v, B, L, slots, stream);
  if (dtype == LLK_DTYPE_FP16) return read_t<__half>(p, k, v, B, L, slots, stream);
  return read_t<__nv_bfloat16>(p, k, v, B, L, slots, stream);
}

}  // namespace llk_b200
