// window_attention.cu -- llk.window_attention on the CUDA cores: the kernel
// for f32, whose products tensor cores would round, and for the 16-bit calls
// that TMA cannot describe (rows that do not start on 16 bytes, a D that is
// not a multiple of 8) or whose head is wider than 128.
//
//   o_i = sum_j softmax_j(scale q_i . k_j) v_j over the keys j that query i
//   sees (AttnMask), one pass over the keys with the running maximum m and
//   sum l of the softmax, everything in f32.
//
// A CTA owns 64 query rows of one head and sweeps the 64-key tiles that any
// of them sees: the sinks' tiles, then the window's.  FMA-bound: 4 D FLOP a
// pair.  A warp owns 2 R neighbouring rows and skips the halves of tiles that
// none of them sees; lane (tx, ty) has R rows x 4 keys of scores and R rows x
// 4 DP/64 columns of O, so 16-byte loads from shared memory feed 2 R / 3 and
// more packed f32 pairs each.  R = 8 with four warps, two CTAs an SM: one
// CTA's loads and softmax run beside the other's products.  (R = 4 with eight
// warps where DP = 256: R = 8 would need more than 255 registers.)  The
// probabilities pass through the warp's own piece of shared memory.
//
// Measured (f32, D = 128, 1965 MHz): 32 heads, 1000 tokens, window 333: 156 us
// for 61 at the nominal FMA rate, 1.45 times the pairs being computed where
// tiles are cut by the window's ends (the FMA pipe works 58 % of the clocks at 8
// warps an SM, stalls are fixed latencies, the pipe itself and the CTA's
// barriers); 4096 tokens without a window 2.96 ms, 0.63 of the rate.  One CTA of
// 256 threads with 4 x 4 scores a thread took 204 us.
#include <cuda.h>
#include <cuda_runtime.h>

#include "attn_common.cuh"

namespace llk_b200 {

namespace {

constexpr int kBQ = 64, kBK = 64, kPad = 4;

__device__ __forceinline__ void cp_async16_zfill(float *dst, const float *src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(in ? 16 : 0)
               : "memory");
}

// Eight consecutive elements of a 16-byte row piece as f32.
template <typename T>
__device__ __forceinline__ void load8(const T *src, float *x) {
  const uint4 w = *reinterpret_cast<const uint4 *>(src);
  const T *e = reinterpret_cast<const T *>(&w);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = to_f32(e[i]);
}

// Rows row0 .. row0 + 63 of src into dst [64][DP + kPad]; rows outside
// [begin, end) and columns past D become zero (they are not read: what lies
// there may be anything).  kVec: rows start on 16 bytes and D is a multiple
// of the 16-byte piece.
template <typename T, int DP, bool kVec, int kThreads>
__device__ __forceinline__ void load_rows(float *dst, const T *src, int64_t sl, int row0, int begin, int end, int D) {
  constexpr int kLd = DP + kPad;
  if constexpr (kVec && sizeof(T) == 4) {
    constexpr int kRows = kThreads / (DP / 4);  // of a round
    const int r0 = threadIdx.x / (DP / 4), c = 4 * (threadIdx.x % (DP / 4));
    const T *from = src + (row0 + r0) * sl + c;
    float *to = dst + r0 * kLd + c;
#pragma unroll
    for (int r = 0; r < kBQ; r += kRows) {
      const int row = row0 + r0 + r;
      const bool in = row >= begin && row < end && c < D;
      cp_async16_zfill(to + r * kLd, reinterpret_cast<const float *>(in ? from : src), in);
      from += kRows * sl;
    }
  } else if constexpr (kVec) {
    for (int e = threadIdx.x; e < kBQ * (DP / 8); e += kThreads) {
      const int r = e / (DP / 8), c = 8 * (e % (DP / 8)), row = row0 + r;
      float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (row >= begin && row < end && c < D) load8(src + row * sl + c, x);
      float4 *to = reinterpret_cast<float4 *>(dst + r * kLd + c);
      to[0] = make_float4(x[0], x[1], x[2], x[3]);
      to[1] = make_float4(x[4], x[5], x[6], x[7]);
    }
  } else {
    for (int e = threadIdx.x; e < kBQ * DP; e += kThreads) {
      const int r = e / DP, c = e % DP, row = row0 + r;
      dst[r * kLd + c] = row >= begin && row < end && c < D ? to_f32(src[row * sl + c]) : 0.f;
    }
  }
}

__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t twice(float x) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %1};" : "=l"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float2 split2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}

// Scores (scaled) of a lane's R rows (2 apart) and the keys tx + 16 j, j0 <= j < j1.
template <int R, int DP, int j0, int j1>
__device__ __forceinline__ void dot_products(const float *q, const float *k, float scale, float (&s)[R][4]) {
  constexpr int kLd = DP + kPad;
  uint64_t acc[R][j1 - j0];  // sums of the even and of the odd d
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = j0; j < j1; ++j) acc[i][j - j0] = 0;
#pragma unroll 4
  for (int d = 0; d < DP; d += 4) {
    ulonglong2 a[R], b[j1 - j0];
#pragma unroll
    for (int j = j0; j < j1; ++j) b[j - j0] = *reinterpret_cast<const ulonglong2 *>(k + 16 * j * kLd + d);
#pragma unroll
    for (int i = 0; i < R; ++i) a[i] = *reinterpret_cast<const ulonglong2 *>(q + 2 * i * kLd + d);
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < j1 - j0; ++j) acc[i][j] = fma2(a[i].x, b[j].x, acc[i][j]);
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < j1 - j0; ++j) acc[i][j] = fma2(a[i].y, b[j].y, acc[i][j]);
  }
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      s[i][j] = 0.f;
      if (j >= j0 && j < j1) {
        const float2 x = split2(acc[i][j - j0]);
        s[i][j] = (x.x + x.y) * scale;
      }
    }
}

template <typename T, int DP>
struct Simt {
  static constexpr int R = DP > 128 ? 4 : 8;  // rows of a lane
  static constexpr int kWarps = kBQ / (2 * R), kThreads = 32 * kWarps;
  static constexpr int kCtas = DP > 128 ? 1 : 2;
  static constexpr int kLdP = 2 * R + kPad;  // [key][row] of a half tile
  static constexpr int kSmem = (3 * kBQ * (DP + kPad) + kWarps * kBK / 2 * kLdP) * static_cast<int>(sizeof(float));
  static_assert(kCtas * (kSmem + 1024) <= 228 * 1024, "shared memory");
};

template <typename T, int DP, bool kVec>
__global__ void __launch_bounds__(Simt<T, DP>::kThreads, Simt<T, DP>::kCtas)
    window_simt_kernel(const AttnProblem P, int q_tiles) {
  using G = Simt<T, DP>;
  extern __shared__ __align__(16) float sm[];
  constexpr int kLd = DP + kPad, kOC = DP / 64, R = G::R, kLdP = G::kLdP;
  float *Qs = sm, *Ks = Qs + kBQ * kLd, *Vs = Ks + kBK * kLd;
  const int warp = threadIdx.x >> 5, ty = threadIdx.x >> 4 & 1, tx = threadIdx.x & 15;
  float *Pt = Vs + kBK * kLd + warp * (kBK / 2 * kLdP);
  // the last query tiles first: under the causal mask they have the most keys
  const int BH = P.B * P.H;
  const int b = (blockIdx.x % BH) / P.H, h = blockIdx.x % P.H;
  const int q0 = (q_tiles - 1 - static_cast<int>(blockIdx.x / BH)) * kBQ;
  const int hk = h / (P.H / P.Hkv), D = P.D;
  const T *qb = static_cast<const T *>(P.q.p) + b * P.q.sb + h * P.q.sh;
  const T *kb = static_cast<const T *>(P.k.p) + b * P.k.sb + hk * P.k.sh;
  const T *vb = static_cast<const T *>(P.v.p) + b * P.v.sb + hk * P.v.sh;
  T *ob = static_cast<T *>(P.o.p) + b * P.o.sb + h * P.o.sh;

  pdl_launch_dependents();
  pdl_wait();
  int n, m_rows;
  seq_lens(P.mask, b, n, m_rows);
  if (q0 >= m_rows) return;
  const int sinks = P.mask.sinks;
  const int p0 = n - m_rows + q0;                                    // position of the tile's first row
  const int last = p0 + (m_rows - q0 < kBQ ? m_rows - q0 : kBQ) - 1; // and of its last
  const int hi = last + 1;                                           // keys any row sees: < hi (may be <= 0)
  const int lo = window_lo(P.mask, p0);                              // >= lo, or < sinks
  // tiles: s_tiles of sinks in front, then from the window's first
  const int w_first = lo / kBK;
  const int s_keys = sinks < lo ? sinks : lo;
  const int s_all = (s_keys + kBK - 1) / kBK, s_tiles = s_all < w_first ? s_all : w_first;
  const int end_tile = hi > 0 ? (hi + kBK - 1) / kBK : 0;
  const int tiles = end_tile > w_first ? s_tiles + end_tile - w_first : 0;
  auto tile_row = [&](int t) { return (t < s_tiles ? t : w_first + t - s_tiles) * kBK; };
  auto load_tile = [&](float *dst, const T *src, int64_t sl, int t) {
    // a sinks' tile ends with the sinks (unless the window begins inside it)
    const int r0 = tile_row(t);
    const int begin = r0 >= s_keys ? lo : 0;
    const int end = t < s_tiles && r0 + kBK <= lo ? (s_keys < hi ? s_keys : hi) : hi;
    load_rows<T, DP, kVec, G::kThreads>(dst, src, sl, r0, begin, end, D);
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // the warp's rows: row(i) of the tile; the keys they see as lo and hi above
  auto row = [&](int i) { return 2 * R * warp + 2 * i + ty; };
  const int w0 = p0 + 2 * R * warp, w1 = w0 + 2 * R - 1 < last ? w0 + 2 * R - 1 : last;
  const int warp_lo = window_lo(P.mask, w0), warp_hi = w1 >= w0 ? w1 + 1 : 0;
  const float *q_rows = Qs + row(0) * kLd, *k_rows = Ks + tx * kLd;

  load_rows<T, DP, kVec, G::kThreads>(Qs, qb, P.q.sl, q0, 0, m_rows, D);
  if (tiles > 0) load_tile(Ks, kb, P.k.sl, 0);
  float m[R], l[R];  // l: of this lane's keys alone
  uint64_t acc[R][kOC][2];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int j = 0; j < kOC; ++j) acc[i][j][0] = acc[i][j][1] = 0;
  }
  const float sc = P.scale * kLog2e;
  for (int t = 0; t < tiles; ++t) {
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();  // K is there, V is free
    load_tile(Vs, vb, P.v.sl, t);
    const int k0 = tile_row(t);
    bool sees[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int h0 = k0 + u * (kBK / 2);
      sees[u] = h0 < warp_hi && (h0 + kBK / 2 > warp_lo || h0 < sinks);
    }
    float s[R][4];
    if (sees[0] || sees[1]) {
      if (sees[0] && sees[1])
        dot_products<R, DP, 0, 4>(q_rows, k_rows, sc, s);
      else if (sees[0])
        dot_products<R, DP, 0, 2>(q_rows, k_rows, sc, s);
      else
        dot_products<R, DP, 2, 4>(q_rows, k_rows, sc, s);
      // (all rows of the warp see the whole tile: nothing to mask)
      const bool whole = k0 + kBK <= w0 + 1 && (k0 >= window_lo(P.mask, w0 + 2 * R - 1) || k0 + kBK <= sinks);
      float mx[R];
#pragma unroll
      for (int i = 0; i < R; ++i) {
        if (!whole) {
          const int pos = p0 + row(i), row_lo = window_lo(P.mask, pos);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (!key_visible(k0 + tx + 16 * j, pos, row_lo, sinks)) s[i][j] = -INFINITY;
        }
        mx[i] = fmaxf(fmaxf(s[i][0], s[i][1]), fmaxf(s[i][2], s[i][3]));
      }
#pragma unroll
      for (int off = 8; off >= 1; off >>= 1)
#pragma unroll
        for (int i = 0; i < R; ++i) mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], off));
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const float m_new = fmaxf(m[i], mx[i]);
        // exp2f, not the approximation: an f32 result keeps f32's accuracy
        const float corr = m_new == -INFINITY ? 1.f : exp2f(m[i] - m_new), mm = m_new == -INFINITY ? 0.f : m_new;
        float rsum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s[i][j] = exp2f(s[i][j] - mm);
          rsum += s[i][j];
        }
        l[i] = fmaf(l[i], corr, rsum);
        m[i] = m_new;
#pragma unroll
        for (int jj = 0; jj < kOC; ++jj)
#pragma unroll
          for (int c = 0; c < 2; ++c) acc[i][jj][c] = mul2(acc[i][jj][c], twice(corr));
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();  // V is there, K is free
    if (t + 1 < tiles) load_tile(Ks, kb, P.k.sl, t + 1);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (!sees[u]) continue;
      __syncwarp();  // the other half's probabilities are read
#pragma unroll
      for (int j = 2 * u; j < 2 * u + 2; ++j)
#pragma unroll
        for (int i = 0; i < R; i += 4)
          *reinterpret_cast<float4 *>(&Pt[(tx + 16 * (j - 2 * u)) * kLdP + R * ty + i]) =
              make_float4(s[i][j], s[i + 1][j], s[i + 2][j], s[i + 3][j]);
      __syncwarp();
      const int h0 = k0 + u * (kBK / 2);
      int from = h0 < sinks ? 0 : warp_lo - h0, to = warp_hi - h0;  // (the rest's probabilities are 0)
      from = from > 0 ? from & ~7 : 0;
      to = to < kBK / 2 ? (to + 7) & ~7 : kBK / 2;
      const float *v = Vs + u * (kBK / 2) * kLd + 4 * tx, *pr = Pt + R * ty;
      for (int kk = from; kk < to; kk += 8)
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          float4 pv[R / 4];
          ulonglong2 vr[kOC];
#pragma unroll
          for (int i = 0; i < R / 4; ++i) pv[i] = *reinterpret_cast<const float4 *>(pr + (kk + x) * kLdP + 4 * i);
#pragma unroll
          for (int jj = 0; jj < kOC; ++jj)
            vr[jj] = *reinterpret_cast<const ulonglong2 *>(v + (kk + x) * kLd + 64 * jj);
#pragma unroll
          for (int i = 0; i < R; ++i) {
            const float4 f = pv[i / 4];
            const uint64_t p2 = twice(i % 4 == 0 ? f.x : i % 4 == 1 ? f.y : i % 4 == 2 ? f.z : f.w);
#pragma unroll
            for (int jj = 0; jj < kOC; ++jj) {
              acc[i][jj][0] = fma2(p2, vr[jj].x, acc[i][jj][0]);
              acc[i][jj][1] = fma2(p2, vr[jj].y, acc[i][jj][1]);
            }
          }
        }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  HiddenBad hidden = {-1, -1};
  bool looked = false;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = q0 + row(i);
#pragma unroll
    for (int off = 8; off >= 1; off >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], off);
    const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];
    bool bad = false;
#pragma unroll
    for (int jj = 0; jj < kOC; ++jj) {
      const float2 x01 = split2(acc[i][jj][0]), x23 = split2(acc[i][jj][1]);
      const float x[4] = {x01.x * inv, x01.y * inv, x23.x * inv, x23.y * inv};
      const int d = 64 * jj + 4 * tx;
      if (r < m_rows && d < D) {
        T out[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          out[c] = from_f32<T>(x[c]);
          bad |= d + c < D && !isfinite(x[c]);
        }
        T *to = ob + r * P.o.sl + d;
        if constexpr (kVec && sizeof(T) == 4) {
          *reinterpret_cast<float4 *>(to) = make_float4(x[0], x[1], x[2], x[3]);
        } else if constexpr (kVec) {
          *reinterpret_cast<uint2 *>(to) = *reinterpret_cast<const uint2 *>(out);
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (d + c < D) to[c] = out[c];
        }
      }
    }
    // rows i of the warp's two groups, redone by the whole warp where a value
    // that the row does not see may be the cause (not its own scores: see l)
    const unsigned any = __ballot_sync(0xffffffffu, bad && l[i] == l[i]);
    if (any) {
      if (!looked) {
        // (the tile in which the window begins holds keys in front of it too)
        const int front = w_first * kBK > sinks ? w_first * kBK : sinks;
        hidden = hidden_bad<T>(vb, P.v.sl, D, w0, hi, front, window_lo(P.mask, w1));
        looked = true;
      }
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const int at = p0 + row(i) - ty + g;
        if ((any & (g ? 0xffff0000u : 0x0000ffffu)) && hidden.meets(at, window_lo(P.mask, at))) {
          const int rr = r - ty + g, pos = n - m_rows + rr;
          __syncwarp();
          attention_row<T>(qb + rr * P.q.sl, kb, vb, ob + rr * P.o.sl, P.k.sl, P.v.sl, D, pos, window_lo(P.mask, pos),
                           sinks, sc);
        }
      }
    }
  }
}

template <typename T, int DP, bool kVec>
cudaError_t launch_simt(const AttnProblem &p, cudaStream_t stream) {
  using G = Simt<T, DP>;
  auto kern = window_simt_kernel<T, DP, kVec>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, G::kSmem);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
  if (e != cudaSuccess) return e;
  const int q_tiles = (p.mask.Lq + kBQ - 1) / kBQ;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(static_cast<int64_t>(q_tiles) * p.B * p.H));
  cfg.blockDim = dim3(G::kThreads);
  cfg.dynamicSmemBytes = G::kSmem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kern, p, q_tiles);
  return e != cudaSuccess ? e : cudaGetLastError();
}

template <typename T, bool kVec>
cudaError_t launch_simt_d(const AttnProblem &p, cudaStream_t stream) {
  if (p.D <= 64) return launch_simt<T, 64, kVec>(p, stream);
  if (p.D <= 128) return launch_simt<T, 128, kVec>(p, stream);
  return launch_simt<T, 256, kVec>(p, stream);
}

bool rows_on_16_bytes(const View4 &v, int64_t el) {
  return (reinterpret_cast<uintptr_t>(v.p) & 15) == 0 && v.sb * el % 16 == 0 && v.sh * el % 16 == 0 &&
         v.sl * el % 16 == 0;
}

template <typename T>
cudaError_t launch_simt_t(const AttnProblem &p, cudaStream_t stream) {
  constexpr int64_t el = sizeof(T);
  const bool vec = p.D * el % 16 == 0 && rows_on_16_bytes(p.q, el) && rows_on_16_bytes(p.k, el) &&
                   rows_on_16_bytes(p.v, el) && rows_on_16_bytes(p.o, el);
  return vec ? launch_simt_d<T, true>(p, stream) : launch_simt_d<T, false>(p, stream);
}

}  // namespace

bool window_simt_supported(const AttnProblem &p) {
  return p.D >= 1 && p.D <= 256 &&
         (static_cast<int64_t>(p.mask.Lq) + kBQ - 1) / kBQ * p.B * static_cast<int64_t>(p.H) <= INT32_MAX;
}

cudaError_t window_simt_launch(const AttnProblem &p, cudaStream_t stream) {
  if (p.B == 0 || p.H == 0 || p.mask.Lq == 0) return cudaSuccess;
  if (p.dtype == LLK_DTYPE_FP32) return launch_simt_t<float>(p, stream);
  if (p.dtype == LLK_DTYPE_FP16) return launch_simt_t<__half>(p, stream);
  return launch_simt_t<__nv_bfloat16>(p, stream);
}

}  // namespace llk_b200
