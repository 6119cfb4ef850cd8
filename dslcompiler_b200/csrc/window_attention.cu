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
// pair.  Thread (ty, tx) of 16 x 16 owns a 4 x 4 block of scores and 4 rows x
// 4 DP/64 columns of O; row reductions are shuffles over 16 lanes.
#include <cuda.h>
#include <cuda_runtime.h>

#include "attn_common.cuh"

namespace llk_b200 {

namespace {

constexpr int kBQ = 64, kBK = 64, kThreads = 256, kPad = 4;

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
template <typename T, int DP, bool kVec>
__device__ __forceinline__ void load_rows(float *dst, const T *src, int64_t sl, int row0, int begin, int end, int D) {
  constexpr int kLd = DP + kPad;
  if constexpr (kVec && sizeof(T) == 4) {
    for (int e = threadIdx.x; e < kBQ * (DP / 4); e += kThreads) {
      const int r = e / (DP / 4), c = 4 * (e % (DP / 4)), row = row0 + r;
      const bool in = row >= begin && row < end && c < D;
      cp_async16_zfill(dst + r * kLd + c, reinterpret_cast<const float *>(in ? src + row * sl + c : src), in);
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

// kStages 2: the next tile's cp.async copies run while this one computes
// (f32; D <= 128 leaves shared memory for it).
template <typename T, int DP, bool kVec, int kStages>
__global__ void __launch_bounds__(kThreads, 1) window_simt_kernel(const AttnProblem P, int q_tiles) {
  extern __shared__ __align__(16) float sm[];
  constexpr int kLd = DP + kPad, kOC = DP / 64;
  float *Qs = sm;
  float *KV = Qs + kBQ * kLd;                  // kStages x (K tile, V tile)
  float *Pt = KV + kStages * 2 * kBK * kLd;    // [key][row]
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
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
  auto load_tile = [&](int t) {
    float *Ks = KV + (t % kStages) * 2 * kBK * kLd;
    // a sinks' tile ends with the sinks (unless the window begins inside it)
    const int r0 = tile_row(t);
    const int begin = r0 >= s_keys ? lo : 0;
    const int end = t < s_tiles && r0 + kBK <= lo ? (s_keys < hi ? s_keys : hi) : hi;
    load_rows<T, DP, kVec>(Ks, kb, P.k.sl, r0, begin, end, D);
    load_rows<T, DP, kVec>(Ks + kBK * kLd, vb, P.v.sl, r0, begin, end, D);
  };

  load_rows<T, DP, kVec>(Qs, qb, P.q.sl, q0, 0, m_rows, D);
  if (tiles > 0) load_tile(0);
  asm volatile("cp.async.commit_group;" ::: "memory");
  float m[4], l[4], acc[4][kOC][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int j = 0; j < kOC; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) acc[i][j][c] = 0.f;
  }
  const float sc = P.scale * kLog2e;
  for (int t = 0; t < tiles; ++t) {
    if constexpr (kStages == 2) {
      if (t + 1 < tiles) load_tile(t + 1);  // its buffer was last read by tile t-1, before the barrier that ended it
      asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 1;" ::: "memory");
    } else {
      if (t > 0) load_tile(t);
      asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 0;" ::: "memory");
    }
    __syncthreads();
    const float *Ks = KV + (t % kStages) * 2 * kBK * kLd, *Vs = Ks + kBK * kLd;
    const int k0 = tile_row(t);
    float s[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
    float4 a[4], bb[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = *reinterpret_cast<const float4 *>(&Qs[(4 * ty + i) * kLd]);
#pragma unroll
    for (int j = 0; j < 4; ++j) bb[j] = *reinterpret_cast<const float4 *>(&Ks[(tx + 16 * j) * kLd]);
#pragma unroll 4
    for (int d = 0; d < DP; d += 4) {
      // the operands of step d + 4 load while step d computes
      float4 an[4], bn[4];
      const int dn = d + 4 < DP ? d + 4 : d;
#pragma unroll
      for (int i = 0; i < 4; ++i) an[i] = *reinterpret_cast<const float4 *>(&Qs[(4 * ty + i) * kLd + dn]);
#pragma unroll
      for (int j = 0; j < 4; ++j) bn[j] = *reinterpret_cast<const float4 *>(&Ks[(tx + 16 * j) * kLd + dn]);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s[i][j] = fmaf(a[i].x, bb[j].x, s[i][j]);
          s[i][j] = fmaf(a[i].y, bb[j].y, s[i][j]);
          s[i][j] = fmaf(a[i].z, bb[j].z, s[i][j]);
          s[i][j] = fmaf(a[i].w, bb[j].w, s[i][j]);
        }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a[i] = an[i];
        bb[i] = bn[i];
      }
    }
    float p[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int pos = p0 + 4 * ty + i, row_lo = window_lo(P.mask, pos);
      float rmax = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = key_visible(k0 + tx + 16 * j, pos, row_lo, sinks) ? s[i][j] * sc : -INFINITY;
        rmax = fmaxf(rmax, s[i][j]);
      }
#pragma unroll
      for (int off = 8; off >= 1; off >>= 1) rmax = fmaxf(rmax, __shfl_xor_sync(0xffffffffu, rmax, off));
      const float m_new = fmaxf(m[i], rmax);
      // exp2f, not the approximation: an f32 result keeps f32's accuracy
      const float corr = m_new == -INFINITY ? 1.f : exp2f(m[i] - m_new);
      float rsum = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        p[i][j] = s[i][j] == -INFINITY ? 0.f : exp2f(s[i][j] - m_new);
        rsum += p[i][j];
      }
#pragma unroll
      for (int off = 8; off >= 1; off >>= 1) rsum += __shfl_xor_sync(0xffffffffu, rsum, off);
      l[i] = l[i] * corr + rsum;
      m[i] = m_new;
#pragma unroll
      for (int jj = 0; jj < kOC; ++jj)
#pragma unroll
        for (int c = 0; c < 4; ++c) acc[i][jj][c] *= corr;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      *reinterpret_cast<float4 *>(&Pt[(tx + 16 * j) * (kBQ + kPad) + 4 * ty]) =
          make_float4(p[0][j], p[1][j], p[2][j], p[3][j]);
    __syncthreads();
    float4 pr = *reinterpret_cast<const float4 *>(&Pt[4 * ty]);
    float4 vr[kOC];
#pragma unroll
    for (int jj = 0; jj < kOC; ++jj) vr[jj] = *reinterpret_cast<const float4 *>(&Vs[64 * jj + 4 * tx]);
#pragma unroll 8
    for (int kk = 0; kk < kBK; ++kk) {
      const int kn = kk + 1 < kBK ? kk + 1 : kk;
      const float4 prn = *reinterpret_cast<const float4 *>(&Pt[kn * (kBQ + kPad) + 4 * ty]);
      float4 vrn[kOC];
#pragma unroll
      for (int jj = 0; jj < kOC; ++jj) vrn[jj] = *reinterpret_cast<const float4 *>(&Vs[kn * kLd + 64 * jj + 4 * tx]);
      const float pv[4] = {pr.x, pr.y, pr.z, pr.w};
#pragma unroll
      for (int jj = 0; jj < kOC; ++jj) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          acc[i][jj][0] = fmaf(pv[i], vr[jj].x, acc[i][jj][0]);
          acc[i][jj][1] = fmaf(pv[i], vr[jj].y, acc[i][jj][1]);
          acc[i][jj][2] = fmaf(pv[i], vr[jj].z, acc[i][jj][2]);
          acc[i][jj][3] = fmaf(pv[i], vr[jj].w, acc[i][jj][3]);
        }
      }
      pr = prn;
#pragma unroll
      for (int jj = 0; jj < kOC; ++jj) vr[jj] = vrn[jj];
    }
    __syncthreads();  // Pt and this stage's K / V are free
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = q0 + 4 * ty + i;
    const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];
    bool bad = false;
#pragma unroll
    for (int jj = 0; jj < kOC; ++jj)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int d = 64 * jj + 4 * tx + c;
        const float r = acc[i][jj][c] * inv;
        if (row < m_rows && d < D) {
          ob[row * P.o.sl + d] = from_f32<T>(r);
          bad |= !isfinite(r);
        }
      }
    // rows 4 ty + i of the warp's two groups, redone by the whole warp
    const unsigned any = __ballot_sync(0xffffffffu, bad);
    if (any) {
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        if (any & (g ? 0xffff0000u : 0x0000ffffu)) {
          const int r = q0 + 4 * ((ty & ~1) + g) + i, pos = n - m_rows + r;
          __syncwarp();
          attention_row<T>(qb + r * P.q.sl, kb, vb, ob + r * P.o.sl, P.k.sl, P.v.sl, D, pos, window_lo(P.mask, pos),
                           sinks, sc);
        }
      }
    }
  }
}

template <typename T, int DP, bool kVec, int kStages>
cudaError_t launch_simt(const AttnProblem &p, cudaStream_t stream) {
  const int smem = ((kBQ + 2 * kStages * kBK) * (DP + kPad) + kBK * (kBQ + kPad)) * static_cast<int>(sizeof(float));
  auto kern = window_simt_kernel<T, DP, kVec, kStages>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  const int q_tiles = (p.mask.Lq + kBQ - 1) / kBQ;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(static_cast<int64_t>(q_tiles) * p.B * p.H));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kern, p, q_tiles);
  return e != cudaSuccess ? e : cudaGetLastError();
}

template <typename T, bool kVec>
cudaError_t launch_simt_d(const AttnProblem &p, cudaStream_t stream) {
  constexpr int kSt = kVec && sizeof(T) == 4 ? 2 : 1;
  if (p.D <= 64) return launch_simt<T, 64, kVec, kSt>(p, stream);
  if (p.D <= 128) return launch_simt<T, 128, kVec, kSt>(p, stream);
  return launch_simt<T, 256, kVec, 1>(p, stream);
}

bool rows_on_16_bytes(const View4 &v, int64_t el) {
  return (reinterpret_cast<uintptr_t>(v.p) & 15) == 0 && v.sb * el % 16 == 0 && v.sh * el % 16 == 0 &&
         v.sl * el % 16 == 0;
}

template <typename T>
cudaError_t launch_simt_t(const AttnProblem &p, cudaStream_t stream) {
  constexpr int64_t el = sizeof(T);
  const bool vec = p.D * el % 16 == 0 && rows_on_16_bytes(p.q, el) && rows_on_16_bytes(p.k, el) &&
                   rows_on_16_bytes(p.v, el);
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
