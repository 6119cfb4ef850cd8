// window_attention_rows.cu -- llk.window_attention in f32 for few query rows
// over many keys, split along the keys.
//
// The same sums as window_attention.cu's, all in f32 on the CUDA cores.  What
// bounds it is reading K and V once, so a CTA takes up to 8 rows that share a
// key head (query heads of its group times queries; 4 where there are no more)
// and a share of the blocks of 16 keys that any of them sees; its warps take
// blocks in turn, each with its own two stages of cp.async copies and its own
// running maximum and sum, and no barrier until they join.  Scores: a lane has
// one key and half of d (rows of K pitched by 4 banks, so the 16 rows' pieces do
// not collide).
// Output: a lane has DP / 32 columns, the probabilities come back through
// shared memory.  Shares of a block of rows are joined by combine_kernel.
//
// Measured (D = 128): 16 x 32 heads over 8, one token over 4096 keys: 127 us,
// 537 MB at 0.65 of the measured HBM rate; with 8 rows 183 us, the FMA and
// shared-memory instructions of one warp a scheduler and a half.  One sequence
// of 8192 keys: 27 us.  (Tiles of 64 rows: 1049 and 977 us.)
#include <cuda.h>
#include <cuda_runtime.h>

#include "attn_common.cuh"

namespace llk_b200 {

namespace {

constexpr int kKeys = 16;

template <int DP, int R>
struct Geo {
  static constexpr int kRows = R;
  static constexpr int kWarps = DP > 128 ? 3 : DP > 64 ? 6 : 4;
  static constexpr int kLd = DP + 4, kC = DP / 32;
  static constexpr int kStage = 2 * kKeys * kLd;          // floats: K, then V
  static constexpr int kWarp = 2 * kStage + kKeys * kRows; // and the probabilities [key][row]
  static constexpr int kSmem = (kRows * DP + kWarps * kWarp) * static_cast<int>(sizeof(float));
  static constexpr int kCtas = DP > 64 ? 1 : 3;           // of an SM
  static_assert(kCtas * (kSmem + 1152) <= 228 * 1024, "shared memory");
  // lane's column c
  static __device__ __forceinline__ int col(int lane, int c) {
    return DP == 64 ? 2 * lane + c : c / 4 * 128 + 4 * lane + c % 4;
  }
};

struct Params {
  AttnProblem p;
  int splits, row_blocks;
  float2 *part_ml;  // [segments, splits, R] (maximum, sum)
  float *part_o;    // [segments, splits, R, DP]
};

// Row r of a segment (sequence, key head, block of rows).
struct Row {
  int64_t q, o;  // element offsets
  int pos;       // -1 for a row that is not there
  bool there;
};
__device__ __forceinline__ Row row_of(const AttnProblem &P, int b, int hk, int at, int n, int m) {
  const int g = P.H / P.Hkv, i = at / g, h = hk * g + (at - i * g);
  Row w;
  w.there = i < m;
  w.q = b * P.q.sb + h * P.q.sh + i * P.q.sl;
  w.o = b * P.o.sb + h * P.o.sh + i * P.o.sl;
  w.pos = w.there ? n - m + i : -1;
  return w;
}

// Writes one row, of a sequence of n keys and m queries, from its sums x over all
// shares (lane: columns lane + 32 i); one that a value it does not see may have
// made non-finite is redone key by key.
template <int DP>
__device__ __forceinline__ void write_row(const AttnProblem &P, int b, int hk, int n, int m, const Row &w,
                                          const float (&x)[DP / 32], float l) {
  const int lane = threadIdx.x & 31;
  float *o = static_cast<float *>(P.o.p) + w.o;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < DP / 32; ++i) {
    const int d = lane + 32 * i;
    if (d < P.D) {
      o[d] = x[i] * inv;
      bad |= !isfinite(x[i] * inv);
    }
  }
  if (l == l && __any_sync(0xffffffffu, bad)) {
    const float *v = static_cast<const float *>(P.v.p) + b * P.v.sb + hk * P.v.sh;
    const int lo = window_lo(P.mask, w.pos);
    if (redo_row<float, false>(v, P.v.sl, P.mask, P.D, n, m, w.pos, lo, false)) {
      __syncwarp();
      attention_row<float>(static_cast<const float *>(P.q.p) + w.q,
                           static_cast<const float *>(P.k.p) + b * P.k.sb + hk * P.k.sh, v, o, P.k.sl, P.v.sl, P.D,
                           w.pos, lo, P.mask.sinks, P.scale * kLog2e);
    }
  }
}

template <int DP, int R>
__global__ void __launch_bounds__(32 * Geo<DP, R>::kWarps, Geo<DP, R>::kCtas) rows_kernel(const Params A) {
  using G = Geo<DP, R>;
  constexpr int kRows = R;
  extern __shared__ __align__(16) float sm[];
  __shared__ int2 see[kRows];  // (position, first key of the window) of each row
  const AttnProblem &P = A.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float *Qs = sm, *mine = sm + kRows * DP + warp * G::kWarp, *Pt = mine + 2 * G::kStage;
  const int split = blockIdx.x % A.splits, seg = blockIdx.x / A.splits;
  const int rb = seg % A.row_blocks, hk = seg / A.row_blocks % P.Hkv, b = seg / A.row_blocks / P.Hkv;
  const int g = P.H / P.Hkv, D = P.D;

  pdl_launch_dependents();
  pdl_wait();
  int n, m;
  seq_lens(P.mask, b, n, m);
  const int first = rb * kRows / g;
  if (first >= m) return;
  const int last = (rb * kRows + kRows - 1) / g < m ? (rb * kRows + kRows - 1) / g : m - 1;
  const int hi = n - m + last + 1, lo = window_lo(P.mask, n - m + first), sinks = P.mask.sinks;
  const int s_end = sinks < lo ? sinks : lo, wb0 = lo / kKeys, s_blocks = (s_end + kKeys - 1) / kKeys;
  const int nsb = s_blocks < wb0 ? s_blocks : wb0;
  const int blocks = hi > 0 ? nsb + (hi + kKeys - 1) / kKeys - wb0 : 0;
  const int begin = static_cast<int>(static_cast<int64_t>(blocks) * split / A.splits);
  const int end = static_cast<int>(static_cast<int64_t>(blocks) * (split + 1) / A.splits);
  auto key0 = [&](int t) { return (t < nsb ? t : wb0 + t - nsb) * kKeys; };
  const float *kb = static_cast<const float *>(P.k.p) + b * P.k.sb + hk * P.k.sh;
  const float *vb = static_cast<const float *>(P.v.p) + b * P.v.sb + hk * P.v.sh;
  auto load = [&](int t, int stage) {  // keys that no row sees become 0: what lies there may be anything
    const int k0 = key0(t);
    float *to = mine + stage * G::kStage;
#pragma unroll
    for (int e = lane; e < kKeys * DP / 4; e += 32) {
      const int r = e / (DP / 4), c = 4 * (e % (DP / 4)), j = k0 + r;
      const bool in = c < D && j < hi && (j >= lo || j < sinks);
      const int bytes = in ? 16 : 0;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(to + r * G::kLd + c)),
                   "l"(in ? kb + j * P.k.sl + c : kb), "r"(bytes)
                   : "memory");
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(to + (kKeys + r) * G::kLd + c)),
                   "l"(in ? vb + j * P.v.sl + c : vb), "r"(bytes)
                   : "memory");
    }
  };
  if (begin + warp < end) load(begin + warp, 0);
  asm volatile("cp.async.commit_group;" ::: "memory");
  if (threadIdx.x < kRows) {
    const int pos = row_of(P, b, hk, rb * kRows + threadIdx.x, n, m).pos;
    see[threadIdx.x] = make_int2(pos, window_lo(P.mask, pos));
  }
  const float sc = P.scale * kLog2e;
  for (int e = threadIdx.x; e < kRows * DP; e += 32 * G::kWarps) {
    const int r = e / DP, d = e % DP;
    const Row w = row_of(P, b, hk, rb * kRows + r, n, m);
    Qs[e] = w.there && d < D ? static_cast<const float *>(P.q.p)[w.q + d] * sc : 0.f;
  }
  __syncthreads();

  float mx[kRows], l[kRows], o[kRows][G::kC];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    mx[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int c = 0; c < G::kC; ++c) o[r][c] = 0.f;
  }
  const int key = lane & 15, half = (lane >> 4) * (DP / 2);
  int stage = 0;
  for (int t = begin + warp; t < end; t += G::kWarps, stage ^= 1) {
    if (t + G::kWarps < end) load(t + G::kWarps, stage ^ 1);
    asm volatile("cp.async.commit_group;\n\tcp.async.wait_group 1;" ::: "memory");
    __syncwarp();
    const float *K = mine + stage * G::kStage, *V = K + kKeys * G::kLd;
    float s[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) s[r] = 0.f;
#pragma unroll 4
    for (int d = 0; d < DP / 2; d += 4) {
      const float4 k = *reinterpret_cast<const float4 *>(K + key * G::kLd + half + d);
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const float4 q = *reinterpret_cast<const float4 *>(Qs + r * DP + half + d);
        s[r] = fmaf(q.x, k.x, fmaf(q.y, k.y, fmaf(q.z, k.z, fmaf(q.w, k.w, s[r]))));
      }
    }
    const int j = key0(t) + key;
    float top[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      s[r] += __shfl_xor_sync(0xffffffffu, s[r], 16);
      const int2 row = see[r];
      if (!key_visible(j, row.x, row.y, sinks)) s[r] = -INFINITY;
      top[r] = s[r];
    }
#pragma unroll
    for (int off = 8; off >= 1; off >>= 1)
#pragma unroll
      for (int r = 0; r < kRows; ++r) top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], off));
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
      const float now = fmaxf(mx[r], top[r]), ref = now == -INFINITY ? 0.f : now;
      const float corr = exp2f(mx[r] - ref);  // (of no key yet: 0 times sums of 0)
      mx[r] = now;
      s[r] = exp2f(s[r] - ref);
      l[r] = fmaf(l[r], corr, s[r]);
#pragma unroll
      for (int c = 0; c < G::kC; ++c) o[r][c] *= corr;
    }
    if (lane < kKeys) {
#pragma unroll
      for (int r = 0; r < kRows; r += 4)
        *reinterpret_cast<float4 *>(Pt + key * kRows + r) = make_float4(s[r], s[r + 1], s[r + 2], s[r + 3]);
    }
    __syncwarp();
#pragma unroll 4
    for (int kk = 0; kk < kKeys; ++kk) {
      float p[kRows], v[G::kC];
#pragma unroll
      for (int r = 0; r < kRows; r += 4) {
        const float4 x = *reinterpret_cast<const float4 *>(Pt + kk * kRows + r);
        p[r] = x.x, p[r + 1] = x.y, p[r + 2] = x.z, p[r + 3] = x.w;
      }
      const float *row = V + kk * G::kLd;
      if constexpr (DP == 64) {
        const float2 x = *reinterpret_cast<const float2 *>(row + 2 * lane);
        v[0] = x.x, v[1] = x.y;
      } else {
#pragma unroll
        for (int c = 0; c < G::kC; c += 4) {
          const float4 x = *reinterpret_cast<const float4 *>(row + 32 * c + 4 * lane);
          v[c] = x.x, v[c + 1] = x.y, v[c + 2] = x.z, v[c + 3] = x.w;
        }
      }
#pragma unroll
      for (int r = 0; r < kRows; ++r)
#pragma unroll
        for (int c = 0; c < G::kC; ++c) o[r][c] = fmaf(p[r], v[c], o[r][c]);
    }
    __syncwarp();  // the stage and Pt are free
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  // the warps' sums: [R][DP], then (maximum, sum) of each row
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
#pragma unroll
    for (int off = 8; off >= 1; off >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], off);
#pragma unroll
    for (int c = 0; c < G::kC; ++c) mine[r * DP + G::col(lane, c)] = o[r][c];
    if (lane == 0) {
      mine[R * DP + 2 * r] = mx[r];
      mine[R * DP + 2 * r + 1] = l[r];
    }
  }
  __syncthreads();
  for (int r = warp; r < kRows; r += G::kWarps) {
    const Row w = row_of(P, b, hk, rb * kRows + r, n, m);
    if (!w.there) continue;
    const float *parts = sm + kRows * DP;
    float top = -INFINITY, sum = 0.f, x[DP / 32];
#pragma unroll
    for (int i = 0; i < G::kWarps; ++i) top = fmaxf(top, parts[i * G::kWarp + kRows * DP + 2 * r]);
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) x[i] = 0.f;
#pragma unroll
    for (int i = 0; i < G::kWarps; ++i) {
      const float *part = parts + i * G::kWarp;
      const float f = top == -INFINITY ? 0.f : exp2f(part[kRows * DP + 2 * r] - top);
      sum = fmaf(f, part[kRows * DP + 2 * r + 1], sum);
#pragma unroll
      for (int c = 0; c < DP / 32; ++c) x[c] = fmaf(f, part[r * DP + lane + 32 * c], x[c]);
    }
    if (A.splits == 1) {
      write_row<DP>(P, b, hk, n, m, w, x, sum);
    } else {
      const int64_t at = static_cast<int64_t>(blockIdx.x) * kRows + r;
      if (lane == 0) A.part_ml[at] = make_float2(top, sum);
#pragma unroll
      for (int c = 0; c < DP / 32; ++c) A.part_o[at * DP + lane + 32 * c] = x[c];
    }
  }
}

// Joins the shares of a segment: CTA a segment, warp a row.
template <int DP, int R>
__global__ void __launch_bounds__(32 * R) combine_kernel(const Params A) {
  constexpr int kRows = R;
  const AttnProblem &P = A.p;
  const int r = threadIdx.x >> 5, lane = threadIdx.x & 31, seg = blockIdx.x;
  const int rb = seg % A.row_blocks, hk = seg / A.row_blocks % P.Hkv, b = seg / A.row_blocks / P.Hkv;
  pdl_launch_dependents();
  pdl_wait();
  int n, m;
  seq_lens(P.mask, b, n, m);
  const Row w = row_of(P, b, hk, rb * kRows + r, n, m);
  if (!w.there) return;
  const int64_t at = static_cast<int64_t>(seg) * A.splits * kRows + r;
  float top = -INFINITY, sum = 0.f, x[DP / 32];
  for (int s = 0; s < A.splits; ++s) top = fmaxf(top, A.part_ml[at + s * kRows].x);
#pragma unroll
  for (int c = 0; c < DP / 32; ++c) x[c] = 0.f;
#pragma unroll 4
  for (int s = 0; s < A.splits; ++s) {
    const float2 ml = A.part_ml[at + s * kRows];
    const float f = top == -INFINITY ? 0.f : exp2f(ml.x - top);
    sum = fmaf(f, ml.y, sum);
#pragma unroll
    for (int c = 0; c < DP / 32; ++c) x[c] = fmaf(f, A.part_o[(at + s * kRows) * DP + lane + 32 * c], x[c]);
  }
  // (a share whose scores are all NaN keeps the maximum -inf, but 0 * NaN is NaN)
  write_row<DP>(P, b, hk, n, m, w, x, sum);
}

template <int DP, int R>
cudaError_t launch_rows(const Params &a, int segments, cudaStream_t stream) {
  using G = Geo<DP, R>;
  auto kern = rows_kernel<DP, R>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, G::kSmem);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(static_cast<int64_t>(segments) * a.splits));
  cfg.blockDim = dim3(32 * G::kWarps);
  cfg.dynamicSmemBytes = G::kSmem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kern, a);
  if (e == cudaSuccess && a.splits > 1) {
    cfg.gridDim = dim3(static_cast<unsigned>(segments));
    cfg.blockDim = dim3(32 * R);
    cfg.dynamicSmemBytes = 0;
    e = cudaLaunchKernelEx(&cfg, combine_kernel<DP, R>, a);
  }
  return e != cudaSuccess ? e : cudaGetLastError();
}

int64_t segments_of(const AttnProblem &p, int64_t row_blocks) { return static_cast<int64_t>(p.B) * p.Hkv * row_blocks; }

}  // namespace

bool rows_supported(const AttnProblem &p) {
  const auto on16 = [](const View4 &v) {
    return (reinterpret_cast<uintptr_t>(v.p) & 15) == 0 && v.sb % 4 == 0 && v.sh % 4 == 0 && v.sl % 4 == 0;
  };
  const int64_t rows = p.Hkv > 0 ? static_cast<int64_t>(p.H / p.Hkv) * p.mask.Lq : 0;
  return p.dtype == LLK_DTYPE_FP32 && p.D >= 4 && p.D <= 256 && p.D % 4 == 0 && on16(p.k) && on16(p.v) &&
         rows <= (int64_t(1) << 30) && segments_of(p, (rows + 7) / 8) <= (int64_t(1) << 24);
}

// Shares: two CTAs for each place on the SMs, but no share of fewer than two
// blocks a warp.
RowsPlan rows_plan(const AttnProblem &p, int sm_count) {
  RowsPlan s;
  const int dp = p.D <= 64 ? 64 : p.D <= 128 ? 128 : 256;
  const int rows = p.H / p.Hkv * p.mask.Lq, warps = dp > 128 ? 3 : dp > 64 ? 6 : 4;
  s.rows = rows <= 4 ? 4 : 8;
  s.row_blocks = (rows + s.rows - 1) / s.rows;
  int64_t keys = p.mask.Lk;
  if (p.mask.window > 0) {
    const int64_t seen = static_cast<int64_t>(p.mask.window) + p.mask.sinks + s.rows;
    if (seen < keys) keys = seen;
  }
  const int64_t segments = segments_of(p, s.row_blocks), room = 2 * static_cast<int64_t>(sm_count) * (dp == 64 ? 3 : 1);
  const int64_t most = keys / (kKeys * 2 * warps);
  int64_t splits = (room + segments - 1) / segments;
  if (splits > most) splits = most;
  s.splits = static_cast<int>(splits < 1 ? 1 : splits);
  s.ws_bytes = s.splits == 1 ? 0 : static_cast<size_t>(segments) * s.splits * s.rows * (dp * 4 + sizeof(float2));
  return s;
}

cudaError_t rows_launch(const AttnProblem &p, const RowsPlan &plan, void *workspace, cudaStream_t stream) {
  Params a = {};
  a.p = p;
  a.splits = plan.splits;
  a.row_blocks = plan.row_blocks;
  const int segments = static_cast<int>(segments_of(p, plan.row_blocks));
  if (plan.splits > 1) {
    a.part_ml = static_cast<float2 *>(workspace);
    a.part_o = reinterpret_cast<float *>(a.part_ml + static_cast<size_t>(segments) * plan.splits * plan.rows);
  }
  const bool few = plan.rows == 4;
  if (p.D <= 64) return few ? launch_rows<64, 4>(a, segments, stream) : launch_rows<64, 8>(a, segments, stream);
  if (p.D <= 128) return few ? launch_rows<128, 4>(a, segments, stream) : launch_rows<128, 8>(a, segments, stream);
  return few ? launch_rows<256, 4>(a, segments, stream) : launch_rows<256, 8>(a, segments, stream);
}

}  // namespace llk_b200
