// window_attention_tc.cu -- llk.window_attention for prompts in bf16 / f16 on
// the tensor cores (tcgen05, TMEM, TMA).
//
//   S = Q K^T,  P = 2^(scale log2 e S - m),  O = O + P V,  l = l + sum P
// per key tile, with the running reference m of the softmax (a row's maximum,
// or up to 2^8 below it: see kSlack) and O / l at the end.
//
// One CTA an SM takes 256 query rows of one head after another, as two tiles
// of 128, and sweeps the key tiles that any of the rows sees: the sinks' tiles,
// then the window's.  A query tile skips the key tiles that none of its own
// rows sees.  The next rows' queries and keys are on their way while these are
// finished (started anew, a CTA waits 4000 clocks for its first scores).
//   warps 0-3, 4-7  softmax of query tile 0 / 1, one thread a row: S from
//                   TMEM to registers, P back to TMEM in 16 bits, O's rescale
//                   when the reference moves, the output
//   warps 8, 9      tcgen05.mma of query tile 0 / 1: S = Q K^T (both operands
//                   in shared memory), O += P V (P from TMEM)
//   warp 10         TMA: Q once, K and V tiles through one ring of stages
// TMEM columns: O0, O1, S0, S1, P0, P1.  S and P do not share columns, so
// the next S of a query tile is computed while its softmax runs on the
// registers, and the softmax warps never wait for the tensor core; that, and
// 512 columns, make the key tile 80 wide at D = 128 (80 + 40 + 128 columns a
// query tile) and 96 at D = 64.
//
// 4 D FLOP and one exponential a pair: at D = 128 the tensor core (8192 FLOP
// a clock and SM) and the exponential unit (16 a clock and SM) need the same
// 512 clocks for 128 x 64 pairs.  Neither is what bounds it: under a window of
// 1024 the tensor core works 44 % of the clocks and an instruction issues in
// 39 %; a key tile of both query tiles takes 2000 to 2300 clocks, and a softmax
// warp's chain (wait, TMEM load, maximum, exponentials, TMEM store, arrive) is
// as long as that.
//
// P is rounded to the inputs' 16 bits, as the tensor core takes it, and its sum
// is not: the error against 64 bits is 0.0018 (bf16) and 0.00023 (f16) of the
// result's size, where rounding the result alone makes 0.0017 and 0.00021.
//
// Measured (bf16, D = 128): 32 heads over 8 of keys, 8192 tokens, window 4096
// and 4 sinks: 371 us at 1965 MHz, 0.68 of the time of the products at the
// measured bf16 rate, 251 us; called for seconds the power limit sets the clock,
// 437 us at 1670 MHz.  32 heads, 4096 tokens, window 1024: 86 us for 37, for
// seconds 98 us at 1730 MHz (512 items on 148 SMs: four rounds are paid, 3.46
// worked).  Tried and slower: key tiles of 64 (569 for then 497 us), one commit
// for several products (107 for 92), exponentials partly by a polynomial on the
// FMA pipe (95 to 91 for 87), registers moved from the MMA warps to the softmax
// (85 for 86: no difference).
#include <cuda.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include "attn_common.cuh"

namespace llk_b200 {

namespace {

constexpr int kBM = 128;                // rows of a query tile
constexpr int kThreads = 352;
constexpr uint64_t kWaitLimitNs = 2000000000ull;
// The reference m may lag a row's maximum by up to this power of two before O
// is rescaled: P stays below 2^8, far inside f16, its relative rounding is
// the same, and the f32 sums do not mind.
constexpr float kSlack = 8.f;

struct TcMaps {
  CUtensorMap q, k, v;
};

struct TcArgs {
  AttnProblem p;
  int q_blocks;
  // 0 for a broadcast dimension of the maps, else 1
  int qb, qh, kb, kh, vb, vh;
  int vec_o;  // output rows start on 16 bytes
  int *status;
};

template <int D>
struct Cfg {
  static constexpr int kKT = D == 128 ? 80 : 96;       // keys of a tile
  static constexpr int kSlabs = D / 64;
  static constexpr int kQBytes = kBM * D * 2;          // one query tile
  static constexpr int kStageBytes = kKT * D * 2;      // one K or V tile
  static constexpr int kStages = D == 128 ? 7 : 8;
  static constexpr int kColO = 0, kColS = 2 * D, kColP = kColS + 2 * kKT, kCols = 512;
  static_assert(kColP + kKT <= kCols, "TMEM columns");
};

struct Tail {
  uint64_t q_full[2], q_empty[2], o_free[2], kv_full[8], kv_empty[8], s_full[2], s_empty[2], p_ready[2], pv_done[2], landed, mma_done;
  uint32_t tmem;
  int abort;
  int bad;  // some row of the CTA is not finite
};

__device__ __forceinline__ uint64_t pack_f32x2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack_f32x2(uint64_t v, float &a, float &b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

__device__ __forceinline__ void tma_load_4d(void *dst, const CUtensorMap *map, uint64_t *bar, int c0, int c1, int c2,
                                            int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], "
      "[%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}

// D[tmem] (+)= A[tmem, 16-bit pairs along K in a column] * B[smem].
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}

// One lane of the warp, the same one every time (the compiler knows that it
// is one, and keeps the issuing code in uniform registers).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p != 0;
}

__device__ __forceinline__ void tmem_st_x8(uint32_t t, const uint32_t *r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(t), "r"(r[0]), "r"(r[1]),
               "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__host__ __device__ constexpr uint32_t idesc_16(bool bf16, uint32_t m, uint32_t n, bool b_mn_major) {
  const uint32_t t = bf16 ? 1u : 0u;
  return (1u << 4) | (t << 7) | (t << 10) | ((b_mn_major ? 1u : 0u) << 16) | ((n >> 3) << 17) | ((m >> 4) << 24);
}

template <bool kBf16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  uint32_t r;
  if constexpr (kBf16) {
    asm("cvt.rn.bf16x2.f32 %0, %2, %1;" : "=r"(r) : "f"(lo), "f"(hi));
  } else {
    asm("cvt.rn.f16x2.f32 %0, %2, %1;" : "=r"(r) : "f"(lo), "f"(hi));
  }
  return r;
}

// The key tiles of a CTA: s_tiles of sinks, then from the window's first.
struct Sweep {
  int b, h, q0;  // the rows: sequence, head, first query
  int m, rows;   // queries of the sequence, of these rows (may be <= 0 or > 256)
  int p0, hi, lo, s_keys, s_tiles, w_first, tiles, sinks;
  // of each query tile: the window's tiles that some row sees, [from, to) (no
  // row: to = -1); and the tiles that hold a sink, [0, sink_to)
  int from0, from1, to0, to1, sink_to;
  __device__ __forceinline__ int key0(int j, int kt) const { return (j < s_tiles ? j : w_first + j - s_tiles) * kt; }
  __device__ __forceinline__ bool any(int t) const { return (t ? to1 : to0) > 0; }
  __device__ __forceinline__ bool active(int t, int j) const {
    return j < (t ? to1 : to0) && (j >= (t ? from1 : from0) || j < sink_to);
  }
  // values of the tile at k0 that no row sees
  __device__ __forceinline__ bool dead(int k0, int kt) const { return k0 + kt > hi || (k0 < lo && k0 + kt > s_keys); }
  __device__ __forceinline__ bool dead_key(int key) const { return key >= hi || (key < lo && key >= s_keys); }
};

// A place in the ring of stages.
template <int ST>
struct Ring {
  int stage = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next() {
    if (++stage == ST) {
      stage = 0;
      phase ^= 1;
    }
  }
};

// The rows of one item (256 from q0 on) whose written result is not finite:
// those that a value they do not see may have made so are redone from the
// definition.  By all warps of the CTA, 8 rows at a time, when its last item is
// done: nobody waits for it with a limit, however many rows and keys there are.
template <typename T>
__device__ __noinline__ void redo_item(const AttnProblem &P, int b, int h, int q0) {
  constexpr int kRows = 8;
  const int lane = threadIdx.x & 31, hk = h / (P.H / P.Hkv), sinks = P.mask.sinks, D = P.D;
  const T *v = static_cast<const T *>(P.v.p) + b * P.v.sb + hk * P.v.sh;
  T *o = static_cast<T *>(P.o.p) + b * P.o.sb + h * P.o.sh;
  int n, m;
  seq_lens(P.mask, b, n, m);
  // the keys that the CTA swept for these rows, as in the kernel's plan
  const int end = m < q0 + 2 * kBM ? m : q0 + 2 * kBM, p0 = n - m + q0, hi = n - m + end;
  const int lo = window_lo(P.mask, p0), s_keys = sinks < lo ? sinks : lo;
  int infinities = -1;  // among all values of the sweep (not looked yet)
  for (int row = q0 + kRows * (threadIdx.x >> 5); row < end; row += kRows * (kThreads / 32)) {
    const int rows = end - row < kRows ? end - row : kRows, pos = n - m + row;
    unsigned bad = 0, nan = 0;
#pragma unroll
    for (int r = 0; r < kRows; ++r)
#pragma unroll
      for (int d = lane; d < 128; d += 32) {
        const float x = r < rows && d < D ? to_f32(o[static_cast<int64_t>(row + r) * P.o.sl + d]) : 0.f;
        bad |= (fabsf(x) < INFINITY ? 0u : 1u) << r;
        nan |= (x != x ? 1u : 0u) << r;
      }
    bad = __reduce_or_sync(0xffffffffu, bad);
    if (!bad) continue;
    nan = __reduce_or_sync(0xffffffffu, nan);
    const HiddenBad hidden = hidden_bad<T>(v, P.v.sl, D, pos, hi, lo > sinks ? lo : sinks,
                                           window_lo(P.mask, pos + rows - 1));
    for (; bad; bad &= bad - 1) {
      const int r = __ffs(bad) - 1, p = pos + r, row_lo = window_lo(P.mask, p);
      bool again = hidden.meets(p, row_lo);
      if (std::is_same<T, __half>::value && !again && (nan >> r & 1)) {
        // a weight below f16's least times an infinity that the row does see: NaN here, not by the definition
        if (infinities < 0)
          infinities = bad_row<T>(v, P.v.sl, D, 0, s_keys, 1, true) >= 0 ||
                       bad_row<T>(v, P.v.sl, D, lo, hi - lo, 1, true) >= 0;
        again = infinities > 0;
      }
      if (again)
        attention_row<T>(
            static_cast<const T *>(P.q.p) + b * P.q.sb + h * P.q.sh + static_cast<int64_t>(row + r) * P.q.sl,
            static_cast<const T *>(P.k.p) + b * P.k.sb + hk * P.k.sh, v, o + static_cast<int64_t>(row + r) * P.o.sl,
            P.k.sl, P.v.sl, D, p, row_lo, sinks, P.scale * kLog2e);
    }
  }
}

template <int D, bool kBf16>
__global__ void __launch_bounds__(kThreads, 1)
    window_tc_kernel(const __grid_constant__ TcMaps maps, const __grid_constant__ TcArgs A) {
  using C = Cfg<D>;
  constexpr int KT = C::kKT, ST = C::kStages;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t *smem_kv = smem + 2 * C::kQBytes;
  Tail *st = reinterpret_cast<Tail *>(smem_kv + ST * C::kStageBytes);
  const AttnProblem &P = A.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&st->q_full[i], 1);
      mbar_init(&st->q_empty[i], 1);
      mbar_init(&st->o_free[i], kBM);
      mbar_init(&st->s_full[i], 1);
      mbar_init(&st->s_empty[i], kBM);
      mbar_init(&st->p_ready[i], kBM);
      mbar_init(&st->pv_done[i], 1);
    }
    for (int i = 0; i < ST; ++i) {
      mbar_init(&st->kv_full[i], 1);
      mbar_init(&st->kv_empty[i], 2);
    }
    mbar_init(&st->landed, 1);
    mbar_init(&st->mma_done, 2);
    st->abort = 0;
    st->bad = 0;
    fence_mbar_init();
    tma_prefetch_desc(&maps.q);
    tma_prefetch_desc(&maps.k);
    tma_prefetch_desc(&maps.v);
  }
  if (warp == 9) {
    tmem_alloc(&st->tmem, C::kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t tmem = st->tmem;
  volatile int *abort = &st->abort;

  // This CTA's blocks of rows: the last ones of the sequences, which have the
  // most keys, first, and every other round of them in reverse.
  const int BH = P.B * P.H, items = A.q_blocks * BH;
  auto item_of = [&](int round) {
    return round * static_cast<int>(gridDim.x) +
           static_cast<int>(round & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
  };
  auto plan = [&](int item) {
    Sweep w;
    const int bh = item % BH;
    w.b = bh / P.H;
    w.h = bh - w.b * P.H;
    w.q0 = (A.q_blocks - 1 - item / BH) * 2 * kBM;
    int n;
    seq_lens(P.mask, w.b, n, w.m);
    w.sinks = P.mask.sinks;
    w.rows = w.m - w.q0;
    w.p0 = n - w.m + w.q0;
    w.hi = w.p0 + (w.rows < 2 * kBM ? w.rows : 2 * kBM);
    w.lo = window_lo(P.mask, w.p0);
    w.s_keys = w.sinks < w.lo ? w.sinks : w.lo;
    w.w_first = w.lo / KT;
    const int s_all = (w.s_keys + KT - 1) / KT, s_sinks = (w.sinks + KT - 1) / KT;
    w.s_tiles = s_all < w.w_first ? s_all : w.w_first;
    const int end_tile = w.hi > 0 ? (w.hi + KT - 1) / KT : 0;
    w.tiles = w.rows > 0 && end_tile > w.w_first ? w.s_tiles + end_tile - w.w_first : 0;
    const int shift = w.s_tiles - w.w_first;
    auto last_tile = [&](int first) {
      const int last = first + kBM - 1 < w.hi - 1 ? first + kBM - 1 : w.hi - 1;
      return w.tiles > 0 && last >= first && last >= 0 ? shift + last / KT + 1 : -1;
    };
    w.from0 = shift + w.lo / KT;
    w.from1 = shift + window_lo(P.mask, w.p0 + kBM) / KT;
    w.to0 = last_tile(w.p0);
    w.to1 = last_tile(w.p0 + kBM);
    w.sink_to = w.s_tiles + (s_sinks > w.w_first ? s_sinks - w.w_first : 0);
    return w;
  };
  const int g = P.H / P.Hkv;

  if (warp == 10) {
    // ------------------------------------------------------------ producer
    // K and V tiles share the ring in the order K0, K1, V0, K2, V1, ..  The
    // whole warp follows, one lane issues.  Rows of V that no row of the CTA
    // sees may hold anything (a weight of 0 does not undo a NaN): such a tile
    // lands on a barrier of the warp's own, the warp makes the rows zero and
    // only then says that the stage is full.
    bool ok = true;
    Ring<ST> ring;
    int issued = 0;
    uint32_t landings = 0, queries[2] = {0, 0};
    auto wait = [&](uint64_t *bar, uint32_t phase) {
      const bool r = mbar_wait_bounded(bar, phase & 1, abort, LLK_ERR_TIMEOUT, kWaitLimitNs);
      return static_cast<bool>(__all_sync(0xffffffffu, r));
    };
    for (int round = 0; ok && item_of(round) < items; ++round) {
      const Sweep w = plan(item_of(round));
      const int n = w.tiles, hk = w.h / g;
      if (n == 0) continue;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if (!ok || !w.any(t)) continue;
        if (queries[t] > 0 && !(ok = wait(&st->q_empty[t], queries[t] - 1))) continue;
        if (elect_one()) {
          mbar_arrive_expect_tx(&st->q_full[t], C::kQBytes);
          for (int s = 0; s < C::kSlabs; ++s)
            tma_load_4d(smem + t * C::kQBytes + s * kBM * 128, &maps.q, &st->q_full[t], 64 * s, w.q0 + kBM * t,
                        w.h * A.qh, w.b * A.qb);
        }
        __syncwarp();
        ++queries[t];
      }
      auto load = [&](const CUtensorMap *map, int j, int ch, int cb, uint64_t *full) {
        if (issued >= ST && !wait(&st->kv_empty[ring.stage], ring.phase ^ 1)) return false;
        if (elect_one()) {
          uint8_t *dst = smem_kv + ring.stage * C::kStageBytes;
          mbar_arrive_expect_tx(full, C::kStageBytes);
          for (int s = 0; s < C::kSlabs; ++s) tma_load_4d(dst + s * KT * 128, map, full, 64 * s, w.key0(j, KT), ch, cb);
        }
        __syncwarp();
        ++issued;
        return true;
      };
      ok = ok && load(&maps.k, 0, hk * A.kh, w.b * A.kb, &st->kv_full[ring.stage]);
      ring.next();
      for (int j = 0; j < n && ok; ++j) {
        if (j + 1 < n) {
          ok = load(&maps.k, j + 1, hk * A.kh, w.b * A.kb, &st->kv_full[ring.stage]);
          ring.next();
        }
        const int k0 = w.key0(j, KT);
        const bool dead = w.dead(k0, KT);
        if (!ok || !(ok = load(&maps.v, j, hk * A.vh, w.b * A.vb, dead ? &st->landed : &st->kv_full[ring.stage]))) break;
        if (dead) {
          if (!(ok = wait(&st->landed, landings))) break;
          ++landings;
          uint8_t *v = smem_kv + ring.stage * C::kStageBytes;
          for (int e = lane; e < KT * C::kSlabs * 8; e += 32)
            if (w.dead_key(k0 + (e >> 3) % KT)) *reinterpret_cast<uint4 *>(v + e * 16) = make_uint4(0, 0, 0, 0);
          fence_proxy_async_smem();
          __syncwarp();
          if (elect_one()) mbar_arrive(&st->kv_full[ring.stage]);
        }
        ring.next();
      }
    }
    if (!ok && lane == 0) {
      // the copies in flight land before the CTA's shared memory goes (where
      // nothing is on its way, the wait runs out)
      int dummy = 0;
      for (int t = 0; t < 2; ++t)
        if (queries[t] > 0) mbar_wait_bounded(&st->q_full[t], (queries[t] - 1) & 1, &dummy, 1, 100000000ull);
      dummy = 0;
      mbar_wait_bounded(&st->landed, landings & 1, &dummy, 1, 100000000ull);
      for (int i = issued > ST ? issued - ST : 0; i < issued; ++i) {
        dummy = 0;
        mbar_wait_bounded(&st->kv_full[i % ST], (i / ST) & 1, &dummy, 1, 100000000ull);
      }
    }
    __syncwarp();
  } else if (warp >= 8) {
    // ----------------------------------------------------------------- MMA
    // One lane, for one query tile.  What lies between two products costs more
    // than it looks (the softmax warps take most issue slots, and only about 7
    // products queue up): descriptors are made once, an operand's place is
    // added to the address field (in 16-byte units, its 14 bits hold any
    // address of the CTA), and the ring's places are counted along.  A warp a
    // query tile: products that wait for the tensor core also hold up the
    // exponentials of the softmax warps on their scheduler, and two schedulers
    // share that (with one warp for both tiles its scheduler's softmax warps
    // ran 1000 clocks a key tile behind the others).
    if (elect_one()) {
      const int t = warp - 8;
      const uint64_t q_desc = make_smem_desc_sw128(smem_u32(smem) + t * C::kQBytes, 16, 1024);
      const uint64_t k_desc = make_smem_desc_sw128(smem_u32(smem_kv), 16, 1024);
      const uint64_t v_desc = make_smem_desc_sw128(smem_u32(smem_kv), KT * 128, 1024);
      constexpr uint32_t idesc_s = idesc_16(kBf16, kBM, KT, false), idesc_o = idesc_16(kBf16, kBM, D, true);
      const uint32_t ts = tmem + C::kColS + t * KT, tp = tmem + C::kColP + t * (KT / 2), to = tmem + C::kColO + t * D;
      uint32_t cnt_s = 0, cnt_o = 0, queries = 0;  // score tiles, value tiles, blocks of rows so far
      bool ok = true;
      Ring<ST> ring;
      auto wait = [&](uint64_t *bar, uint32_t phase) {
        if (!mbar_try_wait(bar, phase & 1)) ok = mbar_wait_bounded(bar, phase & 1, abort, LLK_ERR_TIMEOUT, kWaitLimitNs);
        tc_fence_after();
        return ok;
      };
      for (int round = 0; ok && item_of(round) < items; ++round) {
        const Sweep w = plan(item_of(round));
        const int n = w.tiles, last = (t ? w.to1 : w.to0) - 1;
        if (n == 0) continue;
        bool first_s = true, first_o = true;
        auto scores = [&](int j) {
          if (!wait(&st->kv_full[ring.stage], ring.phase)) return;
          if (!w.active(t, j)) {
            mbar_arrive(&st->kv_empty[ring.stage]);  // (of a full stage: not a lap ahead of the copies)
          } else {
            if (first_s && !wait(&st->q_full[t], queries)) return;
            if (cnt_s > 0 && !wait(&st->s_empty[t], cnt_s - 1)) return;
            const uint64_t k_at = k_desc + ring.stage * (C::kStageBytes >> 4);
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk)
              tc_mma_bf16(ts, q_desc + (((kk >> 2) * kBM * 128 + (kk & 3) * 32) >> 4),
                          k_at + (((kk >> 2) * KT * 128 + (kk & 3) * 32) >> 4), idesc_s, kk > 0);
            tc_commit(&st->s_full[t]);
            tc_commit(&st->kv_empty[ring.stage]);
            if (j == last) tc_commit(&st->q_empty[t]);
            ++cnt_s;
            first_s = false;
          }
          ring.next();
        };
        scores(0);
        for (int j = 0; j < n && ok; ++j) {
          if (j + 1 < n) scores(j + 1);
          if (!ok || !wait(&st->kv_full[ring.stage], ring.phase)) break;
          if (!w.active(t, j)) {
            mbar_arrive(&st->kv_empty[ring.stage]);
          } else {
            if (!wait(&st->p_ready[t], cnt_o)) break;
            if (first_o && queries > 0 && !wait(&st->o_free[t], queries - 1)) break;
            const uint64_t v_at = v_desc + ring.stage * (C::kStageBytes >> 4);
#pragma unroll
            for (int kk = 0; kk < KT / 16; ++kk)
              mma_ts(to, tp + kk * 8, v_at + (kk * 2048 >> 4), idesc_o, !first_o || kk > 0);
            tc_commit(&st->pv_done[t]);
            tc_commit(&st->kv_empty[ring.stage]);
            ++cnt_o;
            first_o = false;
          }
          ring.next();
        }
        if (last >= 0) ++queries;
      }
      // every MMA of this CTA has finished before TMEM is released
      tc_commit(&st->mma_done);
      int dummy = 0;
      mbar_wait_bounded(&st->mma_done, 0, &dummy, 1, 100000000ull);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------- softmax
    using T = typename std::conditional<kBf16, __nv_bfloat16, __half>::type;
    const int t = warp >> 2, quarter = warp & 3;
    const int row_in = quarter * 32 + lane;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t ts = t_lane + C::kColS + t * KT, tp = t_lane + C::kColP + t * (KT / 2),
                   to = t_lane + C::kColO + t * D;
    const float sc = P.scale * kLog2e;
    const uint64_t sc2 = pack_f32x2(sc, sc);
    uint32_t cnt = 0;  // score tiles so far
    bool ok = true;
    auto wait = [&](uint64_t *bar, uint32_t phase) {
      const bool r = mbar_try_wait(bar, phase & 1) ||
                     mbar_wait_bounded(bar, phase & 1, abort, LLK_ERR_TIMEOUT, kWaitLimitNs);
      ok = __all_sync(0xffffffffu, r);
      tc_fence_after();
      return ok;
    };
    for (int round = 0; ok && item_of(round) < items; ++round) {
      const Sweep w = plan(item_of(round));
      if (w.rows <= kBM * t) continue;  // no query of this tile: nothing is written
      const int n = w.tiles;
      const int row = w.q0 + kBM * t + row_in, pos = w.p0 + kBM * t + row_in;
      const int row_lo = window_lo(P.mask, pos);
      const int first = w.p0 + kBM * t;  // of the tile's rows that exist, the first and the last position
      const int last = first + kBM - 1 < w.hi - 1 ? first + kBM - 1 : w.hi - 1;
      const int last_lo = window_lo(P.mask, last);
      float m = -INFINITY;
      uint64_t l2 = 0;  // two partial sums
      bool begun = false;
      for (int j = 0; j < n; ++j) {
        if (!w.active(t, j)) continue;
        const int k0 = w.key0(j, KT);
        if (!wait(&st->s_full[t], cnt)) break;
        uint32_t sb[KT];
#pragma unroll
        for (int c = 0; c < KT; c += 16) tmem_ld_32x32b_x16(ts + c, *reinterpret_cast<uint32_t(*)[16]>(&sb[c]));
        tmem_ld_wait();
        tc_fence_before();
        mbar_arrive(&st->s_empty[t]);
        float s[KT];
#pragma unroll
        for (int i = 0; i < KT; ++i) s[i] = __uint_as_float(sb[i]);
        // every row of the tile sees every key of it, or the rows look key by key
        if (!(k0 + KT - 1 <= first && (k0 >= last_lo || k0 + KT <= w.sinks))) {
          auto below = [](int x) { return x <= 0 ? 0u : x >= 32 ? 0xffffffffu : (1u << x) - 1u; };
#pragma unroll
          for (int c = 0; c < KT; c += 32) {
            const uint32_t see = below(pos + 1 - k0 - c) & (~below(row_lo - k0 - c) | below(w.sinks - k0 - c));
#pragma unroll
            for (int i = 0; i < 32 && c + i < KT; ++i)
              if (!(see >> i & 1)) s[c + i] = -INFINITY;
          }
        }
        float mx0 = s[0], mx1 = s[1];
#pragma unroll
        for (int i = 2; i < KT; i += 2) {
          mx0 = fmaxf(mx0, s[i]);
          mx1 = fmaxf(mx1, s[i + 1]);
        }
        const float top = fmaxf(mx0, mx1) * sc;  // scale > 0
        float corr = 1.f;
        bool move = false;
        if (!begun) {
          m = top;
        } else {
          move = __any_sync(0xffffffffu, top > m + kSlack);
          if (move) {
            const float m_new = fmaxf(m, top);
            corr = m_new == -INFINITY ? 1.f : exp2_approx(m - m_new);
            m = m_new;
            float a, c;
            unpack_f32x2(l2, a, c);
            l2 = pack_f32x2(a * corr, c * corr);
          }
        }
        const float ref = m == -INFINITY ? 0.f : m;
        const uint64_t ref2 = pack_f32x2(-ref, -ref);
        uint32_t pk[KT / 2];
#pragma unroll
        for (int i = 0; i < KT; i += 2) {
          float a, c;
          unpack_f32x2(fma_f32x2(pack_f32x2(s[i], s[i + 1]), sc2, ref2), a, c);
          a = exp2_approx(a);
          c = exp2_approx(c);
          l2 = add_f32x2(l2, pack_f32x2(a, c));
          pk[i / 2] = pack16<kBf16>(a, c);
        }
        if (begun) {
          // P's columns are free and O is whole
          if (!wait(&st->pv_done[t], cnt - 1)) break;
          if (move) {
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
              uint32_t x[16];
              tmem_ld_32x32b_x16(to + c, x);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) x[i] = __float_as_uint(__uint_as_float(x[i]) * corr);
              tmem_st_x8(to + c, x);
              tmem_st_x8(to + c + 8, x + 8);
            }
          }
        }
#pragma unroll
        for (int c = 0; c < KT / 2; c += 8) tmem_st_x8(tp + c, pk + c);
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(&st->p_ready[t]);
        ++cnt;
        begun = true;
      }
      // ----------------------------------------------------------- output
      if (!ok || (begun && !wait(&st->pv_done[t], cnt - 1))) break;
      float l0, l1;
      unpack_f32x2(l2, l0, l1);
      const float l = l0 + l1;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const bool mine = row < w.m;
      T *orow = static_cast<T *>(P.o.p) + w.b * P.o.sb + w.h * P.o.sh + static_cast<int64_t>(row) * P.o.sl;
      bool bad = false;
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        uint32_t x[32];
        if (begun) {
          tmem_ld_32x32b_x32(to + c, x);
          tmem_ld_wait();
          if (c + 32 == D) {
            // O is read: the next rows' products may begin
            tc_fence_before();
            mbar_arrive(&st->o_free[t]);
          }
        }
        float y[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          y[i] = begun ? __uint_as_float(x[i]) * inv : 0.f;
          bad |= !(fabsf(y[i]) < INFINITY);
          if constexpr (!kBf16) y[i] = within_f16(y[i]);
        }
        if (mine) {
          if (A.vec_o && c + 32 <= P.D) {
#pragma unroll
            for (int i = 0; i < 32; i += 8)
              *reinterpret_cast<uint4 *>(orow + c + i) =
                  make_uint4(pack16<kBf16>(y[i], y[i + 1]), pack16<kBf16>(y[i + 2], y[i + 3]),
                             pack16<kBf16>(y[i + 4], y[i + 5]), pack16<kBf16>(y[i + 6], y[i + 7]));
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (c + i < P.D) orow[c + i] = from_f32<T>(y[i]);
          }
        }
      }
      if (mine && bad) st->bad = 1;  // (redo_item looks at it when the CTA's items are done)
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kCols);
  }
  if (threadIdx.x == 0 && st->abort != 0) atomicExch(A.status, st->abort);
  if (st->bad && !st->abort)
    for (int round = 0; item_of(round) < items; ++round) {
      const int item = item_of(round), bh = item % BH;
      redo_item<typename std::conditional<kBf16, __nv_bfloat16, __half>::type>(
          P, bh / P.H, bh % P.H, (A.q_blocks - 1 - item / BH) * 2 * kBM);
    }
}

// {D, L, H, B} map of a view with a box of 64 x rows; a broadcast or size-1
// dimension becomes one of size 1 (*f = 0: its coordinate is always 0).
bool encode(PFN_cuTensorMapEncodeTiled_v12000 enc, CUtensorMap *map, bool bf16, const View4 &v, int64_t D, int64_t L,
            int64_t H, int64_t B, int rows, int *fh, int *fb) {
  *fh = H > 1 && v.sh != 0;
  *fb = B > 1 && v.sb != 0;
  const int64_t some = (D * 2 + 15) / 16 * 16;
  cuuint64_t dims[4] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(L), static_cast<cuuint64_t>(*fh ? H : 1),
                        static_cast<cuuint64_t>(*fb ? B : 1)};
  cuuint64_t strides[3] = {static_cast<cuuint64_t>(L > 1 ? v.sl * 2 : some),
                           static_cast<cuuint64_t>(*fh ? v.sh * 2 : some),
                           static_cast<cuuint64_t>(*fb ? v.sb * 2 : some)};
  cuuint32_t box[4] = {64, static_cast<cuuint32_t>(rows), 1, 1}, es[4] = {1, 1, 1, 1};
  return enc(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, v.p, dims, strides, box,
             es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool kBf16>
cudaError_t launch_tc(PFN_cuTensorMapEncodeTiled_v12000 enc, const AttnProblem &p, int *status, int sm_count,
                      cudaStream_t stream) {
  using C = Cfg<D>;
  TcMaps maps;
  TcArgs a = {};
  a.p = p;
  a.q_blocks = (p.mask.Lq + 2 * kBM - 1) / (2 * kBM);
  a.status = status;
  a.vec_o = (reinterpret_cast<uintptr_t>(p.o.p) & 15) == 0 && p.o.sb % 8 == 0 && p.o.sh % 8 == 0 && p.o.sl % 8 == 0;
  if (!encode(enc, &maps.q, kBf16, p.q, p.D, p.mask.Lq, p.H, p.B, kBM, &a.qh, &a.qb) ||
      !encode(enc, &maps.k, kBf16, p.k, p.D, p.mask.Lk, p.Hkv, p.B, C::kKT, &a.kh, &a.kb) ||
      !encode(enc, &maps.v, kBf16, p.v, p.D, p.mask.Lk, p.Hkv, p.B, C::kKT, &a.vh, &a.vb))
    return cudaErrorInvalidValue;
  const int smem = 2 * C::kQBytes + C::kStages * C::kStageBytes + static_cast<int>(sizeof(Tail)) + 1024;
  auto kern = window_tc_kernel<D, kBf16>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  const int64_t items = static_cast<int64_t>(a.q_blocks) * p.B * p.H;
  cfg.gridDim = dim3(static_cast<unsigned>(items < sm_count ? items : sm_count));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kern, maps, a);
  return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace

// What TMA can describe: 16-bit rows on 16 bytes (a row's start needs it, D
// a multiple of 8 with it), D <= 128; a scale that keeps the order of scores (and
// -inf).
bool window_tc_supported(const AttnProblem &p) {
  const auto rows16 = [&](const View4 &v, int64_t L) {
    return (reinterpret_cast<uintptr_t>(v.p) & 15) == 0 && v.sb % 8 == 0 && v.sh % 8 == 0 && v.sl % 8 == 0 &&
           (L <= 1 || v.sl > 0) && v.sl < (int64_t(1) << 38) && v.sh < (int64_t(1) << 38) && v.sb < (int64_t(1) << 38);
  };
  return (p.dtype == LLK_DTYPE_BF16 || p.dtype == LLK_DTYPE_FP16) && p.D % 8 == 0 && p.D <= 128 && p.mask.Lk > 0 &&
         p.scale > 0.f && rows16(p.q, p.mask.Lq) && rows16(p.k, p.mask.Lk) && rows16(p.v, p.mask.Lk) &&
         (static_cast<int64_t>(p.mask.Lq) + 255) / 256 * p.B * p.H <= INT32_MAX / 2;
}

cudaError_t window_tc_launch(void *encode_fn, const AttnProblem &p, int *status, int sm_count, cudaStream_t stream) {
  if (p.B == 0 || p.H == 0 || p.mask.Lq == 0) return cudaSuccess;
  auto enc = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(encode_fn);
  const bool bf16 = p.dtype == LLK_DTYPE_BF16;
  if (p.D <= 64)
    return bf16 ? launch_tc<64, true>(enc, p, status, sm_count, stream)
                : launch_tc<64, false>(enc, p, status, sm_count, stream);
  return bf16 ? launch_tc<128, true>(enc, p, status, sm_count, stream)
              : launch_tc<128, false>(enc, p, status, sm_count, stream);
}

}  // namespace llk_b200
