// kv_attention.cu -- attention over the quantised paged cache in bf16, and the
// plan of the split kernels (kv_attention.cuh).
#include <type_traits>

#include "kv_attention.cuh"

namespace llk_b200 {

using namespace split_attn;

bool split_supported(const AttnProblem &p, const KvPool *pool) {
  const int64_t g = p.Hkv > 0 ? p.H / p.Hkv : 0, rows = g * p.mask.Lq;
  if (p.dtype != LLK_DTYPE_BF16 && p.dtype != LLK_DTYPE_FP16) return false;
  if (rows * p.Hkv > (int64_t(1) << 30) / (p.B > 0 ? p.B : 1)) return false;  // rows are counted in 32 bits
  // so are the units of work (and a sum of two of them), and the rows of a pool
  const int64_t units = (static_cast<int64_t>(p.mask.Lk) / kSpan + 2 + kStart) * p.B;  // kMaxLen's bounds: below 2^53
  if (units >= (int64_t(1) << 30) || units * p.Hkv >= (int64_t(1) << 30) ||
      units * p.Hkv * ((rows + 7) / 8) >= (int64_t(1) << 30))
    return false;
  if (pool) return kv_pool_supported(*pool) && pool->num_pages <= 0xffffffffll / pool->Hkv / pool->page;
  const auto on16 = [](const View4 &v) {
    return (reinterpret_cast<uintptr_t>(v.p) & 15) == 0 && v.sb % 8 == 0 && v.sh % 8 == 0 && v.sl % 8 == 0;
  };
  return (p.D == 64 || p.D == 80 || p.D == 96 || p.D == 128 || p.D == 256) && on16(p.k) && on16(p.v);
}

// As many workers as the GPU holds at once, or as there can be units of work
// when those are fewer (the lengths are on the device, so this goes by the
// most keys a sequence can have).
SplitPlan split_plan(const AttnProblem &p, const KvPool *pool, int sm_count) {
  SplitPlan s;
  const int rows = p.H / p.Hkv * p.mask.Lq, nt = row_tiles(rows, p.D);
  s.row_blocks = (rows + 8 * nt - 1) / (8 * nt);
  int64_t keys = p.mask.Lk;
  if (p.mask.window > 0) {
    // the window and the sinks, each with a block begun at either end
    const int64_t seen = static_cast<int64_t>(p.mask.window) + p.mask.Lq + p.mask.sinks + 4 * kTok;
    if (seen < keys) keys = seen;
  }
  const int64_t segments = static_cast<int64_t>(p.B) * p.Hkv * s.row_blocks;
  const int64_t units = segments * (keys > kSpan ? (keys + kSpan - 1) / kSpan : 1), cost = units + segments * kStart;
  const bool two = pool && p.dtype == LLK_DTYPE_FP16;
  const int64_t room = static_cast<int64_t>(sm_count) *
                       ctas_per_sm(pool ? pool->bits : 16, p.D, pool ? p.D / pool->group : 1, nt, two);
  s.workers = static_cast<int>(cost < room ? cost : room);
  s.ws_bytes = 0;
  if (units > segments)  // else no segment has more than one unit: none is cut
    s.ws_bytes = 2 * static_cast<size_t>(s.workers) * 8 * nt * (static_cast<size_t>(p.D) * 4 + sizeof(float2));
  return s;
}

cudaError_t split_launch(const AttnProblem &p, const KvPool *pool, const int *block_table, int64_t table_width,
                         const SplitPlan &plan, void *workspace, cudaStream_t stream) {
  if (p.B == 0 || p.H == 0 || p.mask.Lq == 0) return cudaSuccess;
  Params a = {};
  a.p = p;
  if (pool) a.pool = *pool;
  a.table = block_table;
  a.table_width = table_width;
  a.workers = plan.workers;
  a.row_blocks = plan.row_blocks;
  a.page_shift = -1;
  for (int i = 4; pool && i < 17; ++i)
    if (pool->page == 1 << i) a.page_shift = i;
  a.q_vec = (reinterpret_cast<uintptr_t>(p.q.p) & 3) == 0 && p.q.sb % 2 == 0 && p.q.sh % 2 == 0 && p.q.sl % 2 == 0;
  if (plan.ws_bytes) {
    const int nt = row_tiles(p.H / p.Hkv * p.mask.Lq, p.D);
    a.part_ml = static_cast<float2 *>(workspace);
    a.part_o = reinterpret_cast<float *>(a.part_ml + 2 * static_cast<size_t>(plan.workers) * 8 * nt);
  }
  if (!pool) return launch_dense(a, stream);
  if (p.dtype == LLK_DTYPE_FP16) return launch_cache_f16(a, stream);
  return pool->bits == 4 ? launch_bits<4, false>(a, stream) : launch_bits<8, false>(a, stream);
}

}  // namespace llk_b200
