// kv_kernels.h -- launch interface of the serving attention kernels: windowed
// attention over dense keys and values (window_attention.cu), the quantised
// paged KV cache's writer and reader (kv_cache.cu), and attention over few
// query rows split along the keys (kv_attention.cu).
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace llk_b200 {

// A [B, H, L, D] tensor: strides in elements, unit stride along D.
struct View4 {
  void *p;
  int64_t sb, sh, sl;
};

// Which keys a query sees.  Sequence b has n = kv_lens[b] keys and m =
// q_lens[b] queries (nullptr: Lk and Lq; both are clamped to [0, Lk] and
// [0, Lq]); query i < m is at position p = n - m + i and sees key j iff
// j <= p and (window == 0 or j > p - window or j < sinks).  Rows i >= m of O
// are not written; a row that sees no key is zero.
struct AttnMask {
  const int *q_lens;
  const int *kv_lens;
  int Lq, Lk;
  int window;  // 0: no window
  int sinks;
};

struct AttnProblem {
  View4 q, k, v, o;  // k, v: dense keys / values (unused over a cache)
  int B, H, Hkv, D;
  int dtype;  // enum llk_dtype of q, k, v, o
  float scale;
  AttnMask mask;
};

// The quantised pool: codes [num_pages, Hkv, page, D * bits / 8] bytes and
// params [num_pages, Hkv, page, D / group] (scale, min) bf16 pairs.
struct KvPool {
  void *k_codes, *k_params, *v_codes, *v_params;
  int64_t num_pages;
  int page, Hkv, D, bits, group;
};

// CUDA-core kernel: any type, strides and alignment, D <= 256.
bool window_simt_supported(const AttnProblem &p);
cudaError_t window_simt_launch(const AttnProblem &p, cudaStream_t stream);

// f32, few query rows over many keys, split along the keys: rows of K and V
// on 16 bytes, D a multiple of 4.
struct RowsPlan {
  int splits;       // shares of the keys
  int rows;         // query rows of a block, 4 or 8
  int row_blocks;   // blocks of query rows of one key head
  size_t ws_bytes;  // device workspace the launch needs
};
bool rows_supported(const AttnProblem &p);
RowsPlan rows_plan(const AttnProblem &p, int sm_count);
cudaError_t rows_launch(const AttnProblem &p, const RowsPlan &plan, void *workspace, cudaStream_t stream);

// Tensor-core kernel for prompts: bf16 / f16, D <= 128, rows on 16 bytes.
// encode_fn: cuTensorMapEncodeTiled; status: the device's error word (a
// bounded wait that gave up).
bool window_tc_supported(const AttnProblem &p);
cudaError_t window_tc_launch(void *encode_fn, const AttnProblem &p, int *status, int sm_count, cudaStream_t stream);

bool kv_pool_supported(const KvPool &p);
// k, v: [B, Hkv, L, D] views of type dtype; slots [B, L].
cudaError_t kv_write_launch(const KvPool &p, const View4 &k, const View4 &v, int dtype, int64_t B, int64_t L,
                            const int64_t *slots, int sm_count, cudaStream_t stream);
cudaError_t kv_read_launch(const KvPool &p, const View4 &k, const View4 &v, int dtype, int64_t B, int64_t L,
                           const int64_t *slots, int sm_count, cudaStream_t stream);

// Few query rows over many keys, split along the keys.  Over a cache: pool
// and block_table [B, table_width]; dense: pool == nullptr.
struct SplitPlan {
  int workers;      // CTAs that share the work
  int row_blocks;   // blocks of query rows of one key head
  size_t ws_bytes;  // device workspace the launch needs (0: no work is cut)
};
bool split_supported(const AttnProblem &p, const KvPool *pool);
SplitPlan split_plan(const AttnProblem &p, const KvPool *pool, int sm_count);
cudaError_t split_launch(const AttnProblem &p, const KvPool *pool, const int *block_table, int64_t table_width,
                         const SplitPlan &plan, void *workspace, cudaStream_t stream);

}  // namespace llk_b200
