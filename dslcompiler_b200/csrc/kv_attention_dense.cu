// kv_attention_dense.cu -- the split kernels over dense bf16 / f16 keys and
// values (kv_attention.cuh).
#include <type_traits>

#include "kv_attention.cuh"

namespace llk_b200 {
namespace split_attn {

namespace {

template <bool kBf16, int D>
cudaError_t launch_nt(const Params &a, cudaStream_t stream) {
  if constexpr (row_tiles(16, D) == 2)
    if (row_tiles(a.p.H / a.p.Hkv * a.p.mask.Lq, D) == 2) return launch_split<16, D, 1, kBf16, kBf16, 2>(a, stream);
  return launch_split<16, D, 1, kBf16, kBf16, 1>(a, stream);
}

template <bool kBf16>
cudaError_t launch_d(const Params &a, cudaStream_t stream) {
  switch (a.p.D) {
    case 64: return launch_nt<kBf16, 64>(a, stream);
    case 80: return launch_nt<kBf16, 80>(a, stream);
    case 96: return launch_nt<kBf16, 96>(a, stream);
    case 128: return launch_nt<kBf16, 128>(a, stream);
    default: return launch_nt<kBf16, 256>(a, stream);
  }
}

}  // namespace

cudaError_t launch_dense(const Params &a, cudaStream_t stream) {
  return a.p.dtype == LLK_DTYPE_FP16 ? launch_d<false>(a, stream) : launch_d<true>(a, stream);
}

}  // namespace split_attn
}  // namespace llk_b200
