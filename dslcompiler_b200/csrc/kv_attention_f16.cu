// kv_attention_f16.cu -- the split kernels over the quantised paged cache in
// f16 (kv_attention.cuh).
#include <type_traits>

#include "kv_attention.cuh"

namespace llk_b200 {
namespace split_attn {

cudaError_t launch_cache_f16(const Params &a, cudaStream_t stream) {
  return a.pool.bits == 4 ? launch_bits<4, true>(a, stream) : launch_bits<8, true>(a, stream);
}

}  // namespace split_attn
}  // namespace llk_b200
