"""dslcompiler_b200 -- B200 (sm_100a) backend for DSLCompiler's fused SwiGLU
and micro.mma matmul path.

    import dslcompiler_b200 as llk
    y = llk.fused_swiglu(x, wg, wu)          # bf16 torch tensors on cuda
    c = llk.matmul(a, b)                      # f32 C = A B
    pw = llk.PackedWeights(wg, wu); y = pw(x)
    y = llk.rope(x, pos); o = llk.attention(q, k, v, causal=True)   # f32 ops
    o = llk.window_attention(q, k, v, window=1024, sinks=4)         # bf16 / f16 / f32, grouped heads
    cache = llk.QuantizedKVCache.empty(pages, 64, kv_heads, 128)    # 4-bit paged KV cache
    cache.write(k, v, slots); o = cache.attention(q, block_table, kv_lens)

All compute runs in the hand-written CUDA kernels of ``lib/libllk_b200.so``
(built by ``python -m dslcompiler_b200.build``); there is no CPU fallback.
"""
from .attention import attention, rope  # noqa: F401
from .capi import LLKError, lib  # noqa: F401
from .serving import QuantizedKVCache, window_attention  # noqa: F401
from .swiglu import (  # noqa: F401
    KernelKey,
    PackedWeights,
    cache_clear,
    cache_level_clear,
    cache_level_set_max_entries,
    cache_level_stats,
    cache_set_max_entries,
    cache_stats,
    classify_m,
    fused_swiglu,
    matmul,
    probe,
    shard_columns,
    swiglu_c_abi,
    synchronize,
    tensor2d,
    weight_key,
)

__version__ = "0.1.0"
