"""Attention for serving on the B200: windowed attention with sinks over dense
keys and values (``llk_window_attention``), and the quantised paged KV cache
with its writer, reader and attention (``llk_kv_cache_*``).

Tensors are torch CUDA tensors, [B, H, L, D] in any order of strides (unit
stride along D); calls run asynchronously on the current torch stream of
their device, or on ``stream``: the caller orders that stream behind what made
the inputs, and its own use of the result behind that stream.  There is no CPU
path and no host staging.
"""
from __future__ import annotations

import ctypes
import functools
import math
import threading

from . import capi
from .capi import KernelContext, KvCache, Tensor4D, check, lib
from .swiglu import _is_torch, _made_on, _out_on, _stream_of, gpu_context

try:
    import torch

    _DTYPES = {torch.bfloat16: capi.LLK_DTYPE_BF16, torch.float16: capi.LLK_DTYPE_FP16,
               torch.float32: capi.LLK_DTYPE_FP32}
except Exception:  # pragma: no cover
    torch = None
    _DTYPES = {}


class _Views(threading.local):
    """This thread's descriptors by argument, sizes and strides (building one costs more than a launch)."""

    def __init__(self):
        self.known = {}


_views = _Views()


def _tensor4d(t, arg=0) -> Tensor4D:
    """t's descriptor for the next call of this thread; `arg` tells a call's tensors apart."""
    key = (arg, t.shape, t.stride())
    d = _views.known.get(key)
    if d is None:
        if len(_views.known) >= 1024:
            _views.known.clear()
        d = _views.known[key] = Tensor4D(0, tuple(t.shape), t.stride())
    d.data = t.data_ptr()
    return d


def _check_data(what, t, dtypes=None, dtype=None):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{what} must be a torch CUDA tensor")
    if t.dim() != 4:
        raise ValueError(f"{what} must be [B, H, L, D]")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{what} must be {dtype}")
    if t.dtype not in (dtypes or _DTYPES):
        raise TypeError(f"{what} must be one of {', '.join(str(d) for d in (dtypes or _DTYPES))}")


def _check_ints(what, t, dtype, shape):
    if not _is_torch(t) or not t.is_cuda or t.dtype != dtype:
        raise TypeError(f"{what} must be a {dtype} CUDA tensor")
    if tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous {list(shape)}")
    return t.data_ptr()


def _ranges(window, sinks):
    w, s = int(window or 0), int(sinks)
    if w != (window or 0) or s != sinks:  # (a fraction would be cut to another window)
        raise ValueError("window and sinks must be whole numbers")
    if w < 0 or s < 0:
        raise ValueError("window and sinks must not be negative")
    return min(w, 2**62), min(s, 2**62)


def _out_like(q, q_lens, stream):
    # rows behind a sequence's queries are not written: they read as zeros
    return _out_on(stream, q.device, lambda: torch.empty_like(q) if q_lens is None else torch.zeros_like(q))


def _scratch(nbytes, like, stream):
    """Device memory of the caller's allocator for one call: calls on different streams or in different graphs do not
    share it."""
    if not nbytes:
        return None, None
    buf = _made_on(stream, like.device, lambda: like.new_empty((nbytes + 1) // 2))
    return buf, KernelContext(buf.data_ptr(), nbytes)


# How much scratch a call needs follows from its sizes.
@functools.lru_cache(maxsize=4096)
def _window_scratch(q_shape, k_shape, k_stride, k_on16, dtype, window, sinks, device):
    out = ctypes.c_int64()
    tq = Tensor4D(0, q_shape, (0, 0, 0, 1))
    tk = Tensor4D(0 if k_on16 else 8, k_shape, k_stride)
    g = gpu_context(device)
    check(lib().llk_window_attention_scratch(tq, tk, dtype, window, sinks, g, ctypes.byref(out)),
          "llk_window_attention_scratch")
    return out.value


def window_attention(q, k, v, *, window=0, sinks: int = 0, scale: float | None = None, q_lens=None, kv_lens=None,
                     out=None, stream=None):
    """Causal attention under a sliding window with sinks, for prompts and for single tokens.

    q [B, H, Lq, D]; k, v [B, Hkv, Lk, D] with Hkv dividing H; bf16, f16 or
    f32, all of one type; D <= 256.  Sequence b has ``kv_lens[b]`` keys
    (default Lk) and ``q_lens[b]`` queries (default Lq; int32 [B] CUDA
    tensors); its query i is the token at position p = kv_lens[b] - q_lens[b]
    + i, and sees the keys j <= p with ``window`` == 0 (or None) or
    j > p - window or j < ``sinks``.  A query that sees no key gives zeros;
    rows behind q_lens[b] are left as they were in ``out`` (zeros without
    one).  scale defaults to 1/sqrt(D).  Returns O [B, H, Lq, D]."""
    _check_data("q", q)
    _check_data("k", k, dtype=q.dtype)
    _check_data("v", v, dtype=q.dtype)
    window, sinks = _ranges(window, sinks)
    B, D = q.shape[0], q.shape[3]
    pq = None if q_lens is None else _check_ints("q_lens", q_lens, torch.int32, (B,))
    pk = None if kv_lens is None else _check_ints("kv_lens", kv_lens, torch.int32, (B,))
    if out is None:
        out = _out_like(q, q_lens, stream)
    else:
        _check_data("out", out, dtype=q.dtype)
    dtype = _DTYPES[q.dtype]
    need = _window_scratch(tuple(q.shape), tuple(k.shape), k.stride(), k.data_ptr() % 16 == 0, dtype, window, sinks,
                           q.device.index)
    buf, ctx = _scratch(need, q, stream)
    g = gpu_context(q.device.index, _stream_of(q, stream))
    rc = lib().llk_window_attention(_tensor4d(q), _tensor4d(k, 1), _tensor4d(v, 2), _tensor4d(out, 3), dtype, pq, pk,
                                    window, sinks, 1.0 / math.sqrt(max(D, 1)) if scale is None else float(scale), ctx, g)
    if rc:
        check(rc, "llk_window_attention")
    return out


class QuantizedKVCache:
    """A paged KV cache held in 4 or 8 bits: the handle on its four tensors

    * k_codes, v_codes uint8 [num_pages, kv_heads, page_size, head_dim * bits / 8]
      (4 bits: element 2j in the low nibble of byte j),
    * k_params, v_params bf16 [num_pages, kv_heads, page_size, head_dim / group_size, 2]: (scale, min),

    an element standing for scale * code + min (a zero-filled slot for zeros).  head_dim 64, 128 or 256;
    group_size 32, 64 or 128; page_size a multiple of 16.  Slot number =
    page * page_size + offset; token t of a sequence lies in page
    block_table[b, t // page_size] at offset t % page_size."""

    def __init__(self, k_codes, k_params, v_codes, v_params, *, bits: int):
        for name, t, dt, nd in (("k_codes", k_codes, torch.uint8, 4), ("k_params", k_params, torch.bfloat16, 5),
                                ("v_codes", v_codes, torch.uint8, 4), ("v_params", v_params, torch.bfloat16, 5)):
            if not _is_torch(t) or not t.is_cuda or t.dtype != dt:
                raise TypeError(f"{name} must be a {dt} CUDA tensor")
            if t.dim() != nd or not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous with {nd} dimensions")
            if t.device != k_codes.device:
                raise ValueError("the cache's tensors must be on one device")
        if bits not in (4, 8):
            raise ValueError("bits must be 4 or 8")
        pages, heads, page, row_bytes = k_codes.shape
        groups = k_params.shape[3]
        dim = row_bytes * 8 // bits
        if (v_codes.shape != k_codes.shape or v_params.shape != k_params.shape or groups < 1 or dim % groups
                or tuple(k_params.shape) != (pages, heads, page, groups, 2)):
            raise ValueError("codes must be [pages, heads, page, head_dim * bits / 8] and params "
                             "[pages, heads, page, head_dim / group_size, 2]")
        group = dim // groups
        if dim not in (64, 128, 256) or group not in (32, 64, 128) or page < 16 or page % 16:
            raise ValueError("head_dim must be 64, 128 or 256, group_size 32, 64 or 128, page_size a multiple of 16: got "
                             f"{dim}, {group}, {page}")
        self.k_codes, self.k_params, self.v_codes, self.v_params = k_codes, k_params, v_codes, v_params
        self.num_pages, self.kv_heads, self.page_size, self.head_dim = pages, heads, page, dim
        self.bits, self.group_size, self.device = bits, group, k_codes.device
        self._c = KvCache(k_codes.data_ptr(), k_params.data_ptr(), v_codes.data_ptr(), v_params.data_ptr(), pages, page,
                          heads, dim, bits, group)

    @classmethod
    def empty(cls, num_pages: int, page_size: int, kv_heads: int, head_dim: int, *, bits: int = 4,
              group_size: int = 64, device="cuda") -> "QuantizedKVCache":
        """A new cache of num_pages pages, zero-filled."""
        if bits not in (4, 8) or group_size < 1 or head_dim % group_size:
            raise ValueError("bits must be 4 or 8 and group_size must divide head_dim")
        shape = (num_pages, kv_heads, page_size)

        def pair():
            return (torch.zeros(shape + (head_dim * bits // 8,), dtype=torch.uint8, device=device),
                    torch.zeros(shape + (head_dim // group_size, 2), dtype=torch.bfloat16, device=device))

        return cls(*pair(), *pair(), bits=bits)

    def write(self, k, v, slots, *, stream=None) -> None:
        """Quantises k, v [B, kv_heads, L, head_dim] (bf16, f16 or f32) into the slots [B, L] (int64).  Values are
        saturated to +-65504 and NaN counts as 0.  A slot outside the cache (such as -1, padding) is not written;
        where a slot is named more than once, its last token in [B, L] order stands."""
        _check_data("k", k)
        _check_data("v", v, dtype=k.dtype)
        ps = _check_ints("slots", slots, torch.int64, (k.shape[0], k.shape[2]))
        g = gpu_context(self.device.index, _stream_of(k, stream))
        rc = lib().llk_kv_cache_write(self._c, _tensor4d(k), _tensor4d(v, 1), _DTYPES[k.dtype], ps, g)
        if rc:
            check(rc, "llk_kv_cache_write")

    def read(self, slots, *, dtype=None, out=None, stream=None):
        """(k, v) [B, kv_heads, L, head_dim] of the slots [B, L] in ``dtype`` (default bf16), or into the pair
        ``out``.  A slot outside the cache reads as zeros.  What was written within 2^-8 of +-65504, or saturated to
        it, may stand for more than f16 holds (-65504 for -65536) and read as an infinity there; bf16 and f32 hold it."""
        if not _is_torch(slots) or slots.dim() != 2:
            raise TypeError("slots must be a torch.int64 CUDA tensor [B, L]")
        ps = _check_ints("slots", slots, torch.int64, tuple(slots.shape))
        if out is None:
            if dtype is not None and dtype not in _DTYPES:
                raise TypeError(f"dtype must be one of {', '.join(str(d) for d in _DTYPES)}")
            # (on the cache's device, where the slots have to be too)
            shape = (2, slots.shape[0], self.kv_heads, slots.shape[1], self.head_dim)
            k, v = _out_on(stream, self.device, lambda: self.k_params.new_empty(shape, dtype=dtype)).unbind(0)
        else:
            k, v = out
            if dtype is not None and k.dtype != dtype:
                raise TypeError(f"out must be {dtype}")
            _check_data("k", k)
            _check_data("v", v, dtype=k.dtype)
            if (k.shape[0], k.shape[2]) != tuple(slots.shape):
                raise ValueError("out must be [B, kv_heads, L, head_dim] with the slots' B and L")
        g = gpu_context(self.device.index, _stream_of(slots, stream))
        rc = lib().llk_kv_cache_read(self._c, _tensor4d(k), _tensor4d(v, 1), _DTYPES[k.dtype], ps, g)
        if rc:
            check(rc, "llk_kv_cache_read")
        return k, v

    def attention(self, q, block_table, kv_lens, *, window=0, sinks: int = 0, scale: float | None = None, q_lens=None,
                  out=None, stream=None):
        """Attention of q [B, H, Lq, head_dim] (bf16 or f16) over the cache, causal under a sliding window with sinks
        (the ranges of :func:`window_attention`).  Sequence b's keys are the first ``kv_lens[b]`` tokens of the pages
        ``block_table[b]`` (int32 [B, W], rows may be a slice of a wider table); its own new tokens are written
        first, so kv_lens counts them.  An entry of the table outside the cache holds tokens that no query sees."""
        _check_data("q", q, dtypes=(torch.bfloat16, torch.float16))
        window, sinks = _ranges(window, sinks)
        B, D = q.shape[0], q.shape[3]
        if not _is_torch(block_table) or not block_table.is_cuda or block_table.dtype != torch.int32:
            raise TypeError("block_table must be a torch.int32 CUDA tensor")
        if block_table.dim() != 2 or block_table.shape[0] != B or (block_table.shape[1] > 1 and block_table.stride(1) != 1):
            raise ValueError("block_table must be [B, pages a sequence] with unit stride along its rows")
        pk = _check_ints("kv_lens", kv_lens, torch.int32, (B,))
        pq = None if q_lens is None else _check_ints("q_lens", q_lens, torch.int32, (B,))
        if out is None:
            out = _out_like(q, q_lens, stream)
        else:
            _check_data("out", out, dtype=q.dtype)
        W = block_table.shape[1]
        buf, ctx = _scratch(_cache_scratch(tuple(q.shape), self.page_size, self.kv_heads, self.head_dim, self.bits,
                                           self.group_size, W, window, sinks, q.device.index), q, stream)
        g = gpu_context(self.device.index, _stream_of(q, stream))
        rc = lib().llk_kv_cache_attention(_tensor4d(q), self._c, block_table.data_ptr(), W,
                                          block_table.stride(0) if B > 1 else W, pq, pk, _tensor4d(out, 1),
                                          _DTYPES[q.dtype], window, sinks,
                                          1.0 / math.sqrt(max(D, 1)) if scale is None else float(scale), ctx, g)
        if rc:
            check(rc, "llk_kv_cache_attention")
        return out


@functools.lru_cache(maxsize=4096)
def _cache_scratch(q_shape, page, heads, dim, bits, group, width, window, sinks, device):
    out = ctypes.c_int64()
    c = KvCache(0, 0, 0, 0, 0, page, heads, dim, bits, group)
    check(lib().llk_kv_cache_attention_scratch(Tensor4D(0, q_shape, (0, 0, 0, 1)), c, width, window, sinks,
                                               gpu_context(device), ctypes.byref(out)),
          "llk_kv_cache_attention_scratch")
    return out.value


__all__ = ["window_attention", "QuantizedKVCache"]
