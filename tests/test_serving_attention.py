"""Refusals of the serving attention entry points that need no GPU, and the
plain forms the GPU tests measure against."""
import ctypes
import math

import pytest

torch = pytest.importorskip("torch")

import dslcompiler_b200 as llk  # noqa: E402
from dslcompiler_b200 import capi  # noqa: E402
from tests import serving_ref as ref  # noqa: E402


def t4(shape, stride=None, data=64):
    if stride is None:
        stride, n = [], 1
        for d in reversed(shape):
            stride.insert(0, n)
            n *= d
    return capi.Tensor4D(data, tuple(shape), tuple(stride))


def window(q, k, v, o, dtype=capi.LLK_DTYPE_BF16, win=0, sinks=0):
    return capi.lib().llk_window_attention(q, k, v, o, dtype, None, None, win, sinks, 1.0, None, None)


def test_window_attention_refuses_before_any_device_use():
    q, k, o = t4((2, 8, 4, 64)), t4((2, 2, 9, 64), data=1 << 20), t4((2, 8, 4, 64), data=1 << 21)
    L = capi.lib()
    assert L.llk_window_attention(None, k, k, o, 0, None, None, 0, 0, 1.0, None, None) == capi.LLK_ERR_ARG
    assert window(q, t4((2, 3, 9, 64)), t4((2, 3, 9, 64)), o) == capi.LLK_ERR_SHAPE
    assert window(q, t4((1, 2, 9, 64)), t4((1, 2, 9, 64)), o) == capi.LLK_ERR_SHAPE
    assert window(q, k, t4((2, 2, 8, 64)), o) == capi.LLK_ERR_SHAPE
    assert window(q, k, k, t4((2, 8, 5, 64))) == capi.LLK_ERR_SHAPE
    assert window(q, t4((2, 0, 9, 64)), t4((2, 0, 9, 64)), o) == capi.LLK_ERR_SHAPE
    assert window(t4((2, 8, 4, -1)), k, k, o) == capi.LLK_ERR_SHAPE
    assert window(q, k, k, o, dtype=7) == capi.LLK_ERR_ARG
    assert window(q, k, k, o, win=-1) == capi.LLK_ERR_ARG
    assert window(q, k, k, o, sinks=-1) == capi.LLK_ERR_ARG
    assert window(q, t4((2, 2, 9, 64), (1152, 576, 64, 2)), k, o) == capi.LLK_ERR_ALIGN
    assert window(q, t4((2, 2, 9, 64), (1152, -576, 64, 1)), k, o) == capi.LLK_ERR_ALIGN
    assert window(q, k, k, t4((2, 8, 4, 64), (0, 256, 64, 1))) == capi.LLK_ERR_ALIGN
    assert window(q, t4((2, 2, 9, 64), data=65), k, o) == capi.LLK_ERR_ALIGN
    assert window(q, k, k, t4((2, 8, 4, 64))) == capi.LLK_ERR_ARG  # o is q
    assert window(t4((1, 1, 1, 300)), t4((1, 1, 1, 300)), t4((1, 1, 1, 300)), t4((1, 1, 1, 300), data=4096)) == \
        capi.LLK_ERR_UNSUPPORTED
    assert window(q, t4((2, 2, 2**30 + 1, 64)), t4((2, 2, 2**30 + 1, 64)), o) == capi.LLK_ERR_UNSUPPORTED
    # nothing to do
    assert window(t4((0, 8, 4, 64)), t4((0, 2, 9, 64)), t4((0, 2, 9, 64)), t4((0, 8, 4, 64))) == capi.LLK_OK


def cache(**kw):
    f = dict(k_codes=1 << 12, k_params=1 << 13, v_codes=1 << 14, v_params=1 << 15, num_pages=4, page_size=16,
             kv_heads=2, head_dim=64, bits=4, group_size=32)
    f.update(kw)
    return capi.KvCache(**f)


def move(c, k=None, v=None, dtype=capi.LLK_DTYPE_BF16, slots=8, write=True):
    k = k or t4((2, 2, 3, 64), data=1 << 20)
    v = v or t4((2, 2, 3, 64), data=1 << 21)
    f = capi.lib().llk_kv_cache_write if write else capi.lib().llk_kv_cache_read
    return f(c, k, v, dtype, slots, None)


def test_cache_moves_refuse_before_any_device_use():
    assert move(None) == capi.LLK_ERR_ARG
    assert move(cache(head_dim=96)) == capi.LLK_ERR_UNSUPPORTED
    assert move(cache(bits=2)) == capi.LLK_ERR_UNSUPPORTED
    assert move(cache(group_size=16)) == capi.LLK_ERR_UNSUPPORTED
    assert move(cache(group_size=128)) == capi.LLK_ERR_SHAPE
    assert move(cache(group_size=0)) == capi.LLK_ERR_SHAPE
    assert move(cache(page_size=24)) == capi.LLK_ERR_UNSUPPORTED
    assert move(cache(num_pages=-1)) == capi.LLK_ERR_SHAPE
    assert move(cache(k_codes=None)) == capi.LLK_ERR_ARG
    assert move(cache(v_params=(1 << 15) + 8)) == capi.LLK_ERR_ALIGN
    bad = cache()
    bad.reserved[1] = 1
    assert move(bad) == capi.LLK_ERR_ARG
    assert move(cache(), k=t4((2, 3, 3, 64)), v=t4((2, 3, 3, 64))) == capi.LLK_ERR_SHAPE
    assert move(cache(), v=t4((2, 2, 4, 64))) == capi.LLK_ERR_SHAPE
    assert move(cache(), slots=None) == capi.LLK_ERR_ARG
    assert move(cache(), slots=4) == capi.LLK_ERR_ALIGN
    assert move(cache(), dtype=9) == capi.LLK_ERR_ARG
    assert move(cache(), k=t4((2, 2, 3, 64), (0, 192, 64, 1)), write=False) == capi.LLK_ERR_ALIGN
    same = t4((2, 2, 3, 64))
    assert move(cache(), k=same, v=same, write=False) == capi.LLK_ERR_ARG
    assert move(cache(), k=t4((2**30, 2, 1, 64)), v=t4((2**30, 2, 1, 64))) == capi.LLK_ERR_UNSUPPORTED
    assert move(cache(), k=t4((2, 2, 0, 64)), v=t4((2, 2, 0, 64)), slots=None) == capi.LLK_OK


def attend(c, q=None, o=None, table=16, width=3, stride=3, q_lens=None, kv_lens=16, dtype=capi.LLK_DTYPE_BF16, win=0,
           sinks=0):
    q = q or t4((2, 4, 1, 64), data=1 << 20)
    o = o or t4((2, 4, 1, 64), data=1 << 21)
    return capi.lib().llk_kv_cache_attention(q, c, table, width, stride, q_lens, kv_lens, o, dtype, win, sinks, 1.0,
                                             None, None)


def test_cache_attention_refuses_before_any_device_use():
    assert attend(None) == capi.LLK_ERR_ARG
    assert attend(cache(), q=t4((2, 3, 1, 64)), o=t4((2, 3, 1, 64))) == capi.LLK_ERR_SHAPE
    assert attend(cache(), q=t4((2, 4, 1, 128)), o=t4((2, 4, 1, 128))) == capi.LLK_ERR_SHAPE
    assert attend(cache(), o=t4((2, 4, 2, 64))) == capi.LLK_ERR_SHAPE
    assert attend(cache(), stride=2) == capi.LLK_ERR_SHAPE
    assert attend(cache(), width=-1) == capi.LLK_ERR_SHAPE
    assert attend(cache(), width=2**30) == capi.LLK_ERR_UNSUPPORTED
    assert attend(cache(), dtype=capi.LLK_DTYPE_FP32) == capi.LLK_ERR_UNSUPPORTED
    assert attend(cache(), kv_lens=None) == capi.LLK_ERR_ARG
    assert attend(cache(), table=None) == capi.LLK_ERR_ARG
    assert attend(cache(), table=18) == capi.LLK_ERR_ALIGN
    assert attend(cache(), win=-2) == capi.LLK_ERR_ARG
    assert attend(cache(), o=t4((2, 4, 1, 64), data=1 << 20)) == capi.LLK_ERR_ARG
    assert attend(cache(), o=t4((2, 4, 1, 64), (256, 0, 64, 1), data=1 << 21)) == capi.LLK_ERR_ALIGN


def test_python_face_refuses_host_tensors():
    q = torch.zeros((1, 1, 1, 64), dtype=torch.bfloat16)
    with pytest.raises(TypeError):
        llk.window_attention(q, q, q)
    z = torch.zeros((1, 1, 16, 32), dtype=torch.uint8)
    with pytest.raises(TypeError):
        llk.QuantizedKVCache(z, z, z, z, bits=4)
    with pytest.raises(ValueError):
        llk.QuantizedKVCache.empty(1, 16, 1, 64, bits=3, device="cpu")


def test_struct_layouts():
    assert ctypes.sizeof(capi.Tensor4D) == 72
    assert ctypes.sizeof(capi.KvCache) == 72


def test_plain_forms_agree_with_themselves():
    """The 64-bit form the GPU tests use: a window over everything is none, sinks over everything neither; rows that
    see nothing are zero; quantising what a cache holds changes nothing."""
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn((1, 2, 9, 8), generator=g) for _ in range(3))
    a = ref.attention(q, k, v)[0]
    assert torch.allclose(a, ref.attention(q, k, v, window=9)[0])
    assert torch.allclose(a, ref.attention(q, k, v, window=1, sinks=9)[0])
    want = torch.softmax((q @ k.transpose(-1, -2) / math.sqrt(8)).masked_fill(
        ~torch.ones(9, 9, dtype=torch.bool).tril(), -math.inf), -1) @ v
    assert torch.allclose(a.float(), want, atol=1e-5)
    b = ref.attention(q, k[:, :, :4], v[:, :, :4])[0]
    assert (b[:, :, :5] == 0).all()
    x = torch.randn((1, 1, 5, 64), generator=g)
    c, s, m = ref.quantise(x, 4, 32)
    assert (x.double() - ref.values(c, s, m)).abs().max() <= 0.51 * s.max()
