"""Refusals of layouts whose output rows lie on one another (no GPU needed:
they are found before any device is used)."""
import pytest

pytest.importorskip("torch")

from dslcompiler_b200 import capi  # noqa: E402


def t4(shape, stride, data):
    return capi.Tensor4D(data, tuple(shape), tuple(stride))


def dense(shape, data):
    n, stride = 1, []
    for d in reversed(shape):
        stride.insert(0, n)
        n *= d
    return t4(shape, stride, data)


@pytest.mark.parametrize("stride", [(64, 64, 64, 1),          # every dimension steps over one row
                                    (512, 256, 32, 1),        # rows half on the next
                                    (2048, 64, 256, 1),       # 8 heads of 64 reach over 512, tokens step 256
                                    (1024, 256, 64, 1),       # the next sequence begins inside this one
                                    (2**62, 2**62, 2**62, 1)])
def test_outputs_whose_rows_overlap_are_refused(stride):
    L = capi.lib()
    q, k = dense((2, 8, 4, 64), 1 << 20), dense((2, 2, 9, 64), 1 << 21)
    o = t4((2, 8, 4, 64), stride, 1 << 22)
    assert L.llk_window_attention(q, k, k, o, 0, None, None, 0, 0, 1.0, None, None) == capi.LLK_ERR_ALIGN
    c = capi.KvCache(1 << 12, 1 << 13, 1 << 14, 1 << 15, 4, 16, 8, 64, 4, 32)
    kv = dense((2, 8, 4, 64), 1 << 23)
    assert L.llk_kv_cache_read(c, kv, o, 0, 8, None) == capi.LLK_ERR_ALIGN
    assert L.llk_kv_cache_read(c, o, kv, 0, 8, None) == capi.LLK_ERR_ALIGN
    assert L.llk_kv_cache_attention(q, c, 4, 1, 1, None, 4, o, 0, 0, 0, 1.0, None, None) == capi.LLK_ERR_ALIGN
