"""The cache's writer where a whole group saturates, and where a call has many
tokens.  Codes, scales and minima are serving_ref.quantise's bit for bit."""
import math

import pytest

torch = pytest.importorskip("torch")

import dslcompiler_b200 as llk  # noqa: E402
from tests import serving_ref as ref  # noqa: E402

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("bits,D,group", [(4, 64, 32), (4, 128, 128), (8, 64, 64), (8, 256, 32)])
def test_groups_that_saturate_whole(bits, D, group, dtype):
    """All elements of a group at or beyond the largest held magnitude: the minimum rounds to above them, and the
    codes stay within their range."""
    rows = [[math.inf] * 4, [65536.0, 65504.0, 65280.0, 1e9], [-math.inf] * 4, [-65536.0, -1e9, -65504.0, -math.inf],
            [65504.0] * 4, [-65504.0] * 4, [math.inf, 65504.0, math.inf, 7e4], [math.nan, math.inf, math.inf, math.inf],
            [math.nan] * 4, [math.inf, 1.0, -1.0, 0.0], [-math.inf, 65504.0, 0.5, math.nan], [0.0] * 4]
    L = len(rows)
    x = torch.tensor(rows, dtype=torch.float64).repeat_interleave(D // 4, 1).reshape(1, 1, L, D)
    x[..., 1::2] = x[..., 1::2].flip(-1)
    x = torch.cat([x, x.roll(1, 2)], 1).to(dtype)
    cache = llk.QuantizedKVCache.empty(1, 16, 2, D, bits=bits, group_size=group)
    cache.write(x.cuda(), x.cuda(), torch.arange(L)[None].cuda())
    c, s, m = ref.quantise(x, bits, group)
    for codes, params in ((cache.k_codes, cache.k_params), (cache.v_codes, cache.v_params)):
        par = params.cpu().double()[0, :, :L]
        assert torch.equal(par[..., 0], s[0]) and torch.equal(par[..., 1], m[0])
        assert torch.equal(ref.unpack(codes, bits)[0, :, :L], c.long()[0])
