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


@pytest.mark.parametrize("n,D,dtype", [(32768, 64, BF16), (32769, 64, F32), (100_003, 64, BF16), (70_001, 128, F16)])
def test_last_of_a_slot_stands_in_long_calls(n, D, dtype):
    """Slots named again far behind their first token, and right behind it; padding; the slots from an odd place."""
    page, slots_n = 64, -(-n // 64) * 64
    cache = llk.QuantizedKVCache.empty(slots_n // page, page, 1, D, group_size=D)
    g = torch.Generator().manual_seed(n)
    slots = torch.randperm(slots_n, generator=g)[:n]
    slots[n // 3 : n // 3 + 500] = slots[:500]
    slots[n - 700 : n] = slots[n // 2 : n // 2 + 700]
    slots[n - 100 : n] = slots[0]
    slots[7::1000], slots[11::1000] = -1, slots_n
    held = torch.empty(n + 1, dtype=torch.int64, device="cuda")[1:].copy_(slots).reshape(1, n)
    x = torch.randn((1, 1, n, D), generator=g).to(dtype)
    cache.write(x.cuda(), -x.cuda(), held)
    last = torch.full((slots_n,), -1, dtype=torch.int64)
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < slots_n:
            last[s] = t
    there = last >= 0
    for t, codes, params in ((x, cache.k_codes, cache.k_params), (-x, cache.v_codes, cache.v_params)):
        c, s, m = ref.quantise(t[0, 0], 4, D)
        got = ref.unpack(codes, 4).reshape(slots_n, D)
        par = params.cpu().double().reshape(slots_n, 2)
        assert torch.equal(got[there], c.long()[last[there]])
        assert torch.equal(par[there], torch.cat([s, m], -1)[last[there]])
        assert (got[~there] == 0).all() and (par[~there] == 0).all()


def test_a_long_write_takes_time_in_proportion():
    """16 times the tokens take about 16 times as long, and not 16 times that."""
    D, page, top = 64, 64, 1 << 19
    cache = llk.QuantizedKVCache.empty(top // page, page, 1, D, group_size=D)
    x = torch.randn((1, 1, top, D), device="cuda").to(BF16)
    slots = torch.randperm(top, device="cuda")[None]

    def ms(n):
        k, s = x[:, :, :n], slots[:, :n].contiguous()
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        best = math.inf
        for _ in range(4):
            a.record()
            for _ in range(4):
                cache.write(k, k, s)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b) / 4)
        return best

    ms(1 << 15)
    short, long = ms(1 << 15), ms(top)
    print(f"{1 << 15} tokens {short * 1e3:.1f} us, {top} tokens {long * 1e3:.1f} us")
    assert long < 2.5 * 16 * short + 0.1
