"""Attention over caches whose scales the cache's own writer does not make:
zero (slots never written, constant rows of another writer), negative,
subnormal.  An element stands for scale * code + min whatever the scale is."""
import pytest

torch = pytest.importorskip("torch")

import dslcompiler_b200 as llk  # noqa: E402
from tests import serving_ref as ref  # noqa: E402

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32

FORMATS = [(4, 64, 32, 16), (4, 64, 64, 32), (4, 128, 32, 16), (4, 128, 64, 48), (4, 128, 128, 64), (4, 256, 32, 16),
           (4, 256, 64, 16), (4, 256, 128, 32), (8, 64, 32, 16), (8, 64, 64, 32), (8, 128, 32, 16), (8, 128, 64, 16),
           (8, 128, 128, 64), (8, 256, 32, 16), (8, 256, 64, 16), (8, 256, 128, 32)]


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def pool(B, Hkv, L, D, bits, group, page, seed):
    """(cache, table, generator): random codes, scales in (0, 0.2), minima in (-1, 1)."""
    W = -(-L // page)
    cache = llk.QuantizedKVCache.empty(B * W, page, Hkv, D, bits=bits, group_size=group)
    g = torch.Generator().manual_seed(seed)
    for codes, params in ((cache.k_codes, cache.k_params), (cache.v_codes, cache.v_params)):
        codes.copy_(torch.randint(0, 256, codes.shape, generator=g, dtype=torch.uint8))
        shape = params.shape[:-1]
        params.copy_(torch.stack([torch.rand(shape, generator=g) * 0.2, 2 * torch.rand(shape, generator=g) - 1], -1))
    return cache, torch.randperm(B * W, generator=g).reshape(B, W).to(torch.int32).cuda(), g


def held(cache, table, L):
    """k, v, and |scale| code + |min| of v, [B, Hkv, L, D] in float64."""
    out = []
    for codes, params in ((cache.k_codes, cache.k_params), (cache.v_codes, cache.v_params)):
        at = table.cpu().long()
        c = ref.unpack(codes, cache.bits)[at].transpose(2, 3).flatten(1, 2)[:, :L].transpose(1, 2).double()
        p = params.cpu().double()[at].transpose(2, 3).flatten(1, 2)[:, :L].transpose(1, 2)
        out.append((ref.values(c, p[..., 0], p[..., 1]), ref.values(c, p[..., 0].abs(), p[..., 1].abs())))
    return out[0][0], out[1][0], out[1][1]


def check(cache, table, q, lens, L, **kw):
    got = cache.attention(q, table, ints(lens), **kw).cpu().double()
    k, v, slack = held(cache, table, L)
    o, A, S = ref.attention(q, k, v, kv_lens=lens, slack=slack, **kw)
    # weights times scale in f16: half a step of each, or, of one small against the largest, 2^-25 of that
    tol = ref.bound(o, A, S, q.shape[3], L, q.dtype, 2.0**-11) + L * 2.0**-24 * slack.amax()
    assert torch.isfinite(got).all()
    over = ((got - o).abs() - tol).max().item()
    assert over <= 0, f"{over:.3e} over the bound; worst {(got - o).abs().max().item():.3e}"


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("bits,D,group,page", FORMATS)
def test_a_new_cache_is_zeros(bits, D, group, page, dtype):
    """Slots that were never written and yet counted stand for zeros, alone and beside written ones."""
    B, Hkv, g, L = 2, 2, 5, 150
    W = -(-L // page)
    cache = llk.QuantizedKVCache.empty(B * W, page, Hkv, D, bits=bits, group_size=group)
    table = torch.arange(B * W, device="cuda", dtype=torch.int32).reshape(B, W)
    gen = torch.Generator().manual_seed(D)
    for Lq in (1, 3):
        q = torch.randn((B, Hkv * g, Lq, D), generator=gen).to(dtype).cuda()
        assert (cache.attention(q, table, ints([L, 20])) == 0).all()
    # half the tokens are skipped (-1) and counted all the same
    k, v = (torch.randn((B, Hkv, L, D), generator=gen).to(dtype).cuda() for _ in range(2))
    t = torch.arange(L, device="cuda")
    slots = (table.long()[:, t // page] * page + t % page).contiguous()
    slots[:, ::2] = -1
    cache.write(k, v, slots)
    check(cache, table, q, [L, 21], L)
    check(cache, table, q, [L, 21], L, window=30, sinks=3)


def kinds(shape, gen):
    """(name, scales) of v that a weight cannot carry as they are."""
    some = torch.rand(shape, generator=gen) < 0.3
    scale = torch.rand(shape, generator=gen) * 0.2
    sign = torch.where(torch.rand(shape, generator=gen) < 0.5, -1.0, 1.0)
    yield "all zero", torch.zeros(shape)
    yield "all -0", -torch.zeros(shape)
    yield "some zero", torch.where(some, 0.0, scale)
    yield "one token positive", torch.where(torch.arange(shape[2])[:, None] == 1, scale, 0.0)
    yield "all negative", -scale
    yield "either sign", scale * sign
    yield "zero or negative", torch.where(some, 0.0, -scale)
    yield "subnormal among others", torch.where(some, 2.0**-130, scale * sign)
    yield "far apart", scale * sign * torch.exp2(torch.randint(-60, 10, shape, generator=gen).float()) * ~some


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("bits,D,group,page", FORMATS)
def test_value_scales_of_any_sign_and_zero(bits, D, group, page, dtype):
    B, Hkv, L = 2, 2, 77
    cache, table, gen = pool(B, Hkv, L, D, bits, group, page, D + group)
    few = torch.randn((B, 3 * Hkv, 1, D), generator=gen).to(dtype).cuda()
    more = torch.randn((B, 5 * Hkv, 3, D), generator=gen).to(dtype).cuda()
    for name, scale in kinds(cache.v_params.shape[:-1], gen):
        cache.v_params[..., 0] = scale.to(BF16).cuda()
        check(cache, table, few, [L, 18], L)
        check(cache, table, more, [L, 40], L, window=25, sinks=2)
    cache.v_params.zero_()  # and minima of zero
    assert (cache.attention(few, table, ints([L, 18])) == 0).all()


@pytest.mark.parametrize("bits,D,group,page", FORMATS)
def test_key_scales_of_any_sign_and_zero(bits, D, group, page):
    B, Hkv, L = 1, 2, 77
    cache, table, gen = pool(B, Hkv, L, D, bits, group, page, D + group)
    q = torch.randn((B, 3 * Hkv, 2, D), generator=gen).to(BF16).cuda()
    for name, scale in kinds(cache.k_params.shape[:-1], gen):
        cache.k_params[..., 0] = scale.to(BF16).cuda()
        check(cache, table, q, [L], L)


def test_zero_scales_in_a_long_context():
    """Pages of zeros among written ones, over many workers and their join."""
    B, Hkv, g, L, D, page = 2, 2, 8, 9000, 128, 64
    cache, table, gen = pool(B, Hkv, L, D, 4, 128, page, 1)
    cache.v_params[::3] = 0
    cache.k_params[::3] = 0
    q = torch.randn((B, Hkv * g, 1, D), generator=gen).to(BF16).cuda()
    check(cache, table, q, [L, 5000], L)
    # the definition by the reader and the dense operator
    t = torch.arange(L, device="cuda")
    k, v = cache.read((table.long()[:, t // page] * page + t % page).contiguous(), dtype=F32)
    lens = ints([L, 5000])
    dense = llk.window_attention(q.float(), k, v, kv_lens=lens)
    got = cache.attention(q, table, lens)
    assert ((got.float() - dense).abs() <= 2.0**-7 * dense.abs() + 2.0**-10 * v.abs().amax()).all()


@pytest.mark.parametrize("bits,D,group,page", [(4, 64, 32, 16), (4, 128, 128, 64), (8, 256, 64, 16)])
def test_queries_of_any_magnitude(bits, D, group, page):
    """From the least to the largest bf16: with a scale to match, an ordinary result; with the usual one, the largest
    score takes all."""
    B, Hkv, g, L = 1, 2, 3, 90
    cache, table, gen = pool(B, Hkv, L, D, bits, group, page, D)
    q = torch.randn((B, g * Hkv, 2, D), generator=gen).to(BF16)
    for e in (-120, -60, 60, 100):
        check(cache, table, (q * 2.0**e).cuda(), [L], L, scale=D**-0.5 * 2.0**-e)
    k, v, slack = held(cache, table, L)
    for e in (40, 100, 112, 115, 119):
        big = (q * 2.0**e).to(BF16)
        got = cache.attention(big.cuda(), table, ints([L])).cpu().double()
        s = big.double() @ k.repeat_interleave(g, 1).transpose(2, 3)
        s.masked_fill_(~ref.visible(2, L, L, 2, 0, 0), -float("inf"))
        want = torch.gather(v.repeat_interleave(g, 1), 2, s.argmax(-1, keepdim=True).expand(-1, -1, -1, D))
        a = torch.gather(slack.repeat_interleave(g, 1), 2, s.argmax(-1, keepdim=True).expand(-1, -1, -1, D))
        assert ((got - want).abs() <= ref.HALF_STEP[BF16] * want.abs() + (2.0**-11 + L * 2.0**-22) * a).all(), e


@pytest.mark.parametrize("bits", [4, 8])
def test_tokens_at_the_ends_of_the_held_range(bits):
    """Infinities and +-65504 are held as up to +-65536, which bf16 and f32 read back; attention works on that."""
    B, Hkv, g, L, D = 1, 2, 3, 60, 64
    cache, table, gen = pool(B, Hkv, L, D, bits, 32, 16, 1)
    k, v = (torch.randn((B, Hkv, L, D), generator=gen) for _ in range(2))
    v[:, :, 3], v[:, :, 9, ::2], v[:, :, 20, 5], v[:, :, 31] = -65504.0, float("inf"), -float("inf"), 65504.0
    t = torch.arange(L, device="cuda")
    slots = (table.long()[:, t // 16] * 16 + t % 16).contiguous()
    cache.write(k.cuda(), v.cuda(), slots)
    for dtype in (BF16, F32):
        back = cache.read(slots, dtype=dtype)[1]
        assert torch.isfinite(back).all() and (back.abs() <= 65536 + 256).all()
        assert torch.equal(back.cpu(), held(cache, table, L)[1].float().to(dtype))
    check(cache, table, torch.randn((B, Hkv * g, 2, D), generator=gen).to(BF16).cuda(), [L], L)
