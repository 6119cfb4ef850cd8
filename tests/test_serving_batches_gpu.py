"""The serving attention kernels where one CTA has many pieces of work: more
query tiles than SMs, more sequences' ends in a worker's share than one, CTAs
of the cache's writer with any number of tokens.  Against plain forms in 64
bits, whole tensors at a time; tolerances are serving_ref.bound's."""
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


def rand(seed, shape, dtype):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def plain(q, k, v, slack, q_lens, kv_lens, window, sinks):
    """ref.attention's (o, A, S) on the GPU, a sequence at a time; k, v and slack hold no NaN or infinity."""
    B, H, Lq, D = q.shape
    g, Lk = H // k.shape[1], k.shape[2]
    o, A = (torch.zeros((B, H, Lq, D), dtype=torch.float64, device="cuda") for _ in range(2))
    S = torch.zeros((B, H, Lq, 1), dtype=torch.float64, device="cuda")
    for b in range(B):
        qb = q[b].double() / math.sqrt(D)
        kb, vb, ab = (t[b].double().repeat_interleave(g, 0) for t in (k, v, slack))
        see = ref.visible(Lq, Lk, kv_lens[b], q_lens[b], window, sinks).cuda()
        s = (qb @ kb.transpose(1, 2)).masked_fill(~see, -math.inf)
        top = s.amax(-1, keepdim=True)
        w = torch.exp(s - top.masked_fill(top == -math.inf, 0.0))
        total = w.sum(-1, keepdim=True)
        w = w / total.masked_fill(total == 0, 1.0)
        o[b], A[b] = w @ vb, w @ ab
        S[b] = (qb.abs() @ kb.abs().transpose(1, 2)).masked_fill(~see, 0.0).amax(-1, keepdim=True)
    return o, A, S


def check(got, o, A, S, D, keys, dtype, step, q_lens, left):
    tol = ref.bound(o, A, S, D, keys, dtype, step)
    for b, m in enumerate(q_lens):
        over = ((got[b, :, :m].double() - o[b, :, :m]).abs() - tol[b, :, :m]).amax().item() if m else 0.0
        assert over <= 0, (b, over)
        assert (got[b, :, m:] == left).all(), b


def lens_of(seed, B, top, ends):
    g = torch.Generator().manual_seed(seed)
    return (ends + torch.randint(0, top + 1, (B,), generator=g).tolist())[:B]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D,Hkv,g,L,window,sinks", [(128, 4, 4, 700, 0, 0), (128, 8, 2, 600, 130, 5),
                                                    (64, 2, 10, 515, 300, 260), (80, 20, 1, 400, 17, 40),
                                                    (72, 5, 4, 257, 0, 0)])
def test_window_attention_more_tiles_than_sms(D, Hkv, g, L, window, sinks, dtype):
    """Padded prompts of uneven length, in runs: a CTA goes from a long tile to a short one, to an empty one."""
    B = 14
    q, k, v = rand(1, (B, Hkv * g, L, D), dtype), rand(2, (B, Hkv, L, D), dtype), rand(3, (B, Hkv, L, D), dtype)
    kv = lens_of(L, B, L, [L, 0, 1, L])
    ql = [min(n, m) for n, m in zip(kv, lens_of(L + 1, B, L, [L, 0, 1, 2, 0]))]
    ql[5] = min(L, kv[5] + 40)  # more queries than keys: the first see nothing
    out = torch.full_like(q, 7.0)
    llk.window_attention(q, k, v, window=window, sinks=sinks, q_lens=ints(ql), kv_lens=ints(kv), out=out)
    o, A, S = plain(q, k, v, v.abs(), ql, kv, window, sinks)
    check(out, o, A, S, D, L, dtype, 0.0 if dtype == F32 else ref.HALF_STEP[dtype], ql, 7.0)
    again = torch.full_like(q, 7.0)
    llk.window_attention(q, k, v, window=window, sinks=sinks, q_lens=ints(ql), kv_lens=ints(kv), out=again)
    assert torch.equal(out, again)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D,Hkv,g,Lq,L,window,sinks", [(128, 8, 4, 1, 900, 0, 0), (128, 8, 4, 3, 700, 200, 9),
                                                       (64, 32, 1, 2, 513, 0, 0), (80, 4, 20, 1, 640, 128, 128),
                                                       (256, 4, 2, 1, 500, 100, 1), (96, 8, 8, 7, 300, 0, 0)])
def test_window_attention_many_short_sequences(D, Hkv, g, Lq, L, window, sinks, dtype):
    B = 50
    q, k, v = rand(1, (B, Hkv * g, Lq, D), dtype), rand(2, (B, Hkv, L, D), dtype), rand(3, (B, Hkv, L, D), dtype)
    kv = lens_of(L, B, L, [L, 0, 1, 0, 0, 127, 128, 129])
    ql = lens_of(Lq, B, Lq, [Lq, Lq, 0, Lq, 0])
    out = torch.full_like(q, 7.0)
    llk.window_attention(q, k, v, window=window, sinks=sinks, q_lens=ints(ql), kv_lens=ints(kv), out=out)
    o, A, S = plain(q, k, v, v.abs(), ql, kv, window, sinks)
    check(out, o, A, S, D, L, dtype, ref.HALF_STEP[dtype], ql, 7.0)


@pytest.mark.parametrize("B,D,Hkv,g,Lq,L,window,sinks", [(50, 128, 8, 4, 1, 900, 0, 0), (2, 128, 2, 4, 3, 5000, 0, 0),
                                                         (1, 64, 4, 1, 1, 4097, 0, 0), (3, 80, 2, 5, 2, 2000, 700, 33),
                                                         (2, 256, 2, 9, 1, 3000, 0, 0), (4, 40, 3, 1, 20, 1111, 100, 7),
                                                         (2, 4, 2, 2, 5, 600, 0, 0), (1, 128, 1, 16, 7, 2500, 17, 300),
                                                         (9, 252, 4, 2, 1, 640, 64, 1)])
def test_window_attention_f32_few_queries(B, D, Hkv, g, Lq, L, window, sinks):
    q, k, v = rand(1, (B, Hkv * g, Lq, D), F32), rand(2, (B, Hkv, L, D), F32), rand(3, (B, Hkv, L, D), F32)
    kv = lens_of(L, B, L, [L, 1, 0, 127])
    ql = lens_of(Lq, B, Lq, [Lq, Lq, Lq, 0])
    out = torch.full_like(q, 7.0)
    llk.window_attention(q, k, v, window=window, sinks=sinks, q_lens=ints(ql), kv_lens=ints(kv), out=out)
    o, A, S = plain(q, k, v, v.abs(), ql, kv, window, sinks)
    check(out, o, A, S, D, L, F32, 0.0, ql, 7.0)
    # infinities and NaN where no query looks, and in the last key of the first sequence
    for b, n in enumerate(kv):
        k[b, :, n:], v[b, :, n:] = math.nan, math.inf
    if window and L > 2 * (window + Lq):
        k[0, :, sinks : L - window - Lq - 20], v[0, :, sinks : L - window - Lq - 20] = math.inf, math.nan
    again = torch.full_like(q, 7.0)
    llk.window_attention(q, k, v, window=window, sinks=sinks, q_lens=ints(ql), kv_lens=ints(kv), out=again)
    assert torch.equal(out, again)
    v[0, :, L - 1] = math.inf
    llk.window_attention(q, k, v, window=window, sinks=sinks, q_lens=ints(ql), kv_lens=ints(kv), out=again)
    assert torch.equal(out[1:], again[1:])
    assert not torch.isfinite(again[0, :, Lq - 1]).any()
    before = out[0, :, : Lq - 1].double()  # the queries before the last do not see it
    assert ((again[0, :, : Lq - 1].double() - before).abs() <= 2 * ref.bound(
        o[0, :, : Lq - 1], A[0, :, : Lq - 1], S[0, :, : Lq - 1], D, L, F32, 0.0)).all()


def pool_of(B, Hkv, L, D, bits, group, page):
    """A cache of random contents, its table, and (k, v, |s code| + |min| of v) in float64."""
    W = -(-L // page)
    cache = llk.QuantizedKVCache.empty(B * W + 3, page, Hkv, D, bits=bits, group_size=group)
    g = torch.Generator().manual_seed(L)
    table = torch.randperm(B * W + 3, generator=g)[: B * W].reshape(B, W).to(torch.int32)
    dense = []
    for codes, params in ((cache.k_codes, cache.k_params), (cache.v_codes, cache.v_params)):
        codes.copy_(torch.randint(0, 256, codes.shape, generator=g, dtype=torch.uint8))
        scale = torch.rand(params.shape[:-1], generator=g) * 0.2
        params.copy_(torch.stack([scale, -torch.rand(scale.shape, generator=g)], -1).to(BF16))
        c = ref.unpack(codes, bits)[table.long()].double()
        p = params.cpu()[table.long()].double()
        s, m = p[..., 0], p[..., 1]
        x = [ref.values(c, s, m), ref.values(c, s, torch.zeros_like(m)) + ref.values(torch.zeros_like(c), s, m.abs())]
        dense.append([t.transpose(1, 2).flatten(2, 3)[:, :, :L].cuda() for t in x])
    (k, _), (v, slack) = dense
    return cache, table.cuda(), k, v, slack


@pytest.mark.parametrize("bits,D,group,Hkv,g,Lq,L,window,sinks",
                         [(4, 128, 64, 8, 4, 1, 700, 0, 0), (4, 128, 128, 8, 8, 2, 500, 150, 7),
                          (4, 64, 32, 16, 1, 1, 600, 0, 0), (8, 64, 64, 32, 1, 4, 400, 128, 4),
                          (8, 128, 32, 8, 5, 1, 333, 0, 0), (4, 256, 64, 4, 3, 3, 450, 40, 200),
                          (8, 256, 128, 6, 2, 1, 300, 0, 0)])
def test_cache_attention_many_short_sequences(bits, D, group, Hkv, g, Lq, L, window, sinks):
    B = 45
    cache, table, k, v, slack = pool_of(B, Hkv, L, D, bits, group, 48)
    q = rand(1, (B, Hkv * g, Lq, D), BF16)
    kv = lens_of(L, B, L, [L, 0, 1, 0, 0, 127, 128, 129])
    ql = lens_of(Lq, B, Lq, [Lq, Lq, 0, Lq, 0])
    out = torch.full_like(q, 7.0)
    cache.attention(q, table, ints(kv), window=window, sinks=sinks, q_lens=ints(ql), out=out)
    o, A, S = plain(q, k, v, slack, ql, kv, window, sinks)
    check(out, o, A, S, D, L, BF16, 2.0**-11, ql, 7.0)
    # the second half's sequences lose their pages: zeros, and the first half's results stay
    lost = table.clone()
    lost[B // 2 :] = -1
    got = torch.full_like(q, 7.0)
    cache.attention(q, lost, ints(kv), window=window, sinks=sinks, q_lens=ints(ql), out=got)
    check(got[: B // 2], o[: B // 2], A[: B // 2], S[: B // 2], D, L, BF16, 2.0**-11, ql[: B // 2], 7.0)
    for b in range(B // 2, B):
        assert (got[b, :, : ql[b]] == 0).all() and (got[b, :, ql[b] :] == 7.0).all()


@pytest.mark.parametrize("bits,D,group,Lq", [(4, 64, 64, 1), (4, 64, 32, 3), (4, 128, 128, 1), (4, 128, 64, 1),
                                             (4, 128, 32, 4), (4, 256, 64, 1), (8, 64, 32, 2), (8, 128, 32, 1),
                                             (8, 128, 128, 5), (8, 256, 128, 1)])
def test_cache_attention_f16_keeps_its_precision(bits, D, group, Lq):
    """In f16 the weights are sums of two f16: 2^-22 of each, and of a small one 2^-25 of the largest."""
    B, Hkv, g, L = 3, 4, 4, 333
    cache, table, k, v, slack = pool_of(B, Hkv, L, D, bits, group, 16)
    lens = [L, 3, 40]
    q = rand(1, (B, Hkv * g, Lq, D), F16)
    out = cache.attention(q, table, ints(lens))
    o, A, S = plain(q, k, v, slack, [Lq] * B, lens, 0, 0)
    tol = ref.bound(o, A, S, D, L, F16, 2.0**-22) + L * 2.0**-24 * slack.amax()
    assert ((out.double() - o).abs() <= tol).all()


@pytest.mark.parametrize("dtype,bits", [(BF16, 4), (F16, 8), (F32, 4)])
@pytest.mark.parametrize("B,L,Hkv,D", [(1, 1, 1, 64), (3, 5, 7, 64), (1, 149, 3, 128), (2, 4097, 1, 64),
                                       (5, 1111, 2, 256), (1, 9001, 4, 128)])
def test_cache_write_any_number_of_tokens(B, L, Hkv, D, dtype, bits):
    """Slots in any order, from any 8-byte boundary; some named twice, some outside the cache."""
    page, n = 32, B * L
    cache = llk.QuantizedKVCache.empty(-(-2 * n // page), page, Hkv, D, bits=bits, group_size=32)
    g = torch.Generator().manual_seed(n)
    slots = torch.randperm(2 * n, generator=g)[:n]
    slots[torch.rand(n, generator=g) < 0.1] = -1
    twice = torch.rand(n, generator=g) < 0.2
    slots[twice] = slots[torch.randint(0, n, (int(twice.sum()),), generator=g)]
    held = torch.empty(n + 1, dtype=torch.int64, device="cuda")[1 if n % 2 else 0 :][:n].copy_(slots).reshape(B, L)
    k, v = rand(1, (B, Hkv, L, D), dtype), rand(2, (B, Hkv, L, D), dtype)
    cache.write(k, v, held)
    last = {int(s): i for i, s in enumerate(slots.tolist()) if s >= 0}
    at, who = torch.tensor(list(last.keys())).long(), torch.tensor(list(last.values())).long()
    for x, codes, params in ((k, cache.k_codes, cache.k_params), (v, cache.v_codes, cache.v_params)):
        want, s, m = ref.quantise(x.transpose(1, 2).reshape(n, Hkv, D)[who.cuda()], bits, 32)
        got = ref.unpack(codes, bits).transpose(1, 2).reshape(-1, Hkv, D)
        p = params.cpu().double().transpose(1, 2).reshape(-1, Hkv, D // 32, 2)
        assert torch.equal(got[at].double(), want) and torch.equal(p[at, ..., 0], s) and torch.equal(p[at, ..., 1], m)
        rest = torch.ones(got.shape[0], dtype=torch.bool)
        rest[at] = False
        assert (got[rest] == 0).all() and (p[rest] == 0).all()
    # and read back: as the codes say, zeros where there is no slot
    rk, rv = cache.read(held, dtype=F32)
    for x, out in ((cache.k_codes, rk), (cache.v_codes, rv)):
        c = ref.unpack(x, bits).transpose(1, 2).reshape(-1, Hkv, D)
        p = (cache.k_params if x is cache.k_codes else cache.v_params).cpu().double().transpose(1, 2).reshape(
            -1, Hkv, D // 32, 2)
        dense = torch.cat([ref.values(c.double(), p[..., 0], p[..., 1]), torch.zeros((1, Hkv, D), dtype=torch.float64)])
        # code * scale of 16 bits is exact, the sum rounds once
        want = dense[slots].reshape(B, L, Hkv, D).transpose(1, 2).float()
        assert torch.equal(out.cpu(), want)
