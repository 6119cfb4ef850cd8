"""llk.window_attention and QuantizedKVCache on the GPU against plain 64-bit
forms, at the sizes, masks and pages where they can go wrong.  Every tolerance
is counted from the roundings the kernels make (serving_ref.bound)."""
import math

import pytest

torch = pytest.importorskip("torch")

import dslcompiler_b200 as llk  # noqa: E402
from dslcompiler_b200 import capi  # noqa: E402
from tests import serving_ref as ref  # noqa: E402

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def rand(seed, shape, dtype, order="bhld"):
    g = torch.Generator().manual_seed(seed)
    t = torch.randn(shape, generator=g).to(dtype).cuda()
    return t.transpose(1, 2).contiguous().transpose(1, 2) if order == "blhd" else t


def ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def check_window(q, k, v, weight_step=None, **kw):
    out = llk.window_attention(q, k, v, **kw)
    o, A, S = ref.attention(q, k, v, **kw)
    if weight_step is None:  # 16-bit: weights rounded to the type; f32: not rounded
        weight_step = ref.HALF_STEP[q.dtype] if q.dtype != F32 else 0.0
    tol = ref.bound(o, A, S, q.shape[3], k.shape[2], q.dtype, weight_step)
    got = out.cpu().double()
    assert torch.isfinite(got).all()
    over = ((got - o).abs() - tol).max().item()
    assert over <= 0, f"{over:.3e} over the bound; worst {(got - o).abs().max().item():.3e}"
    return out


SHAPES = [
    # B, H, Hkv, Lq, Lk, D, window, sinks
    (1, 1, 1, 1, 1, 64, 0, 0),
    (2, 4, 2, 1, 33, 64, 0, 0),
    (1, 8, 1, 1, 517, 128, 100, 4),
    (2, 6, 2, 3, 130, 80, 50, 7),
    (1, 5, 5, 7, 300, 128, 0, 0),
    (1, 8, 2, 17, 333, 96, 64, 1),
    (1, 2, 1, 128, 128, 128, 0, 0),
    (1, 2, 2, 129, 129, 64, 17, 3),
    (2, 4, 1, 257, 300, 128, 128, 128),
    (1, 2, 2, 300, 300, 128, 1, 0),
    (1, 2, 1, 400, 700, 64, 300, 65),
    (1, 3, 3, 200, 200, 40, 31, 200),
    (1, 1, 1, 700, 700, 128, 256, 130),
    (1, 2, 1, 65, 190, 256, 70, 2),
    (1, 2, 2, 5, 90, 256, 0, 0),
    (1, 2, 1, 70, 70, 33, 20, 5),
    (1, 1, 1, 10, 4, 64, 0, 0),  # more queries than keys: the first see nothing
    (1, 2, 2, 600, 600, 112, 0, 0),
]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("B,H,Hkv,Lq,Lk,D,window,sinks", SHAPES)
def test_window_attention_shapes(B, H, Hkv, Lq, Lk, D, window, sinks, dtype):
    order = "blhd" if Lk % 2 else "bhld"
    q, k, v = (rand(s, (B, h, L, D), dtype, order) for s, h, L in ((1, H, Lq), (2, Hkv, Lk), (3, Hkv, Lk)))
    check_window(q, k, v, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("Lq", [1, 3, 150, 300])
def test_window_attention_ragged_batch(dtype, Lq):
    """Padded batches: lengths of zero and one, lengths outside the tensors, NaN behind each length; rows behind the
    queries stay as they were."""
    B, H, Hkv, Lk, D = 6, 4, 2, 300, 64
    q, k, v = (rand(s, (B, h, L, D), dtype) for s, h, L in ((4, H, Lq), (5, Hkv, Lk), (6, Hkv, Lk)))
    kv = [300, 0, 1, 177, 9999, -5]
    ql = [Lq, Lq, 1, max(1, Lq // 2), 0, Lq]
    for b, n in enumerate(kv):
        n = max(0, min(Lk, n))
        k[b, :, n:] = math.nan
        v[b, :, n:] = math.inf
    out = torch.full((B, H, Lq, D), 7.0, dtype=dtype, device="cuda")
    check_window(q, k, v, window=40, sinks=3, kv_lens=ints(kv))
    got = llk.window_attention(q, k, v, window=40, sinks=3, kv_lens=ints(kv), q_lens=ints(ql), out=out)
    assert got is out
    o, A, S = ref.attention(q, k, v, window=40, sinks=3, kv_lens=kv, q_lens=ql)
    tol = ref.bound(o, A, S, D, Lk, dtype, 0.0 if dtype == F32 else ref.HALF_STEP[dtype])
    for b, m in enumerate(ql):
        m = max(0, min(Lq, m))
        assert ((got[b, :, :m].cpu().double() - o[b, :, :m]).abs() <= tol[b, :, :m]).all(), b
        assert (got[b, :, m:] == 7.0).all(), b


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("Lq,Lk", [(2, 200), (7, 64), (200, 200), (300, 400)])
def test_window_attention_ignores_what_a_query_does_not_see(dtype, Lq, Lk):
    """An infinity or NaN in one token changes only the queries that see it, inside a tile too."""
    q, k, v = (rand(s, (1, 2, L, 64), dtype) for s, L in ((7, Lq), (8, Lk), (9, Lk)))
    kw = dict(window=30, sinks=2)
    clean = llk.window_attention(q, k, v, **kw)
    see = ref.visible(Lq, Lk, Lk, Lq, 30, 2)
    for j, bad_k, bad_v in ((Lk - 1, math.nan, math.nan), (Lk - 3, math.inf, math.inf), (Lk - 20, 0.0, -math.inf),
                            (Lk - 33, math.nan, 0.0)):
        k2, v2 = k.clone(), v.clone()
        k2[:, :, j], v2[:, :, j] = bad_k, bad_v
        out = llk.window_attention(q, k2, v2, **kw)
        blind = ~see[:, j]
        a, c = out[:, :, blind], clean[:, :, blind]
        tol = 4 * ref.HALF_STEP[dtype] * clean.abs().amax().double() if dtype != F32 else 1e-4
        assert torch.isfinite(a).all()
        assert ((a.double() - c.double()).abs() <= tol).all()
        if (~blind).any() and bad_v != 0.0:
            assert not torch.isfinite(out[:, :, ~blind]).all(-1).any()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_window_attention_views_and_out(dtype):
    """q, k, v as slices of one fused projection, odd element offsets, broadcast heads, a strided out."""
    B, L, H, Hkv, D = 2, 90, 4, 2, 64
    fused = rand(11, (B, L, H + 2 * Hkv, D), dtype)
    q, k, v = (fused[:, :, a:e].transpose(1, 2) for a, e in ((0, H), (H, H + Hkv), (H + Hkv, H + 2 * Hkv)))
    check_window(q, k, v, window=33)
    odd = rand(12, (B, Hkv, L, D + 3), dtype)[..., 1:D + 1]  # rows that do not start on 16 bytes
    check_window(q, odd, v, window=33)
    check_window(q[:, :, -2:], odd, odd, window=33)
    one = rand(13, (B, 1, L, D), dtype).expand(B, Hkv, L, D)
    check_window(q, one, one)
    check_window(q[:, :, -1:], one, one)
    room = torch.zeros((B, L, H + 1, D), dtype=dtype, device="cuda")
    out = room[:, :, :H].transpose(1, 2)
    got = llk.window_attention(q, k, v, window=33, out=out)
    assert got is out and torch.equal(out, llk.window_attention(q, k, v, window=33))
    assert (room[:, :, H] == 0).all()


def test_window_attention_large_scores_and_scale():
    """Scores far apart: the running maximum moves at every tile; a scale of its own, zero and negative too."""
    for dtype in (BF16, F16, F32):
        for Lq in (1, 200):
            q, k, v = (rand(s, (1, 2, L, 128), dtype) for s, L in ((21, Lq), (22, 200), (23, 200)))
            k = k * torch.linspace(0.1, 8.0, 200, device="cuda")[:, None].to(dtype)
            check_window(q, k, v, window=150)
            for scale in (0.0, -0.05, 0.3):
                check_window(q, k, v, scale=scale, sinks=2, window=90)


def test_window_attention_equals_llk_attention():
    """Without a window it is llk.attention (f32, causal), to both kernels' f32 sums."""
    q, k, v = (rand(s, (1, 3, 150, 64), F32) for s in (1, 2, 3))
    a, b = llk.window_attention(q, k, v), llk.attention(q, k, v, causal=True)
    assert (a - b).abs().max() <= 1e-5


def test_window_attention_empty_sizes():
    q = rand(1, (2, 4, 3, 64), BF16)
    e = torch.empty((2, 2, 0, 64), dtype=BF16, device="cuda")
    assert (llk.window_attention(q, e, e) == 0).all()
    for shape in ((0, 4, 3, 64), (2, 0, 3, 64), (2, 4, 0, 64)):
        z = torch.empty(shape, dtype=BF16, device="cuda")
        kk = torch.empty((shape[0], max(1, shape[1] // 2), 5, 64), dtype=BF16, device="cuda")
        assert llk.window_attention(z, kk, kk).shape == shape


def test_window_attention_repeats_bit_for_bit_and_on_another_stream():
    q, k, v = (rand(s, (2, 8, L, 128), BF16) for s, L in ((31, 1), (32, 3000), (33, 3000)))
    a = llk.window_attention(q, k, v, sinks=4, window=2500)
    torch.cuda.synchronize()
    for _ in range(3):
        assert torch.equal(a, llk.window_attention(q, k, v, sinks=4, window=2500))
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(10):  # at once on two streams: no scratch is shared
        outs += [llk.window_attention(q, k, v, sinks=4, window=2500, stream=s1),
                 llk.window_attention(q, k, v, sinks=4, window=2500, stream=s2)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, o) for o in outs)


def test_window_attention_captured_and_replayed():
    """Two captured graphs, replayed at once on two streams, with lengths that change between replays."""
    q, k, v = (rand(s, (2, 8, L, 64), F16) for s, L in ((41, 2), (42, 2000), (43, 2000)))
    lens = ints([2000, 700])
    llk.window_attention(q, k, v, kv_lens=lens)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o = llk.window_attention(q, k, v, kv_lens=lens, window=900, sinks=1)
        graphs.append((g, o))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for want_lens in ([2000, 700], [1, 1999], [0, 64]):
        lens.copy_(ints(want_lens))
        want = llk.window_attention(q, k, v, kv_lens=lens, window=900, sinks=1)
        torch.cuda.synchronize()
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for _, o in graphs:
            assert torch.equal(o, want)


# ------------------------------------------------------------------ the cache
def table_of(B, W, pages, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randperm(pages, generator=g)[: B * W].reshape(B, W).to(torch.int32).cuda()


def slots_of(table, page, L):
    t = torch.arange(L, device="cuda")
    return (table.long()[:, t // page] * page + t % page).contiguous()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("bits,D,group,page", [(4, 64, 32, 16), (4, 128, 128, 64), (4, 256, 64, 48), (4, 128, 32, 16),
                                               (8, 64, 64, 32), (8, 128, 32, 16), (8, 256, 128, 64)])
def test_cache_codes_are_the_definition(bits, D, group, page, dtype):
    """Codes, scales and minima bit for bit, exact ties among them; reading back gives scale * code + min."""
    B, Hkv, L = 2, 3, 50
    W = -(-L // page)
    k, v = rand(1, (B, Hkv, L, D), dtype, "blhd"), rand(2, (B, Hkv, L, D), dtype)
    k[0, 0, 0] = 5.0  # a constant group
    k[0, 1, 1, :group] = torch.linspace(0, 2**bits - 1, group).mul(2).round().div(2).to(dtype)  # halves: ties
    k[0, 1, 1, 0], k[0, 1, 1, 1] = 0.0, 2**bits - 1
    k[1, 0, 2] = 0.0
    k[1, 0, 3, 5], k[1, 0, 3, 6], k[1, 0, 3, 7] = math.nan, math.inf, -math.inf
    v[0, 0, 0] *= 1e-6
    v[0, 0, 1] *= 1e4
    cache = llk.QuantizedKVCache.empty(B * W + 1, page, Hkv, D, bits=bits, group_size=group)
    table = table_of(B, W, B * W + 1, 3)
    slots = slots_of(table, page, L)
    cache.write(k, v, slots)
    for x, codes, params, n in ((k, cache.k_codes, cache.k_params, 0), (v, cache.v_codes, cache.v_params, 1)):
        c, s, m = ref.quantise(x, bits, group)
        pg, off = (slots // page).cpu(), (slots % page).cpu()
        got = ref.unpack(codes, bits)[pg, :, off].transpose(1, 2)
        par = params.cpu().double()[pg, :, off].transpose(1, 2)
        assert torch.equal(par[..., 0], s) and torch.equal(par[..., 1], m)
        assert torch.equal(got, c.long())
        for to in (BF16, F16, F32):
            back = cache.read(slots, dtype=to)[n]
            assert torch.equal(back.cpu(), ref.values(c, s, m).float().to(to))


def test_cache_write_skips_and_last_of_a_slot_stands():
    """Padding slots are not written and read as zeros; a slot named more than once holds its last token, whatever
    CTAs the tokens fall to; all other slots stay as they were."""
    Hkv, D, page, pages = 2, 64, 16, 80
    for T in (1, 2, 7, 300, 5000):
        cache = llk.QuantizedKVCache.empty(pages, page, Hkv, D)
        cache.k_codes.fill_(171)
        g = torch.Generator().manual_seed(T)
        slots = torch.randint(0, pages * page, (1, T), generator=g)
        slots[torch.rand(1, T, generator=g) < 0.1] = -1
        if T > 2:
            slots[0, T // 2], slots[0, T // 3] = pages * page, 2**40
        k, v = rand(T, (1, Hkv, T, D), BF16), rand(T + 1, (1, Hkv, T, D), BF16)
        cache.write(k, v, slots.cuda())
        last = {int(s): t for t, s in enumerate(slots[0].tolist()) if 0 <= s < pages * page}
        full = torch.arange(pages * page)[None].cuda()
        gk, gv = cache.read(full, dtype=F32)
        for x, got in ((k, gk), (v, gv)):
            want = ref.values(*ref.quantise(x, 4, 64)).float()
            for s, t in last.items():
                assert torch.equal(got[0, :, s].cpu(), want[0, :, t]), (T, s)
        rest = torch.tensor([s for s in range(pages * page) if s not in last], dtype=torch.long)
        assert (cache.k_codes.cpu()[rest // page, :, rest % page] == 171).all()
        assert (cache.v_params.cpu()[rest // page, :, rest % page] == 0).all()
        rk, rv = cache.read(torch.tensor([[-1, pages * page, 2**62, -(2**62)]]).cuda(), dtype=F16)
        assert (rk == 0).all() and (rv == 0).all()


def filled(B, Hkv, L, D, bits, group, page, seed, spare=2):
    W = -(-L // page) if L else 1
    cache = llk.QuantizedKVCache.empty(B * W + spare, page, Hkv, D, bits=bits, group_size=group)
    # pages that no token was written to hold the worst there is
    cache.k_params.fill_(math.nan)
    cache.v_params.fill_(math.inf)
    table = table_of(B, W, B * W + spare, seed)
    if L:
        g = torch.Generator().manual_seed(seed)
        k, v = (torch.randn((B, Hkv, L, D), generator=g) * torch.exp(torch.randn((Hkv, 1, D), generator=g)) +
                torch.randn((Hkv, 1, D), generator=g) for _ in range(2))
        cache.write(k.cuda(), v.cuda(), slots_of(table, page, L))
    return cache, table


def cache_dense(cache, table, L):
    """What the cache holds, in float64: k, v and |s code| + |min| of v."""
    W = table.shape[1]
    out = []
    for codes, params in ((cache.k_codes, cache.k_params), (cache.v_codes, cache.v_params)):
        c = ref.unpack(codes, cache.bits)[table.cpu().long()].transpose(2, 3).flatten(1, 2)[:, :L].transpose(1, 2)
        p = params.cpu().double()[table.cpu().long()].transpose(2, 3).flatten(1, 2)[:, :L].transpose(1, 2)
        out.append((c.double(), p[..., 0], p[..., 1]))
    (kc, ks, km), (vc, vs, vm) = out
    return ref.values(kc, ks, km), ref.values(vc, vs, vm), ref.values(vc, vs, torch.zeros_like(vm)) + \
        ref.values(torch.zeros_like(vc), vs, vm.abs())


def check_cache(cache, table, q, lens, L, **kw):
    out = cache.attention(q, table, ints(lens), **{k: ints(x) if k == "q_lens" else x for k, x in kw.items()})
    k, v, slack = cache_dense(cache, table, L)
    o, A, S = ref.attention(q, k, v, kv_lens=lens, slack=slack, **kw)
    # weights times scale in f16
    tol = ref.bound(o, A, S, q.shape[3], L, q.dtype, 2.0**-11)
    got = out.cpu().double()
    assert torch.isfinite(got).all()
    over = ((got - o).abs() - tol).max().item()
    assert over <= 0, f"{over:.3e} over the bound; worst {(got - o).abs().max().item():.3e}"


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("bits,D,group,page", [(4, 64, 32, 16), (4, 64, 64, 32), (4, 128, 32, 16), (4, 128, 64, 48),
                                               (4, 128, 128, 64), (4, 256, 32, 16), (4, 256, 64, 16),
                                               (4, 256, 128, 32), (8, 64, 32, 16), (8, 64, 64, 32), (8, 128, 32, 16),
                                               (8, 128, 64, 16), (8, 128, 128, 64), (8, 256, 32, 16), (8, 256, 64, 16),
                                               (8, 256, 128, 32)])
def test_cache_attention_formats(bits, D, group, page, dtype):
    B, H, Hkv, L = 3, 10, 2, 333
    cache, table = filled(B, Hkv, L, D, bits, group, page, 7)
    q = rand(8, (B, H, 1, D), dtype)
    lens = [333, 17, 160]
    check_cache(cache, table, q, lens, L)
    check_cache(cache, table, q, lens, L, window=50, sinks=5)
    check_cache(cache, table, rand(9, (B, H, 3, D), dtype, "blhd"), lens, L, window=20, sinks=1)


@pytest.mark.parametrize("g", [1, 2, 5, 8, 9, 16, 24])
@pytest.mark.parametrize("Lq", [1, 2, 4, 20])
def test_cache_attention_rows(g, Lq):
    """Any number of query heads a key head and queries a sequence, ragged queries among them."""
    B, Hkv, L, D = 3, 2, 70, 64
    cache, table = filled(B, Hkv, L, D, 4, 64, 16, g)
    q = rand(g, (B, g * Hkv, Lq, D), BF16)
    check_cache(cache, table, q, [70, 33, 20], L, window=25, sinks=3)
    check_cache(cache, table, q, [70, 1, 0], L, q_lens=[Lq, max(1, Lq - 1), 0])


@pytest.mark.parametrize("L,window,sinks", [(1, 0, 0), (15, 0, 0), (16, 0, 0), (17, 0, 0), (64, 1, 0), (200, 16, 16),
                                            (200, 17, 1), (200, 184, 15), (1000, 129, 40), (5000, 0, 0),
                                            (5000, 4000, 4), (5000, 300, 4500)])
def test_cache_attention_lengths_and_windows(L, window, sinks):
    B, H, Hkv, D = 2, 8, 1, 128
    cache, table = filled(B, Hkv, L, D, 4, 128, 16, L)
    q = rand(L, (B, H, 1, D), BF16)
    check_cache(cache, table, q, [L, max(0, L - 13)], L, window=window, sinks=sinks)


def test_cache_attention_bad_pages_and_tables():
    """Entries outside the pool hide their tokens; rows of a wider table; empty sequences give zeros."""
    B, H, Hkv, L, D, page = 3, 4, 2, 100, 64, 16
    cache, table = filled(B, Hkv, L, D, 4, 64, page, 5)
    q = rand(6, (B, H, 1, D), BF16)
    wide = torch.full((B, table.shape[1] + 3), -7, dtype=torch.int32, device="cuda")
    wide[:, : table.shape[1]] = table
    want = cache.attention(q, table, ints([100, 50, 0]))
    assert torch.equal(want, cache.attention(q, wide[:, : table.shape[1]], ints([100, 50, 0])))
    assert (want[2] == 0).all()
    bad = table.clone()
    bad[0, 2], bad[1, 0], bad[1, 1] = -1, cache.num_pages, 2**31 - 1
    got = cache.attention(q, bad, ints([100, 32, 100]))
    assert (got[1] == 0).all() and torch.isfinite(got).all()
    k, v, slack = cache_dense(cache, table, L)
    keep = torch.ones(L, dtype=torch.bool)
    keep[32:48] = False
    o, A, S = ref.attention(q[:1, :, :], k[:1, :, keep], v[:1, :, keep], slack=slack[:1, :, keep])
    assert ((got[:1].cpu().double() - o).abs() <= ref.bound(o, A, S, D, L, BF16, 2.0**-11)).all()
    # lengths beyond the table are cut to it (its first 6 pages of tokens)
    assert torch.equal(cache.attention(q, table[:, :6], ints([10**6, 50, -3])),
                       cache.attention(q, table[:, :6], ints([96, 50, 0])))


def test_cache_attention_scales_of_all_sizes():
    """Groups whose scales differ by many orders, constant rows (no scale at all), large queries."""
    B, H, Hkv, L, D = 1, 2, 1, 64, 64
    cache, table = filled(B, Hkv, L, D, 4, 64, 16, 5)
    g = torch.Generator().manual_seed(1)
    k = torch.randn((B, Hkv, L, D), generator=g)
    v = torch.randn((B, Hkv, L, D), generator=g) * (10.0 ** torch.linspace(-9, 4, L))[:, None]
    v[0, 0, ::5] = 3.0
    cache.write(k.cuda(), v.cuda(), slots_of(table, 16, L))
    for f in (1.0, 1e-6, 1e4):
        q = (torch.randn((B, H, 1, D), generator=g) * f).to(BF16).cuda()
        check_cache(cache, table, q, [L], L, scale=0.125 / f)
    check_cache(cache, table, torch.zeros((B, H, 1, D), dtype=BF16, device="cuda"), [L], L)


def test_cache_attention_streams_graphs_and_repeats():
    B, H, Hkv, L, D = 2, 8, 2, 4000, 128
    cache, table = filled(B, Hkv, L, D, 4, 64, 64, 5)
    q, lens = rand(1, (B, H, 1, D), BF16), ints([4000, 1234])
    a = cache.attention(q, table, lens)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(10):
        outs += [cache.attention(q, table, lens, stream=s1), cache.attention(q, table, lens, stream=s2)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, o) for o in outs)
    k, v = rand(2, (B, Hkv, 1, D), BF16), rand(3, (B, Hkv, 1, D), BF16)
    slots = torch.stack([table[0, 3999 // 64] * 64 + 3999 % 64, table[1, 1233 // 64] * 64 + 1233 % 64]).long()[:, None]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.write(k, v, slots)
        o = cache.attention(q, table, lens)
    for seed in (5, 6):
        k.copy_(rand(seed, k.shape, BF16))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, cache.attention(q, table, lens))
        assert not torch.equal(o, a)


def test_serving_run_together():
    """A prompt and the steps after it, as a program runs them: rope, the cache's write, windowed attention of the
    prompt, then single tokens over the cache; a second chunk over what reads back."""
    B, H, Hkv, D, page, L, steps = 2, 8, 2, 64, 16, 100, 5
    W = -(-(L + steps) // page)
    cache = llk.QuantizedKVCache.empty(B * W, page, Hkv, D, bits=8, group_size=32)
    table = table_of(B, W, B * W, 1)
    all_slots = slots_of(table, page, L + steps)
    kw = dict(window=40, sinks=4)
    g = torch.Generator().manual_seed(3)
    qs, ks, vs = (torch.randn((B, h, L + steps, D), generator=g).cuda() for h in (H, Hkv, Hkv))
    pos = torch.arange(L + steps, device="cuda")
    qr, kr = llk.rope(qs, pos), llk.rope(ks, pos)
    o = llk.window_attention(qr[:, :, :L].to(BF16), kr[:, :, :L].to(BF16), vs[:, :, :L].to(BF16), **kw)
    exact, A, S = ref.attention(qr[:, :, :L].to(BF16), kr[:, :, :L].to(BF16), vs[:, :, :L].to(BF16), **kw)
    assert ((o.cpu().double() - exact).abs() <= ref.bound(exact, A, S, D, L, BF16, 2.0**-8)).all()
    cache.write(kr[:, :, :L], vs[:, :, :L], all_slots[:, :L].contiguous())
    for t in range(L, L + steps):
        cache.write(kr[:, :, t:t + 1], vs[:, :, t:t + 1], all_slots[:, t:t + 1].contiguous())
        q = qr[:, :, t:t + 1].to(BF16)
        check_cache(cache, table, q, [t + 1] * B, t + 1, **kw)
    # the last 20 tokens as a chunk over the cache read back, against the cache's own attention of the same tokens
    k, v = cache.read(all_slots, dtype=F16)
    q = qr[:, :, -20:].to(F16)
    a = llk.window_attention(q, k, v, **kw)
    b = cache.attention(q, table, ints([L + steps] * B), **kw)
    # f16 values read back are off by half a step each; scores move by that times |q k|
    kd, vd, slack = cache_dense(cache, table, L + steps)
    o, A, S = ref.attention(q, kd, vd, slack=slack, **kw)
    tol = ref.bound(o, A, S, D, L + steps, F16, 2.0**-11)
    assert ((b.cpu().double() - o).abs() <= tol).all()
    assert ((a.cpu().double() - o).abs() <= tol + (2.0**-11 + 4 * 2.0**-11 * S) * A).all()


def test_serving_refusals_on_device():
    q = rand(1, (1, 4, 2, 64), BF16)
    k = rand(2, (1, 2, 8, 64), BF16)

    def status(f, *a, **kw):
        with pytest.raises(llk.LLKError) as e:
            f(*a, **kw)
        return e.value.status

    assert status(llk.window_attention, q, rand(3, (1, 3, 8, 64), BF16), rand(3, (1, 3, 8, 64), BF16)) == capi.LLK_ERR_SHAPE
    assert status(llk.window_attention, q, rand(3, (1, 2, 8, 32), BF16), k) == capi.LLK_ERR_SHAPE
    assert status(llk.window_attention, q, k, k, out=q) == capi.LLK_ERR_ARG
    assert status(llk.window_attention, q, k, k, out=torch.zeros((1, 4, 1, 64), dtype=BF16, device="cuda").expand(
        1, 4, 2, 64)) == capi.LLK_ERR_ALIGN
    wide = rand(4, (1, 1, 2, 300), BF16)
    assert status(llk.window_attention, wide, wide, wide.clone()) == capi.LLK_ERR_UNSUPPORTED
    cache = llk.QuantizedKVCache.empty(2, 16, 2, 64)
    table, lens = ints([[0, 1]]), ints([20])
    assert status(cache.attention, rand(1, (1, 3, 1, 64), BF16), table, lens) == capi.LLK_ERR_SHAPE
    assert status(cache.attention, rand(1, (1, 4, 1, 128), BF16), table, lens) == capi.LLK_ERR_SHAPE
    with pytest.raises(TypeError):
        cache.attention(rand(1, (1, 4, 1, 64), F32), table, lens)
    assert status(cache.write, rand(1, (1, 3, 1, 64), BF16), rand(1, (1, 3, 1, 64), BF16),
                  ints([[0]], torch.int64)) == capi.LLK_ERR_SHAPE
    with pytest.raises(ValueError):
        cache.write(k[:, :, :1], k[:, :, :1], ints([0], torch.int64))
    kk = torch.zeros((1, 2, 1, 64), dtype=BF16, device="cuda")
    assert status(cache.read, ints([[0]], torch.int64), out=(kk, kk)) == capi.LLK_ERR_ARG
    # a captured C call without scratch does not take the library's buffer
    import ctypes

    big = rand(5, (1, 2, 4000, 64), BF16)
    o = torch.empty_like(q)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        from dslcompiler_b200.serving import _tensor4d
        from dslcompiler_b200.swiglu import _stream_of, gpu_context

        rc = capi.lib().llk_window_attention(_tensor4d(q), _tensor4d(big, 1), _tensor4d(big.clone(), 2), _tensor4d(o, 3),
                                             capi.LLK_DTYPE_BF16, None, None, 0, 0, 0.125, None,
                                             ctypes.byref(gpu_context(0, _stream_of(q, None))))
    assert rc == capi.LLK_ERR_NOMEM


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("bits", [4, 8])
def test_cache_codes_next_to_borders(bits, dtype):
    """Groups whose elements lie on the borders between two codes, a step of the type above and below them, and
    next to a minimum that their difference to does not fit 24 bits: the codes are those of 64 bits."""
    D, L, page = 128, 512, 64
    g = torch.Generator().manual_seed(bits)
    top = 2**bits - 1
    scale = torch.exp2(torch.randint(-6, 7, (1, 1, L, 1), generator=g).double()) * (
        1 + torch.randint(0, 128, (1, 1, L, 1), generator=g) / 128.0)
    low = torch.randn((1, 1, L, 1), generator=g).double() * scale * 4
    low = low.to(BF16).double()
    border = low + scale * (torch.randint(0, top, (1, 1, L, D), generator=g).double() + 0.5)
    x = border.to(dtype)
    step = torch.randint(-1, 2, x.shape, generator=g)
    bump = {BF16: torch.int16, F16: torch.int16, F32: torch.int32}[dtype]
    x = (x.view(bump) + torch.where(x != 0, step, 0).to(bump)).view(dtype)
    x[..., 0], x[..., 1] = low[..., 0].to(dtype), (low + top * scale)[..., 0].to(dtype)
    x[0, 0, ::3, 2::5] = (torch.randn((len(range(0, L, 3)), len(range(2, D, 5))), generator=g) * 2.0**-30).to(dtype)
    x[0, 0, ::7] = x[0, 0, ::7].abs()
    x[0, 0, ::7, 3] = 2.0**-24
    cache = llk.QuantizedKVCache.empty(L // page, page, 1, D, bits=bits, group_size=128)
    cache.write(x.cuda(), x.cuda(), torch.arange(L)[None].cuda())
    c, s, m = ref.quantise(x, bits, 128)
    got = ref.unpack(cache.k_codes, bits).reshape(L, D)
    assert torch.equal(cache.k_params.cpu().double().reshape(L, 2), torch.cat([s, m], -1)[0, 0])
    assert torch.equal(got, c.long()[0, 0])
