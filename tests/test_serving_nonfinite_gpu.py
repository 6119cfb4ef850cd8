"""Infinities and NaN among the keys and values of long prompts and of few
queries: what sees them is not finite by the definition, what does not see them
is untouched, and a call with one takes about as long as one without."""
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


def expected(q, k, v, n, m, window, sinks):
    """(o, A, S) of one sequence's head group in float64 on the GPU: q [g, Lq, D], k, v [Lk, D].  A weight is above
    zero wherever the score is finite, so an infinity or NaN among the values that a row sees decides its component."""
    Lq, Lk = q.shape[1], k.shape[0]
    q, k, v = q.double() / math.sqrt(q.shape[2]), k.double(), v.double()
    see = ref.visible(Lq, Lk, n, m, window, sinks).cuda()
    ok_v = torch.where(torch.isfinite(v), v, 0.0)
    ok_k = torch.where(torch.isfinite(k), k, 0.0)
    s = (q @ ok_k.T).masked_fill(~see, -math.inf)
    top = s.amax(-1, keepdim=True)
    w = torch.exp(s - top.masked_fill(top == -math.inf, 0.0))
    total = w.sum(-1, keepdim=True)
    w = w / total.masked_fill(total == 0, 1.0)
    o, A = w @ ok_v, w @ ok_v.abs()
    f = see.double()
    nan, up, down = (f @ x.double() > 0 for x in (torch.isnan(v), v == math.inf, v == -math.inf))
    o = o.masked_fill(up, math.inf).masked_fill(down, -math.inf).masked_fill(nan | (up & down), math.nan)
    o = o.masked_fill((f @ torch.isnan(k).any(-1, keepdim=True).double()) > 0, math.nan)
    S = (q.abs() @ ok_k.abs().T).masked_fill(~see, 0.0).amax(-1, keepdim=True)
    return o, A, S


def compare(got, o, A, S, D, keys, dtype):
    got = got.double()
    assert torch.equal(torch.isnan(got), torch.isnan(o))
    assert torch.equal(torch.where(torch.isinf(got), got, 0.0), torch.where(torch.isinf(o), o, 0.0))
    fine = torch.isfinite(o)
    step = 0.0 if dtype == F32 else ref.HALF_STEP[dtype]
    tol = ref.bound(torch.where(fine, o, 0.0), A, S, D, keys, dtype, step)
    over = torch.where(fine, (got - o).abs() - tol, -1.0).max().item()
    assert over <= 0, over


# B, H, Hkv, Lq, Lk, D, window, sinks: prompts on the tensor cores and on the CUDA cores, few queries
SHAPES = [(2, 8, 2, 1500, 1500, 128, 0, 0), (2, 8, 2, 1500, 1500, 128, 300, 5), (2, 8, 2, 1101, 1300, 64, 257, 40),
          (2, 6, 2, 700, 700, 256, 0, 0), (2, 6, 2, 700, 700, 256, 100, 70), (2, 4, 2, 600, 650, 72, 130, 3),
          (2, 8, 2, 7, 3000, 128, 0, 0), (2, 8, 2, 7, 3000, 128, 500, 4), (2, 4, 2, 5, 900, 256, 90, 1),
          (2, 4, 2, 40, 2500, 64, 300, 8), (2, 8, 2, 1, 3000, 128, 0, 0), (2, 4, 2, 3, 333, 33, 50, 2)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("B,H,Hkv,Lq,Lk,D,window,sinks", SHAPES)
def test_infinities_and_nan_in_one_head(B, H, Hkv, Lq, Lk, D, window, sinks, dtype):
    q, k, v = rand(1, (B, H, Lq, D), dtype), rand(2, (B, Hkv, Lk, D), dtype), rand(3, (B, Hkv, Lk, D), dtype)
    kw = dict(window=window, sinks=sinks)
    clean = llk.window_attention(q, k, v, **kw)
    g, first = H // Hkv, Lk - Lq
    places = sorted({0, 3, Lk // 3, first + Lq // 2, max(0, Lk - 40), Lk - 1, max(0, first - 60)})
    bad = [("one component NaN", lambda k, v, j: v[j, 1:2].fill_(math.nan)),
           ("infinities of both signs in two tokens", lambda k, v, j: (v[j, 2:3].fill_(math.inf),
                                                                       v[(j + Lk // 5) % Lk, 2:4].fill_(-math.inf))),
           ("a token all NaN", lambda k, v, j: (k[j].fill_(math.nan), v[j].fill_(math.nan)))]
    for name, put in bad:
        for j in places:
            k2, v2 = k.clone(), v.clone()
            put(k2[1, 1], v2[1, 1], j)
            got = llk.window_attention(q, k2, v2, **kw)
            o, A, S = expected(q[1, g:2 * g], k2[1, 1], v2[1, 1], Lk, Lq, window, sinks)
            compare(got[1, g:2 * g], o, A, S, D, Lk, dtype)
            assert torch.equal(got[0], clean[0]) and torch.equal(got[1, :g], clean[1, :g]), (name, j)
            assert torch.equal(got[1, 2 * g:], clean[1, 2 * g:]), (name, j)


@pytest.mark.parametrize("Lq,Lk,H", [(1000, 1000, 8), (6, 2000, 4), (1, 2000, 4)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_an_infinity_under_a_small_weight(Lq, Lk, H, dtype):
    """exp(-30) of the largest weight is below f16's least, and above zero: the infinity shows."""
    D, j = 64, Lk // 3
    q, k, v = rand(1, (1, H, Lq, D), dtype), rand(2, (1, 2, Lk, D), dtype), rand(3, (1, 2, Lk, D), dtype)
    q[..., 0], k[..., 0] = 8.0, 0.0
    k[0, 1, j], k[0, 1, j, 0], v[0, 1, j, 5] = 0.0, -30.0, math.inf
    got = llk.window_attention(q, k, v)
    o, A, S = expected(q[0, H // 2:], k[0, 1], v[0, 1], Lk, Lq, 0, 0)
    assert torch.isinf(o).any()
    compare(got[0, H // 2:], o, A, S, D, Lk, dtype)


def timed(f):
    f()
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    best = math.inf
    for _ in range(3):
        a.record()
        f()
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b))
    return best


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (F16, 64), (F32, 64)])
def test_one_nan_does_not_make_a_prompt_slow(dtype, D):
    """A NaN that every query of a head group sees: their results are NaN, no row is computed a second time.  (Row by
    row these calls would take hundreds of times as long.)"""
    L, H = 8192 if dtype != F32 else 4096, 8
    q, k, v = rand(1, (1, H, L, D), dtype), rand(2, (1, 2, L, D), dtype), rand(3, (1, 2, L, D), dtype)
    clean = llk.window_attention(q, k, v)
    plain = timed(lambda: llk.window_attention(q, k, v))
    for what in ("value", "token"):
        k2, v2 = k.clone(), v.clone()
        v2[0, 1, 0, 7] = math.nan
        if what == "token":
            k2[0, 1, 0] = math.nan
        got = llk.window_attention(q, k2, v2)
        assert torch.equal(got[:, :H // 2], clean[:, :H // 2])
        seen = got[0, H // 2:]
        assert torch.isnan(seen[..., 7]).all()
        if what == "token":
            assert torch.isnan(seen).all()
        else:
            # (the weights of the first rows are the ones they were: only component 7 differs)
            rest = [d for d in range(D) if d != 7]
            assert torch.equal(seen[..., rest], clean[0, H // 2:][..., rest])
        t = timed(lambda: llk.window_attention(q, k2, v2))
        print(f"{what} {dtype} D {D}: {plain:.3f} ms clean, {t:.3f} ms with one NaN")
        assert t < 5 * plain + 0.2, (what, t, plain)


@pytest.mark.parametrize("B,H,Hkv,Lq,Lk,D,window,sinks", [(1, 8, 2, 700, 700, 64, 0, 0), (1, 8, 2, 600, 600, 128, 9, 2),
                                                          (1, 4, 2, 300, 300, 256, 5, 0), (2, 8, 2, 3, 900, 128, 0, 0),
                                                          (8, 8, 2, 1, 40, 64, 3, 0)])
def test_values_at_the_largest_f16_stay_finite(B, H, Hkv, Lq, Lk, D, window, sinks):
    """A weighted mean of finite values is finite: the weights' rounding does not push it over the type's largest."""
    q, k = rand(1, (B, H, Lq, D), F16), rand(2, (B, Hkv, Lk, D), F16)
    v = torch.full((B, Hkv, Lk, D), 65504.0, dtype=F16, device="cuda")
    v[..., 1::2] *= -1
    lens = torch.full((B,), Lk, dtype=torch.int32, device="cuda")
    got = llk.window_attention(q, k, v, window=window, sinks=sinks, kv_lens=lens)
    assert torch.isfinite(got).all()
    # half a step of the result and of each weight
    assert ((got.double().abs() - 65504).abs() <= 65504 * 2 * ref.HALF_STEP[F16]).all()
    v[0, 0, Lk // 2, 0] = math.inf
    got = llk.window_attention(q, k, v, window=window, sinks=sinks, kv_lens=lens)
    see = ref.visible(Lq, Lk, Lk, Lq, window, sinks)[:, Lk // 2].cuda()
    assert (got[0, :H // Hkv, see, 0] == math.inf).all()
    assert torch.isfinite(got[0, :H // Hkv, ~see]).all() and torch.isfinite(got[0, H // Hkv:]).all()


@pytest.mark.parametrize("dtype,D,window", [(BF16, 128, 0), (F16, 64, 700), (F32, 64, 0)])
def test_values_that_are_nan_from_some_token_on(dtype, D, window):
    """The later half of a head's values all NaN, its keys not: each query has such values in front of it and behind;
    those before the half are finite, and the call takes its usual time but for the tiles at the border."""
    L, H = 8192 if dtype != F32 else 4096, 8
    q, k, v = rand(1, (1, H, L, D), dtype), rand(2, (1, 2, L, D), dtype), rand(3, (1, 2, L, D), dtype)
    kw = dict(window=window, sinks=2)
    clean = llk.window_attention(q, k, v, **kw)
    plain = timed(lambda: llk.window_attention(q, k, v, **kw))
    cut = L // 2 + 37  # inside a tile
    v[0, 1, cut:] = math.nan
    got = llk.window_attention(q, k, v, **kw)
    assert torch.equal(got[:, :H // 2], clean[:, :H // 2])
    assert torch.isnan(got[0, H // 2:, cut:]).all()
    before, want = got[0, H // 2:, :cut], clean[0, H // 2:, :cut]
    assert torch.isfinite(before).all()
    step = ref.HALF_STEP[dtype] if dtype != F32 else 2.0**-18  # (the rows at the border: by another order of sums)
    assert ((before.double() - want.double()).abs() <= 4 * step * clean.abs().amax().double()).all()
    t = timed(lambda: llk.window_attention(q, k, v, **kw))
    v[0, 1] = math.nan
    assert torch.isnan(llk.window_attention(q, k, v, **kw)[0, H // 2:]).all()
    t_all = timed(lambda: llk.window_attention(q, k, v, **kw))
    print(f"{dtype} D {D}: {plain:.3f} ms clean, {t:.3f} ms half NaN, {t_all:.3f} ms all NaN")
    # the border's tiles: some rows of a warp, one after another, over half of the keys
    assert t < 5 * plain + 15.0 and t_all < 5 * plain + 0.4
