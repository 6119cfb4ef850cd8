"""Serving attention where offsets pass 32 bits, and from two host threads at
once.  Tolerances are serving_ref.bound's."""
import threading

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


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("Lq", [1, 3, 150, 300])
def test_window_attention_far_apart(dtype, Lq):
    """Sequences, heads and tokens each up to 2^31 elements and more from one another (one 13 GB buffer)."""
    size = (3 << 30) + (1 << 20)
    if torch.cuda.mem_get_info()[0] < 3 * size * 4:
        pytest.skip("not enough memory")
    base = torch.empty(size, dtype=dtype, device="cuda")
    B, H, Lk, D = 2, 2, 300, 64
    for strides in ((1 << 31, 1 << 30, 64, 1), (1 << 16, 1 << 30, 2112, 1), (64, 128, 1 << 23, 1)):
        reach = sum(s * (n - 1) for s, n in zip(strides, (B, H, Lk, D))) + 1
        assert reach <= size
        k = base.as_strided((B, H, Lk, D), strides)
        k.copy_(rand(1, (B, H, Lk, D), dtype))
        q, v = rand(2, (B, H, Lq, D), dtype), rand(3, (B, H, Lk, D), dtype)
        o, A, S = ref.attention(q, k, v, window=100, sinks=2)
        tol = ref.bound(o, A, S, D, Lk, dtype, 0.0 if dtype == F32 else ref.HALF_STEP[dtype])
        assert ((llk.window_attention(q, k, v, window=100, sinks=2).cpu().double() - o).abs() <= tol).all()
        # the same places as values
        o, A, S = ref.attention(q, v, k, window=100, sinks=2)
        tol = ref.bound(o, A, S, D, Lk, dtype, 0.0 if dtype == F32 else ref.HALF_STEP[dtype])
        assert ((llk.window_attention(q, v, k, window=100, sinks=2).cpu().double() - o).abs() <= tol).all()
        # and as queries and output, where they are as many
        out = base.as_strided((B, H, Lk, D), strides, 0)
        if strides[0] == 1 << 16:  # sequences woven into one another's tokens: no output's layout
            with pytest.raises(llk.LLKError, match="stride"):
                llk.window_attention(v, k, v, out=out)
        elif Lq == Lk:
            o, A, S = ref.attention(q, v, v, window=100)
            llk.window_attention(q, v, v, window=100, out=out)
            tol = ref.bound(o, A, S, D, Lk, dtype, 0.0 if dtype == F32 else ref.HALF_STEP[dtype])
            assert ((out.cpu().double() - o).abs() <= tol).all()
            assert torch.equal(llk.window_attention(k, v, v), llk.window_attention(k.contiguous(), v, v))


@pytest.mark.parametrize("bits", [4, 8])
def test_cache_far_pages(bits):
    """A pool whose codes pass 2^32 bytes: pages at both ends and around the middle."""
    Hkv, D, page, L = 2, 128, 64, 400
    per_page = Hkv * page * D * bits // 8
    pages = (1 << 32) // per_page + 1000
    if torch.cuda.mem_get_info()[0] < 4 * pages * per_page:
        pytest.skip("not enough memory")
    cache = llk.QuantizedKVCache.empty(pages, page, Hkv, D, bits=bits, group_size=64)
    mid = (1 << 31) // per_page
    table = ints([[0, pages - 1, mid, mid - 1, (1 << 32) // per_page, 7, mid + 1],
                  [pages - 2, 1, (1 << 32) // per_page - 1, 3, pages - 900, mid + 2, 5]])
    t = torch.arange(L, device="cuda")
    slots = (table.long()[:, t // page] * page + t % page).contiguous()
    k, v = rand(1, (2, Hkv, L, D), F32), rand(2, (2, Hkv, L, D), F32)
    cache.write(k, v, slots)
    gk, gv = cache.read(slots, dtype=F32)
    for x, got in ((k, gk), (v, gv)):
        assert torch.equal(got.cpu(), ref.values(*ref.quantise(x, bits, 64)).float())
    c, s, m = ref.quantise(v, bits, 64)
    slack = ref.values(c, s, torch.zeros_like(m)) + ref.values(torch.zeros_like(c), s, m.abs())
    for g, Lq in ((4, 1), (1, 3)):
        q = rand(3, (2, g * Hkv, Lq, D), BF16)
        out = cache.attention(q, table, ints([L, L - 70]), window=150, sinks=70)
        o, A, S = ref.attention(q, gk, gv, window=150, sinks=70, kv_lens=[L, L - 70], slack=slack)
        assert ((out.cpu().double() - o).abs() <= ref.bound(o, A, S, D, L, BF16, 2.0**-11)).all()


def test_two_threads_at_once():
    """Each thread on its own stream, with other sizes than the other: nothing is shared but the library."""
    def work(seed, out):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            B, Hkv, g, L, D = 3 + seed, 2, 4, 900 + 31 * seed, 128
            q = rand(seed, (B, Hkv * g, 1, D), BF16)
            k, v = rand(seed + 10, (B, Hkv, L, D), BF16), rand(seed + 20, (B, Hkv, L, D), BF16)
            p = rand(seed + 30, (B, Hkv * g, L, D), BF16)
            cache = llk.QuantizedKVCache.empty(B * 64, 16, Hkv, D)
            table = torch.arange(B * 64, device="cuda", dtype=torch.int32).reshape(B, 64)
            slots = (torch.arange(B, device="cuda")[:, None] * 1024 + torch.arange(L, device="cuda")[None]).contiguous()
            lens = ints([L] * B)
            rounds = []
            for _ in range(40):
                cache.write(k, v, slots)
                rounds.append((cache.attention(q, table, lens), llk.window_attention(q, k, v),
                               llk.window_attention(p, k, v, window=200, sinks=3), *cache.read(slots)))
            stream.synchronize()
            out.append(rounds)

    alone = []
    for seed in (0, 1):
        work(seed, alone)
    both = [[], []]
    threads = [threading.Thread(target=work, args=(seed, both[seed])) for seed in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for seed in (0, 1):
        assert len(both[seed]) == 1
        for r in both[seed][0] + alone[seed]:
            for x, y in zip(r, alone[seed][0]):
                assert torch.equal(x, y)
