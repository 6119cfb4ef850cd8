"""Serving calls on a stream of their own while torch's current stream is busy:
what a call makes (outputs, the zeros behind q_lens, scratch) is made on the
stream it runs on, so neither overtakes the other."""
import pytest

torch = pytest.importorskip("torch")

import dslcompiler_b200 as llk  # noqa: E402

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
BUSY = 40_000_000  # clocks, some 20 ms


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")


def rand(seed, shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(BF16).cuda()


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def calls():
    """(name, call(stream)) of every entry point that makes its output; split along the keys or not, padded or not."""
    B, H, Hkv, D, L, page = 2, 8, 2, 64, 600, 16
    q1, qp, k, v = rand(1, (B, H, 2, D)), rand(2, (B, H, L, D)), rand(3, (B, Hkv, L, D)), rand(4, (B, Hkv, L, D))
    cache = llk.QuantizedKVCache.empty(B * 40, page, Hkv, D)
    table = torch.arange(B * 40, device="cuda", dtype=torch.int32).reshape(B, 40)
    slots = (torch.arange(B, device="cuda")[:, None] * 640 + torch.arange(L, device="cuda")[None]).contiguous()
    cache.write(k, v, slots)
    kv, few, some = ints([L, 450]), ints([2, 1]), ints([L, 333])
    q32, k32, v32 = q1.float(), k.float(), v.float()
    torch.cuda.synchronize()
    return [
        ("step", lambda s: llk.window_attention(q1, k, v, kv_lens=kv, stream=s)),
        ("step, padded", lambda s: llk.window_attention(q1, k, v, kv_lens=kv, q_lens=few, stream=s)),
        ("prompt", lambda s: llk.window_attention(qp, k, v, window=100, sinks=2, stream=s)),
        ("prompt, padded", lambda s: llk.window_attention(qp, k, v, q_lens=some, kv_lens=some, stream=s)),
        ("f32 step, padded", lambda s: llk.window_attention(q32, k32, v32, q_lens=few, stream=s)),
        ("cache", lambda s: cache.attention(q1, table, kv, stream=s)),
        ("cache, padded", lambda s: cache.attention(q1, table, kv, q_lens=few, stream=s)),
        ("read", lambda s: cache.read(slots, stream=s)[1]),
    ]


@pytest.mark.parametrize("raw", [False, True])
def test_results_stand_when_the_current_stream_is_late(raw):
    """The call's stream is done long before the current one; nothing that the call queued on the current stream may
    touch the result afterwards."""
    side = torch.cuda.Stream()
    s = side.cuda_stream if raw else side
    for name, call in calls():
        want = call(None)
        torch.cuda.synchronize()
        torch.cuda._sleep(BUSY)
        got = call(s)
        side.synchronize()
        with torch.cuda.stream(side):
            early = got.clone()
        side.synchronize()
        torch.cuda.synchronize()
        assert torch.equal(early, want), name
        assert torch.equal(got, want), name


def test_memory_that_the_current_stream_still_reads_is_not_taken():
    """Blocks of the output's size, given back to the allocator while the current stream has yet to read them."""
    side = torch.cuda.Stream()
    for name, call in calls():
        want = call(None)
        torch.cuda.synchronize()
        blocks = [torch.full_like(want, i + 1.0) for i in range(4)]
        copies = [torch.zeros_like(want) for _ in blocks]
        torch.cuda.synchronize()
        torch.cuda._sleep(BUSY)
        for c, b in zip(copies, blocks):
            c.copy_(b)
        del blocks, b
        side_got = call(side)
        torch.cuda.synchronize()
        for i, c in enumerate(copies):
            assert (c == i + 1.0).all(), (name, i)
        assert torch.equal(side_got, want), name


def test_read_into_its_own_memory_on_another_stream():
    B, Hkv, D, L = 1, 2, 64, 300
    cache = llk.QuantizedKVCache.empty(20, 16, Hkv, D)
    slots = torch.arange(L, device="cuda")[None]
    cache.write(rand(1, (B, Hkv, L, D)), rand(2, (B, Hkv, L, D)), slots)
    want = cache.read(slots)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    blocks = [torch.full((2, B, Hkv, L, D), 3.0, dtype=BF16, device="cuda") for _ in range(4)]
    copies = [torch.zeros_like(b) for b in blocks]
    torch.cuda.synchronize()
    torch.cuda._sleep(BUSY)
    for c, b in zip(copies, blocks):
        c.copy_(b)
    del blocks, b
    got = cache.read(slots, stream=side)
    side.synchronize()
    torch.cuda.synchronize()
    assert all((c == 3.0).all() for c in copies)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_a_result_given_back_early_waits_for_the_current_stream():
    """The result's memory belongs to the call's stream; a use on the current stream, queued before the result is
    dropped, still reads it when the next call on that stream wants memory."""
    side = torch.cuda.Stream()
    q, k, v = rand(1, (2, 8, 2, 64)), rand(2, (2, 2, 600, 64)), rand(3, (2, 2, 600, 64))
    want = llk.window_attention(q, k, v)
    torch.cuda.synchronize()
    for _ in range(3):
        got = llk.window_attention(q, k, v, stream=side)
        side.synchronize()
        torch.cuda._sleep(BUSY)
        copy = got.clone()
        del got
        others = [llk.window_attention(-q, k, v, stream=side) for _ in range(3)]
        torch.cuda.synchronize()
        assert torch.equal(copy, want)
        del others


def test_other_operators_results_stand_when_the_current_stream_is_late():
    """llk.rope, llk.attention (whose output starts from zeros), fused_swiglu, matmul, PackedWeights likewise."""
    q, k, v = (rand(s, (1, 4, 96, 64)).float() for s in (1, 2, 3))
    pos = torch.arange(96, device="cuda")
    x, wg, wu = rand(4, (64, 128)), rand(5, (128, 256)), rand(6, (128, 256))
    pw = llk.PackedWeights(wg, wu)
    side = torch.cuda.Stream()
    for name, call in (("attention", lambda s: llk.attention(q, k, v, causal=True, stream=s)),
                       ("rope", lambda s: llk.rope(q, pos, stream=s)),
                       ("swiglu", lambda s: llk.fused_swiglu(x, wg, wu, stream=s)),
                       ("matmul", lambda s: llk.matmul(x, wg, stream=s)),
                       ("packed", lambda s: pw(x, stream=s))):
        want = call(None)
        torch.cuda.synchronize()
        blocks = [torch.full_like(want, i + 1.0) for i in range(4)]
        copies = [torch.zeros_like(want) for _ in blocks]
        torch.cuda.synchronize()
        torch.cuda._sleep(BUSY)
        for c, b in zip(copies, blocks):
            c.copy_(b)
        del blocks, b
        got = call(side)
        with torch.cuda.stream(side):
            early = got.clone()
        torch.cuda.synchronize()
        assert torch.equal(early, want) and torch.equal(got, want), name
        for i, c in enumerate(copies):
            assert (c == i + 1.0).all(), (name, i)


def test_calls_on_a_forked_stream_of_a_captured_graph():
    """stream= names a stream that the capture has forked to: what the call makes belongs to the graph, and replays
    do not need the memory that eager calls take in between."""
    B, H, Hkv, D, L, page = 2, 8, 2, 64, 600, 16
    q, k, v = rand(1, (B, H, 2, D)), rand(3, (B, Hkv, L, D)), rand(4, (B, Hkv, L, D))
    cache = llk.QuantizedKVCache.empty(B * 40, page, Hkv, D)
    table = torch.arange(B * 40, device="cuda", dtype=torch.int32).reshape(B, 40)
    slots = (torch.arange(B, device="cuda")[:, None] * 640 + torch.arange(L, device="cuda")[None]).contiguous()
    kv, few = ints([L, 450]), ints([2, 1])
    cache.write(k, v, slots)

    def run(s):
        return (llk.window_attention(q, k, v, kv_lens=kv, q_lens=few, stream=s),
                cache.attention(q, table, kv, q_lens=few, stream=s), *cache.read(slots, stream=s))

    run(None)
    torch.cuda.synchronize()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        got = run(side)
        main.wait_stream(side)
    for seed in (5, 6):
        q.copy_(rand(seed, q.shape))
        graph.replay()
        want = run(None)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
