"""Cases of the attention operators that serve a model: attention under a sliding window with sinks, a
KV cache that is quantised as it is written and read back, and attention over that cache.

Layout: q, o [B, H, Lq, D]; k, v [B, Hkv, Lk, D]; a paged pool of codes uint8 [pages, Hkv, page, D * bits / 8]
(4 bits: element 2j in the low nibble of byte j, 2j + 1 in the high one) and of (scale, min) pairs bf16
[pages, Hkv, page, D / group, 2]: an element stands for scale * code + min.
"""
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
LARGEST = 65504.0  # values are held up to this magnitude
LEAST_SCALE = 2.0**-30


def listed():
    return [
        # a prompt of the attention shape the repository benches (32 heads of 128), every head its own keys
        dict(name="window prompt 32x128", op="window", B=1, H=32, Hkv=32, Lq=4096, Lk=4096, D=128, window=1024, sinks=4,
             dtype="bf16", order="bhld", ragged=0),
        # a long prompt with grouped heads and a wide window
        dict(name="window long grouped", op="window", B=1, H=32, Hkv=8, Lq=8192, Lk=8192, D=128, window=4096, sinks=4,
             dtype="bf16", order="bhld", ragged=0),
        # a padded batch of short prompts, heads of 64 in token-major order, odd lengths, in f16
        dict(name="window padded batch f16", op="window", B=5, H=16, Hkv=4, Lq=1001, Lk=1001, D=64, window=255, sinks=17,
             dtype="f16", order="blhd", ragged=131),
        # a prompt in f32, the type of the repository's rope and attention
        dict(name="window prompt f32", op="window", B=1, H=32, Hkv=32, Lq=1000, Lk=1000, D=128, window=333, sinks=1,
             dtype="f32", order="bhld", ragged=0),
        # one new token for each sequence of a batch over an unquantised cache
        dict(name="window single token", op="window", B=16, H=32, Hkv=8, Lq=1, Lk=8192, D=128, window=4096, sinks=4,
             dtype="bf16", order="bhld", ragged=300),
        # the smallest decode step: one sequence, a few hundred tokens
        dict(name="cache one sequence", op="cache", B=1, H=32, Hkv=8, Lq=1, L=517, D=128, bits=4, group=128, page=16,
             window=0, sinks=0, dtype="bf16", ragged=0),
        # an ordinary decode batch with grouped heads, sequences of uneven length
        dict(name="cache batch 32", op="cache", B=32, H=64, Hkv=8, Lq=1, L=4096, D=128, bits=4, group=64, page=64,
             window=0, sinks=0, dtype="bf16", ragged=100),
        # long context: few sequences, the work is along the length
        dict(name="cache long context", op="cache", B=4, H=64, Hkv=8, Lq=1, L=131072, D=128, bits=4, group=128, page=64,
             window=0, sinks=0, dtype="bf16", ragged=1111),
        # several tokens a step (drafted tokens to verify) in 8 bits under a window, every head its own keys
        dict(name="cache drafted 8 bit", op="cache", B=8, H=32, Hkv=32, Lq=4, L=4001, D=64, bits=8, group=32, page=32,
             window=1024, sinks=4, dtype="f16", ragged=77),
        # a decode step's write and its read-back
        dict(name="store step", op="store", B=32, Hkv=8, L=1, D=128, bits=4, group=128, page=16, dtype="bf16", to="bf16"),
        # prompts written and read back for the next chunk's attention
        dict(name="store prompts", op="store", B=4, Hkv=8, L=8191, D=128, bits=4, group=64, page=64, dtype="bf16",
             to="bf16"),
        # f32 keys straight from rope, heads of 64, 8 bits, read back in f16
        dict(name="store f32 8 bit", op="store", B=2, Hkv=32, L=1000, D=64, bits=8, group=32, page=32, dtype="f32",
             to="f16"),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["window", "window", "cache", "cache", "store"])
    Hkv = rng.choice([1, 2, 4, 8, 8, 32])
    if op == "store":
        D = rng.choice([64, 128, 128, 256])
        L = _spread(rng, 1, 4096)
        return dict(op=op, B=min(64, max(1, _spread(rng, 1, 65536) // (L * Hkv))), Hkv=Hkv, L=L, D=D,
                    bits=rng.choice([4, 4, 8]), group=rng.choice([32, 64, D if D < 256 else 128]),
                    page=rng.choice([16, 32, 64, 128]), dtype=rng.choice(["bf16", "bf16", "f16", "f32"]),
                    to=rng.choice(["bf16", "f16", "f32"]))
    g = rng.choice([1, 1, 4, 8, 5] if Hkv < 32 else [1, 2])
    window = rng.choice([0, _spread(rng, 1, 4096), _spread(rng, 64, 2048)])
    sinks = rng.choice([0, 1, 4, _spread(rng, 1, 200)]) if window else 0
    if op == "cache":
        D = rng.choice([64, 128, 128, 256])
        L = _spread(rng, 1, 65536)
        B = min(64, max(1, _spread(rng, 256, 2**20) // (L * Hkv)))
        return dict(op=op, B=B, H=g * Hkv, Hkv=Hkv, Lq=rng.choice([1, 1, 1, 2, 5]), L=L + 5, D=D, bits=rng.choice([4, 4, 8]),
                    group=rng.choice([32, 64, D if D < 256 else 128]), page=rng.choice([16, 32, 64, 128]), window=window,
                    sinks=sinks, dtype=rng.choice(["bf16", "f16"]), ragged=rng.choice([0, L // (2 * B)]))
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    D = rng.choice([64, 128, 128, 80])
    Lk = _spread(rng, 1, 4096)
    step = dtype != "f32" and rng.random() < 0.4  # a few new tokens after many, else a whole prompt
    Lq = min(Lk, rng.choice([1, 1, 2, 7])) if step else Lk
    B = min(16, max(1, _spread(rng, 256, 2**17) // (Lk * Hkv * g)))
    return dict(op=op, B=B, H=g * Hkv, Hkv=Hkv, Lq=Lq, Lk=Lk, D=D, window=window, sinks=sinks, dtype=dtype,
                order=rng.choice(["bhld", "blhd"]), ragged=rng.choice([0, (Lk - Lq if step else Lk) // (2 * B)]))


def _kv_lens(case):
    """Tokens of each sequence: the first is as long as it can be, each further one `ragged` shorter."""
    top = case["Lk"] if case["op"] == "window" else case["L"]
    return [max(min(top, case["Lq"] if case["Lq"] < top else 1), top - b * case["ragged"]) for b in range(case["B"])]


def _q_lens(case):
    """Queries of each sequence: a padded batch of prompts has as many as it has keys."""
    return _kv_lens(case) if case["op"] == "window" and case["Lq"] == case["Lk"] and case["ragged"] else [case["Lq"]] * case["B"]


def _normal(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _kv(gen, shape, dtype):
    """Keys or values [B, Hkv, L, D]: a few channels of each head are much larger than the others and off zero, as
    the caches of trained models have them."""
    h, d = shape[1], shape[3]
    gain = torch.exp(0.5 * torch.randn((h, 1, d), generator=gen, device="cuda"))
    shift = torch.randn((h, 1, d), generator=gen, device="cuda") * 0.3
    return (_normal(gen, shape, torch.float32) * gain + shift).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    B, Hkv, D = case["B"], case["Hkv"], case["D"]
    dt = TYPES[case["dtype"]]
    state = dict(case=case)
    if case["op"] == "window":
        def laid(t):  # the same tensor with tokens before heads in memory
            return t.transpose(1, 2).contiguous().transpose(1, 2) if case["order"] == "blhd" else t
        state["q"] = laid(_normal(gen, (B, case["H"], case["Lq"], D), dt))
        state["k"] = laid(_kv(gen, (B, Hkv, case["Lk"], D), dt))
        state["v"] = laid(_kv(gen, (B, Hkv, case["Lk"], D), dt))
        state["q_lens"] = state["kv_lens"] = None
        if case["ragged"]:
            state["kv_lens"] = torch.tensor(_kv_lens(case), dtype=torch.int32, device="cuda")
            if _q_lens(case)[-1] != case["Lq"]:
                state["q_lens"] = torch.tensor(_q_lens(case), dtype=torch.int32, device="cuda")
        return state
    page, L = case["page"], case["L"]
    width = -(-L // page)
    pages = B * width + 3
    state["table"] = torch.randperm(pages, generator=gen, device="cuda")[: B * width].reshape(B, width).to(torch.int32)
    t = torch.arange(L, device="cuda")
    slots = state["table"].long()[:, t // page] * page + t % page
    shape = (pages, Hkv, page)
    if case["op"] == "store":
        state["k"], state["v"] = _kv(gen, (B, Hkv, L, D), dt), _kv(gen, (B, Hkv, L, D), dt)
        state["slots"] = slots
        state["pool"] = [torch.zeros(shape + tail, device="cuda", dtype=t) for _ in range(2)
                         for tail, t in (((D * case["bits"] // 8,), torch.uint8), ((D // case["group"], 2), torch.bfloat16))]
        return state
    state["q"] = _normal(gen, (B, case["H"], case["Lq"], D), dt)
    state["lens"] = torch.tensor(_kv_lens(case), dtype=torch.int32, device="cuda")
    state["pool"] = []
    for _ in range(2):  # a pool whose every page holds quantised keys or values
        codes = torch.empty(shape + (D * case["bits"] // 8,), device="cuda", dtype=torch.uint8)
        params = torch.empty(shape + (D // case["group"], 2), device="cuda", dtype=torch.bfloat16)
        step = max(1, 2**25 // (Hkv * page * D))
        for a in range(0, pages, step):
            x = _kv(gen, (min(step, pages - a), Hkv, page, D), dt)
            c, p = _quantise(x, case["bits"], case["group"])
            codes[a : a + step], params[a : a + step] = _pack(c, case["bits"]), p
        state["pool"] += [codes, params]
    return state


def _quantise(x, bits, group):
    """Codes [.., D] and (scale, min) [.., D / group, 2] of x [.., D]; the quotients in 64 bits, for values next to the
    border between two codes."""
    x = torch.nan_to_num(x.double(), nan=0.0, posinf=LARGEST, neginf=-LARGEST).clamp(-LARGEST, LARGEST)
    x = x.unflatten(-1, (-1, group))
    least = x.amin(-1, keepdim=True).float().bfloat16()
    scale = ((x.amax(-1, keepdim=True) - least.double()) / (2**bits - 1)).clamp_min(LEAST_SCALE).float().bfloat16()
    codes = torch.round((x - least.double()) / scale.double()).clamp(0, 2**bits - 1).to(torch.uint8)
    return codes.flatten(-2), torch.cat([scale, least], -1)


def _pack(codes, bits):
    return codes if bits == 8 else codes[..., 0::2] | (codes[..., 1::2] << 4)


def _unpack(codes, bits):
    return codes if bits == 8 else torch.stack([codes & 15, codes >> 4], -1).flatten(-2)


def _values(codes, params, bits):
    """What packed codes and their (scale, min) pairs stand for, in 32 bits."""
    groups = params.shape[-2]
    c = _unpack(codes, bits).float().unflatten(-1, (groups, -1))
    p = params.float()
    return (c * p[..., 0:1] + p[..., 1:2]).flatten(-2)


def _attend(q, k, v, q_lens, kv_lens, window, sinks):
    """Attention of q [B, H, Lq, D] over k, v [B, Hkv, Lk, D] in their type; rows behind q_lens are zero."""
    B, H, Lq, D = q.shape
    Hkv, Lk = k.shape[1], k.shape[2]
    i = torch.arange(Lq, device=q.device)
    j = torch.arange(Lk, device=q.device)
    pos = (kv_lens - q_lens)[:, None] + i  # [B, Lq]
    seen = j <= pos[..., None]
    if window:
        seen = seen & ((j > pos[..., None] - window) | (j < sinks))
    seen = seen & (i < q_lens[:, None])[..., None]  # [B, Lq, Lk]
    v = v * (j < kv_lens[:, None])[:, None, :, None]
    q = q.reshape(B, Hkv, H // Hkv, Lq, D)
    s = (q @ k.unsqueeze(2).transpose(-1, -2)) * (1.0 / math.sqrt(D))
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True).clamp_min(torch.finfo(s.dtype).min)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    return ((p @ v.unsqueeze(2)) / torch.where(total == 0, 1.0, total)).reshape(B, H, Lq, D)


def _lens(case, state):
    one = torch.ones(case["B"], dtype=torch.int64, device="cuda")
    if case["op"] == "window":
        q = one * case["Lq"] if state["q_lens"] is None else state["q_lens"].long()
        return q, one * case["Lk"] if state["kv_lens"] is None else state["kv_lens"].long()
    return one * case["Lq"], state["lens"].long()


def _gathered(pool, table, L, bits):
    """The first L tokens of every sequence [B, Hkv, L, D] out of a pool's codes and params."""
    codes, params = (t[table.long()].transpose(1, 2).flatten(2, 3)[:, :, :L] for t in pool)
    return _values(codes, params, bits)


def _run_own(case, state):
    import dslcompiler_b200 as llk

    if case["op"] == "window":
        return llk.window_attention(state["q"], state["k"], state["v"], window=case["window"], sinks=case["sinks"],
                                    q_lens=state["q_lens"], kv_lens=state["kv_lens"])
    if "cache" not in state:  # the handle on the pool's tensors that a program keeps
        state["cache"] = llk.QuantizedKVCache(*state["pool"], bits=case["bits"])
    cache = state["cache"]
    if case["op"] == "cache":
        return cache.attention(state["q"], state["table"], state["lens"], window=case["window"], sinks=case["sinks"])
    cache.write(state["k"], state["v"], state["slots"])
    return cache.read(state["slots"], dtype=TYPES[case["to"]])


def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    if case["op"] == "window":
        q_lens, kv_lens = _lens(case, state)
        o = _attend(state["q"].float(), state["k"].float(), state["v"].float(), q_lens, kv_lens, case["window"],
                    case["sinks"])
        return o.to(state["q"].dtype)
    if case["op"] == "cache":
        q_lens, kv_lens = _lens(case, state)
        k = _gathered(state["pool"][:2], state["table"], case["L"], case["bits"])
        v = _gathered(state["pool"][2:], state["table"], case["L"], case["bits"])
        o = _attend(state["q"].float(), k, v, q_lens, kv_lens, case["window"], case["sinks"])
        return o.to(state["q"].dtype)
    page, at = state["slots"] // case["page"], state["slots"] % case["page"]
    to = TYPES[case["to"]]

    def stored(x, codes, params):
        c, p = _quantise(x, case["bits"], case["group"])
        codes[page, :, at] = _pack(c, case["bits"]).transpose(1, 2)
        params[page, :, at] = p.transpose(1, 2)
        return _values(codes[page, :, at], params[page, :, at], case["bits"]).transpose(1, 2).to(to)

    return stored(state["k"], *state["pool"][:2]), stored(state["v"], *state["pool"][2:])


def exact(case, seed):
    """The operators' definitions in 64 bits, row by row of the batch and its key heads."""
    state = prepare(case, seed)
    B, Hkv, D = case["B"], case["Hkv"], case["D"]
    if case["op"] == "store":
        return tuple(_held(state[n], case["bits"], case["group"]) for n in "kv")
    H, Lq, g = case["H"], case["Lq"], case["H"] // Hkv
    kv_lens, q_lens = _kv_lens(case), _q_lens(case)
    out = torch.zeros((B, H, Lq, D), dtype=torch.float64, device="cuda")
    for b in range(B):
        n, m = kv_lens[b], q_lens[b]
        for h in range(Hkv):
            if case["op"] == "window":
                k, v = state["k"][b, h, :n].double(), state["v"][b, h, :n].double()
            else:
                k, v = (_tokens(state["pool"][2 * t], state["pool"][2 * t + 1], state["table"][b], h, n, case) for t in (0, 1))
            for a in range(0, m, 1024):  # queries a .. e of the sequence, at positions n - m + a ..
                e = min(m, a + 1024)
                pos = torch.arange(n - m + a, n - m + e, device="cuda").repeat(g)[:, None]
                j = torch.arange(n, device="cuda")[None]
                hidden = j > pos
                if case["window"]:
                    hidden |= (pos - j >= case["window"]) & (j >= case["sinks"])
                q = state["q"][b, h * g : (h + 1) * g, a:e].double().reshape(-1, D)
                w = torch.einsum("id,jd->ij", q, k) / D**0.5
                w[hidden] = -math.inf
                w = torch.softmax(w, -1)
                out[b, h * g : (h + 1) * g, a:e] = torch.einsum("ij,jd->id", w, v).reshape(g, e - a, D)
    return out


def _tokens(codes, params, pages, head, n, case):
    """Values of the first n tokens of one sequence and head, in 64 bits."""
    pages = pages[: -(-n // case["page"])].long()
    c = codes[pages, head].reshape(-1, codes.shape[-1])[:n].double()
    sm = params[pages, head].reshape(-1, params.shape[-2], 2)[:n].double().repeat_interleave(case["group"], 1)
    if case["bits"] == 4:
        high = torch.floor(c / 16)
        c = torch.stack([c - 16 * high, high], 2).reshape(n, -1)
    return sm[..., 0] * c + sm[..., 1]


def _held(x, bits, group):
    """What x [B, Hkv, L, D] reads back as: each group of a row on the grid min + scale * (0 .. 2^bits - 1)."""
    B, H, L, D = x.shape
    x = x.double().reshape(B, H, L, D // group, group)
    lo = x.min(-1).values.to(torch.float32).to(torch.bfloat16).double()
    span = x.max(-1).values - lo
    s = torch.maximum(span / (2**bits - 1), torch.full_like(span, LEAST_SCALE)).to(torch.float32).to(torch.bfloat16).double()
    n = torch.round((x - lo[..., None]) / s[..., None])
    return (lo[..., None] + s[..., None] * torch.minimum(torch.maximum(n, torch.zeros_like(n)), torch.full_like(n, 2**bits - 1))).reshape(B, H, L, D)


def work(case):
    el = torch.finfo(TYPES[case["dtype"]]).bits // 8
    Hkv, D = case["Hkv"], case["D"]
    if case["op"] == "store":
        T = case["B"] * case["L"]
        held = D * case["bits"] // 8 + D // case["group"] * 4
        to = torch.finfo(TYPES[case["to"]]).bits // 8
        return {"bytes": 2 * T * Hkv * (D * el + 2 * held + D * to) + 2 * 8 * T, "flops": 2 * T * Hkv * D * 6}
    pairs = rows = queries = 0
    for n, m in zip(_kv_lens(case), _q_lens(case)):
        first = n - m
        w, s = case["window"] or n, min(case["sinks"], n)
        for p in range(max(first, 0), n):  # query at position p sees its window and the sinks before it
            pairs += min(w, p + 1) + min(s, max(0, p + 1 - w))
        start = max(0, max(first, 0) - w + 1)
        rows += n - start + min(s, start)
        queries += m
    token = D * el if case["op"] == "window" else D * case["bits"] // 8 + D // case["group"] * 4
    extra = 4 * case["B"] * (1 if case["op"] == "window" else 1 + -(-case["L"] // case["page"]))
    return {"bytes": 2 * rows * Hkv * token + 2 * queries * case["H"] * D * el + extra, "flops": 4 * D * case["H"] * pairs}
