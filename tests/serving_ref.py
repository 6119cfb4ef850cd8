"""Plain 64-bit forms of the serving attention operators, and the error that
their kernels may have, from the roundings they make."""
import math

import torch

HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}


def visible(Lq, Lk, n, m, window, sinks):
    """[Lq, Lk]: what the queries of a sequence with n keys and m queries see (rows behind m: nothing)."""
    i = torch.arange(Lq)[:, None]
    j = torch.arange(Lk)[None]
    p = n - m + i
    see = (j <= p) & (j < n) & (i < m)
    if window:
        see = see & ((j > p - window) | (j < sinks))
    return see


def attention(q, k, v, *, window=0, sinks=0, scale=None, q_lens=None, kv_lens=None, slack=None):
    """(o, slack bound A, score bound S) in float64: o [B, H, Lq, D]; A = sum_j w_j a_j with a = |v| (or `slack`
    [B, Hkv, Lk, D]): how much a relative error of the weights may move o; S [B, H, Lq, 1] the largest
    scale * sum_d |q_d k_d|."""
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    B, H, Lq, D = q.shape
    Hkv, Lk = k.shape[1], k.shape[2]
    scale = 1 / math.sqrt(D) if scale is None else scale
    a = v.abs() if slack is None else slack.detach().cpu().double()
    o, A, S = torch.zeros(B, H, Lq, D).double(), torch.zeros(B, H, Lq, D).double(), torch.zeros(B, H, Lq, 1).double()
    for b in range(B):
        n = Lk if kv_lens is None else max(0, min(Lk, int(kv_lens[b])))
        m = Lq if q_lens is None else max(0, min(Lq, int(q_lens[b])))
        see = visible(Lq, Lk, n, m, window, sinks)
        used = see.any(0)
        for h in range(H):
            hk = h // (H // Hkv)
            # what no query sees may hold anything: it is not touched
            kk = torch.where(used[:, None], k[b, hk], 0.0)
            s = scale * (q[b, h] @ kk.T)
            s = torch.where(see, s, -math.inf)
            top = s.amax(-1, keepdim=True) if Lk else torch.zeros(Lq, 1).double()
            w = torch.where(see, torch.exp(s - torch.where(top == -math.inf, 0.0, top)), 0.0)
            l = w.sum(-1, keepdim=True)
            w = w / torch.where(l == 0, 1.0, l)
            for i in range(Lq):
                at = see[i].nonzero()[:, 0]
                o[b, h, i] = w[i, at] @ v[b, hk, at]
                A[b, h, i] = w[i, at] @ a[b, hk, at]
            if Lk:
                S[b, h] = torch.where(see, scale * (q[b, h].abs() @ kk.abs().T), 0.0).amax(-1, keepdim=True)
    return o, A, S


def bound(o, A, S, D, keys, out_dtype, weight_step):
    """How far a kernel's result may be from o: the output's rounding; the weights' (each at most weight_step, in the
    sum of values; the sum of weights is not rounded to fewer bits); f32 sums over D products of a score, whose error
    moves a weight by as much again and its normaliser too; exp2 to 2 ulp; f32 sums over the keys (numerator and
    normaliser)."""
    u32 = 2.0**-24
    score = 2 * (D + 4) * u32 * S
    weights = weight_step + 2 * score + 2 * (4 + keys) * u32
    return HALF_STEP[out_dtype] * (o.abs() + weights * A) + weights * A + 1e-30


def quantise(x, bits, group):
    """(codes [.., D], scale [.., D / group], min) by the cache's definition, in float64."""
    x = x.detach().cpu().double()
    x = torch.where(torch.isnan(x), 0.0, x).clamp(-65504.0, 65504.0)
    g = x.reshape(*x.shape[:-1], -1, group)
    mn = g.amin(-1).to(torch.float32).to(torch.bfloat16).double()
    top = 2**bits - 1
    s = ((g.amax(-1) - mn) / top).clamp_min(2.0**-30).to(torch.float32).to(torch.bfloat16).double()
    codes = torch.round((g - mn[..., None]) / s[..., None]).clamp(0, top)
    return codes.reshape(x.shape), s, mn


def values(codes, s, mn):
    g = codes.reshape(*codes.shape[:-1], s.shape[-1], -1)
    return (s[..., None] * g + mn[..., None]).reshape(codes.shape)


def unpack(codes, bits):
    """Codes [.., D] of packed bytes [.., D * bits / 8]."""
    c = codes.detach().cpu().long()
    return c if bits == 8 else torch.stack([c & 15, c >> 4], -1).reshape(*c.shape[:-1], -1)
