"""Plain 64-bit statements of the speculative-serving operators, for the tests:
the quantised cache write and its read-back, attention of drafted trees over a
paged cache, and token log probabilities. Everything runs on the CPU."""
import math

import torch

D = 128


def quantise(x):
    """(values float64 as held, exponents int) of bf16 rows [..., 128]: e4m3 times a power of two."""
    x = x.double()
    top = torch.where(torch.isfinite(x), x.abs(), torch.zeros((), dtype=torch.float64)).amax(-1)
    e = torch.zeros(top.shape, dtype=torch.int64)
    flat = top.reshape(-1)
    ef = e.reshape(-1)
    for i, t in enumerate(flat.tolist()):
        if t > 0:
            m, p = math.frexp(t / 448.0)  # t / 448 = m * 2^p, m in [0.5, 1): the smallest 2^e >= it
            ef[i] = max(-100, p if m > 0.5 else p - 1)
    scale = torch.tensor([math.ldexp(1.0, int(v)) for v in ef.tolist()], dtype=torch.float64).reshape(top.shape)
    y = (x / scale.unsqueeze(-1)).clamp(-448, 448)
    mag = y.abs().clamp(min=2.0 ** -6)
    step = torch.ldexp(torch.ones_like(mag), torch.frexp(mag).exponent - 4)  # 3 mantissa bits, subnormals below 2^-6
    return torch.round(y / step) * step, e  # torch.round: half to even


def attention(q, k, v, seen, scale):
    """q [T, Hq, D], k/v [n, Hkv, D], seen bool [T, n] -> [T, Hq, D] float64; nothing seen gives 0, and only
    seen keys take part (values of others are never touched)."""
    T, hq, _ = q.shape
    g = hq // k.shape[1]
    out = torch.zeros(T, hq, D, dtype=torch.float64)
    for t in range(T):
        idx = seen[t].nonzero().view(-1)
        if not idx.numel():
            continue
        for h in range(k.shape[1]):
            s = q[t, h * g:(h + 1) * g].double() @ k[idx, h].double().T * scale
            out[t, h * g:(h + 1) * g] = torch.softmax(s, -1) @ v[idx, h].double()
    return out


def mask_bits(mask, nodes):
    """bool [T, nodes] of int32 mask words [T, words]."""
    j = torch.arange(nodes)
    return (mask.long()[:, j // 32] >> (j % 32)) & 1 == 1


def logprobs(x, tokens, top):
    x = x.double()
    rows, vocab = x.shape
    m = x.amax(1, keepdim=True)
    empty = (m == -math.inf).view(-1)
    z = x - torch.where(m == -math.inf, torch.zeros_like(m), m)
    S = torch.exp(z).sum(1, keepdim=True)
    lp = z - torch.log(S)
    lp = torch.where(x == -math.inf, torch.where(torch.isnan(S), S, torch.full_like(lp, -math.inf)), lp)
    p = torch.exp(lp)
    ent = -torch.where(p == 0, torch.zeros_like(p), p * lp).sum(1)
    ent = torch.where(empty, torch.zeros_like(ent), ent)
    lp = torch.where(empty[:, None], torch.full_like(lp, -math.inf), lp)
    order = torch.sort(torch.where(torch.isnan(x), torch.full_like(x, math.inf), x) if not torch.isinf(x).any()
                       else x, dim=1, descending=True, stable=True).indices
    has = (tokens >= 0) & (tokens < vocab)
    tk = tokens.clamp(0, vocab - 1)
    rank = (order == tk[:, None]).int().argmax(1)
    return (torch.where(has, lp.gather(1, tk[:, None]).view(-1), torch.zeros(rows, dtype=torch.float64)),
            torch.where(has, rank, torch.full_like(rank, -1)), ent, order[:, :top], lp.gather(1, order[:, :top]))
