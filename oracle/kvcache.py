"""Oracle: the quantised key / value cache and attention over it, in float64 on the CPU (test infrastructure; no counterpart in the
reference, whose decoding cache holds the model's dtype)."""
import math

import torch

GROUP = 32


def held_values(x, bits):
    """x (..., Dh) -> the values the cache holds for it, float64.  Per 32 channels: s = bf16(max|x| * fp32(1 / L)), an fp32 product, c =
    clamp(round-half-even(x / s), -L, L); s below 2^-126 holds zeros; a NaN, an infinity or a magnitude above 2^127 makes the
    group NaN."""
    top = 7 if bits == 4 else 127
    g = x.double().unflatten(-1, (-1, GROUP))
    a = g.abs().amax(-1, keepdim=True)
    broken = ~(a <= 2.0 ** 127)
    s = (torch.where(broken, torch.zeros_like(a), a).float() * torch.tensor(1 / top, dtype=torch.float32)).bfloat16().double()
    s = torch.where(s < 2.0 ** -126, torch.zeros_like(s), s)
    c = torch.round(torch.where(broken, torch.zeros_like(g), g) / torch.where(s == 0, torch.ones_like(s), s)).clamp(-top, top)
    return torch.where(broken, torch.full_like(g, math.nan), c * s).flatten(-2)


def attention(q, k, v, start, counts=None, scale=None):
    """q (B, Hq, T, Dh); k, v (B, H, n, Dh) held values; row (b, t) sees keys 0 .. start[b] + t (t < counts[b]).  -> (out, lse) float64;
    rows that see nothing: 0 and -inf."""
    q, k, v = q.double(), k.double(), v.double()
    B, Hq, T, Dh = q.shape
    scale = 1 / math.sqrt(Dh) if scale is None else scale
    out, lse = torch.zeros_like(q), torch.full((B, Hq, T), -math.inf, dtype=torch.float64)
    for b in range(B):
        for t in range(T if counts is None else min(T, int(counts[b]))):
            n = min(int(start[b]) + t + 1, k.shape[2])
            if n <= 0:
                continue
            for h in range(Hq):
                hk = h // (Hq // k.shape[1])
                s = (k[b, hk, :n] @ q[b, h, t]) * scale
                out[b, h, t] = torch.softmax(s, -1) @ v[b, hk, :n]
                lse[b, h, t] = torch.logsumexp(s, -1)
    return out, lse
