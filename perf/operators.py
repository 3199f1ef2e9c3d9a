"""Operators around a generator's rollouts and the update that trains on them: the quantised key/value cache (append, read back),
attention over it, and the clipped policy loss with its gradient.

`own = False`: the operators in their plain form (elementary torch operations); `own = True`: the calls a user of branchgan makes.
"""
import math
import os
import sys

import torch

own = False

GROUP = 32                       # channels that share one scale
DEV = "cuda"


# ---------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------
def listed():
    return [
        # one sequence, one token per layer: the cache write of a decode step at its smallest (8 heads of 64)
        dict(name="append_token_1", op="append", B=1, H=8, Dh=64, T=1, S=1023, bits=4, dtype="bfloat16", ragged=False),
        # rollouts of a batch: one token of every sequence, each at a position of its own (16 heads of 64)
        dict(name="append_token_64", op="append", B=64, H=16, Dh=64, T=1, S=1500, bits=4, dtype="bfloat16", ragged=True),
        # prompts of uneven length written at once (8 heads of 256), right-padded
        dict(name="append_prompt", op="append", B=16, H=8, Dh=256, T=2017, S=0, bits=4, dtype="bfloat16", ragged=True),
        # the same in 8 bits from float32 keys (12 heads of 64), continuing sequences that already hold tokens
        dict(name="append_prompt_8bit", op="append", B=8, H=12, Dh=64, T=777, S=246, bits=8, dtype="float32", ragged=True),
        # one sequence decodes one token against a short cache: latency
        dict(name="attend_token_1", op="attend", B=1, Hq=12, Hkv=12, Dh=64, T=1, S=257, bits=4, dtype="bfloat16", ragged=False),
        # a batch of rollouts with uneven lengths decodes one token
        dict(name="attend_token_64", op="attend", B=64, Hq=16, Hkv=16, Dh=64, T=1, S=2047, bits=4, dtype="bfloat16", ragged=True),
        # few long sequences, four query heads to a cache head
        dict(name="attend_long", op="attend", B=8, Hq=32, Hkv=8, Dh=128, T=1, S=65537, bits=4, dtype="bfloat16", ragged=False),
        # 8 bits, float32 queries
        dict(name="attend_8bit", op="attend", B=16, Hq=8, Hkv=8, Dh=256, T=1, S=4001, bits=8, dtype="float32", ragged=True),
        # a chunk of new tokens against a cache (a second prompt, or drafted tokens being checked)
        dict(name="attend_chunk", op="attend", B=4, Hq=16, Hkv=16, Dh=64, T=67, S=1980, bits=4, dtype="bfloat16", ragged=True),
        # a small vocabulary in float32, sampled-token KL estimate
        dict(name="policy_small", op="policy", R=96, V=2048, dtype="float32", kl="sampled", temperature=1.0),
        # one micro-batch of rollouts, odd vocabulary (rows off the 16-byte grid), sampled-token KL estimate, rollouts at a temperature
        dict(name="policy_sampled", op="policy", R=2047, V=50257, dtype="bfloat16", kl="sampled", temperature=0.7),
        # a full batch with the KL over the whole vocabulary against a reference model's logits
        dict(name="policy_full_kl", op="policy", R=8 * 1023, V=50304, dtype="bfloat16", kl="full", temperature=1.0),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "policy"])
    bits, dtype = rng.choice([4, 4, 8]), rng.choice(["bfloat16", "bfloat16", "float32"])
    Dh = rng.choice([32, 64, 128, 256])
    if op == "policy":
        V = _spread(rng, 500, 60000)
        R = _spread(rng, 1, max(1, min(8 * 1023, 400_000_000 // V)))
        return dict(op=op, R=R, V=V, dtype=dtype, kl=rng.choice(["none", "sampled", "full"]), temperature=rng.choice([0.7, 1.0, 1.3]))
    if op == "append":
        H = rng.randint(1, 16)
        T = rng.choice([1, _spread(rng, 2, 2048)])
        B = _spread(rng, 1, max(1, min(64, 60_000_000 // (H * Dh * T))))
        S = rng.choice([0, _spread(rng, 1, 2047)])
        return dict(op=op, B=B, H=H, Dh=Dh, T=T, S=S, bits=bits, dtype=dtype, ragged=rng.random() < 0.7)
    G = rng.choice([1, 1, 2, 4, 8])
    Hkv = rng.randint(1, 16)
    T = rng.choice([1, 1, _spread(rng, 2, 100)])
    S = _spread(rng, 1, 40000 if T == 1 else 3000)
    budget = 400_000_000 if T == 1 else 400_000_000 // (T * G)
    B = _spread(rng, 1, max(1, min(64, budget // (Hkv * Dh * S))))
    return dict(op=op, B=B, Hq=G * Hkv, Hkv=Hkv, Dh=Dh, T=T, S=S, bits=bits, dtype=dtype, ragged=rng.random() < 0.7)


def work(case):
    """Bytes and operations that one pass cannot do without."""
    e = 2 if case.get("dtype") == "bfloat16" else 4
    if case["op"] == "append":                  # keys and values in, codes and scales written and read, keys and values out
        _, counts = _lengths(case)
        n = 2 * sum(counts) * case["H"] * case["Dh"]
        return {"bytes": int(n * (2 * e + 2 * (case["bits"] / 8 + 2 / GROUP))), "flops": 6 * n}
    if case["op"] == "attend":                  # the longest visible prefix of every sequence, queries and outputs
        start, counts = _lengths(case)
        keys = sum(s + c for s, c in zip(start, counts) if c > 0)
        pairs = sum(c * s + c * (c + 1) // 2 for s, c in zip(start, counts))
        cache = 2 * keys * case["Hkv"] * case["Dh"] * (case["bits"] / 8 + 2 / GROUP)
        rows = 2 * sum(counts) * case["Hq"] * case["Dh"] * e
        return {"bytes": int(cache + rows), "flops": 4 * case["Dh"] * case["Hq"] * pairs}
    n = case["R"] * case["V"]                   # logits (and reference logits) in, their gradient out
    return {"bytes": n * e * (3 if case["kl"] == "full" else 2), "flops": n * (16 if case["kl"] == "full" else 8)}


def _lengths(case):
    """Tokens held before the call and new tokens of each sequence; uneven lengths repeat a pattern of sevenths."""
    B, S, T = case["B"], case["S"], case["T"]
    held = S - T if case["op"] == "attend" else S
    if not case["ragged"]:
        return [max(held, 0)] * B, [T] * B
    start = [max(held, 0) * (7 - (5 * b) % 7) // 7 for b in range(B)]
    counts = [T if T == 1 or b % 3 == 0 else T - (b * T) // (2 * B) for b in range(B)]
    return start, counts


# ---------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _keys_values(gen, B, H, n, Dh, dtype):
    """Keys with a few strong channels per head and values, as projections of a trained model give them."""
    gain = torch.exp(0.7 * torch.randn(1, H, 1, Dh, generator=gen, device=DEV))
    k = torch.randn(B, H, n, Dh, generator=gen, device=DEV) * gain
    v = torch.randn(B, H, n, Dh, generator=gen, device=DEV)
    return k.to(dtype), v.to(dtype)


def _framework():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "branch-gan_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    from branchgan import kvcache, losses, ops
    return kvcache, losses, ops


def prepare(case, seed):
    gen, dtype = _generator(seed), getattr(torch, case["dtype"])
    state = dict(case=case)
    if case["op"] == "policy":
        R, V = case["R"], case["V"]
        logits = (2.5 * torch.randn(R, V, generator=gen, device=DEV)).to(dtype)
        u = torch.rand(R, V, generator=gen, device=DEV).clamp_(1e-10, 1 - 1e-7)
        x = logits.float() / case["temperature"]
        ids = (x - torch.log(-torch.log(u))).argmax(-1)                 # sampled from the policy itself
        del u
        logp = torch.log_softmax(x, -1).gather(1, ids[:, None])[:, 0]
        del x
        old = logp + 0.25 * torch.randn(R, generator=gen, device=DEV)   # ratios keep off the clip's ends, where the gradient jumps
        for end in (0.8, 1.28):
            old = torch.where((torch.exp(logp - old) - end).abs() < 1e-3, old + 0.01, old)
        state |= dict(logits=logits, ids=ids, old_logp=old,
                      advantages=torch.randn(R, generator=gen, device=DEV), mask=(torch.arange(R, device=DEV) % 8 < 7).float(),
                      clip=(0.2, 0.28), kl_coef=0.0 if case["kl"] == "none" else 0.05)
        if case["kl"] == "sampled":
            state["ref_logp"] = logp + 0.3 * torch.randn(R, generator=gen, device=DEV)
        if case["kl"] == "full":
            state["ref_logits"] = (logits.float() + 0.3 * torch.randn(R, V, generator=gen, device=DEV)).to(dtype)
        if own:
            state["logits"].requires_grad_(True)
        return state

    start, counts = _lengths(case)
    state["start"] = torch.tensor(start, dtype=torch.int32, device=DEV)
    state["counts"] = torch.tensor(counts, dtype=torch.int32, device=DEV) if case["ragged"] else None
    B, Dh, T = case["B"], case["Dh"], case["T"]
    capacity = max(s + T for s in start)
    if case["op"] == "append":
        state["k"], state["v"] = _keys_values(gen, B, case["H"], T, Dh, dtype)
        if own:
            kvcache, _, _ = _framework()
            state["cache"] = kvcache.QuantizedKVCache(1, B, case["H"], capacity, Dh, bits=case["bits"], device=DEV)
        return state
    keys = max(s + c for s, c in zip(start, counts))
    k, v = _keys_values(gen, B, case["Hkv"], keys, Dh, dtype)
    state["q"] = torch.randn(B, case["Hq"], T, Dh, generator=gen, device=DEV).to(dtype)
    state["max_keys"] = keys
    if own:
        kvcache, _, ops = _framework()
        state["cache"] = kvcache.QuantizedKVCache(1, B, case["Hkv"], capacity, Dh, bits=case["bits"], device=DEV)
        ops.kv_cache_append(state["cache"].layer(0), k, v)
    else:
        state["k"], state["v"] = _pack(*_codes(k, case["bits"]), case["bits"]), _pack(*_codes(v, case["bits"]), case["bits"])
    return state


# ---------------------------------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------------------------------
def _codes(x, bits):
    """Codes in [-L, L] and one bf16 scale per 32 channels.  The quotient is taken in 64 bits: codes sit next to borders."""
    top = 7 if bits == 4 else 127
    g = x.float().unflatten(-1, (-1, GROUP))
    scale = (g.abs().amax(-1, keepdim=True) / top).to(torch.bfloat16)
    s = scale.double()
    code = torch.where(s > 0, torch.round(g.double() / s).clamp(-top, top), torch.zeros((), dtype=torch.float64, device=x.device))
    return code.to(torch.int8), scale


def _pack(code, scale, bits):
    """Two 4-bit codes to a byte; 8-bit codes as they are."""
    if bits == 4:
        u = (code + 8).to(torch.uint8)
        code = u[..., 0::2] | (u[..., 1::2] << 4)
    return code, scale


def _values(code, scale, bits):
    """The values that codes stand for, in 32 bits (exact)."""
    if bits == 4:
        code = torch.stack((code & 15, code >> 4), -1).flatten(-2).float() - 8
    return (code.float() * scale.float()).flatten(-2)


def _append_plain(state):
    """The values that the new rows are held as; rows behind a sequence's last one are not written and read as zero."""
    case = state["case"]
    out = []
    for x in (state["k"], state["v"]):
        y = _values(*_pack(*_codes(x, case["bits"]), case["bits"]), case["bits"])
        if state["counts"] is not None:
            keep = torch.arange(case["T"], device=DEV) < state["counts"][:, None]
            y = torch.where(keep[:, None, :, None], y, torch.zeros((), device=DEV))
        out.append(y.to(x.dtype))
    return out


def _attend_plain(state):
    case, q = state["case"], state["q"]
    B, Hq, T, Dh = q.shape
    k, v = _values(*state["k"], case["bits"]), _values(*state["v"], case["bits"])
    Hkv, n = k.shape[1], k.shape[2]
    rows = q.float().reshape(B, Hkv, -1, Dh)                               # (group, token) rows that read one cache head
    s = torch.matmul(rows, k.transpose(-1, -2)) * (1.0 / math.sqrt(Dh))
    s = s.view(B, Hkv, Hq // Hkv, T, n)
    t = torch.arange(T, device=DEV)
    seen = state["start"][:, None] + t + 1                                 # (B, T) keys that each new token sees
    if state["counts"] is not None:
        seen = torch.where(t < state["counts"][:, None], seen, torch.zeros_like(seen))
    visible = (torch.arange(n, device=DEV) < seen[..., None])[:, None, None]
    s = torch.where(visible, s, torch.full((), -math.inf, device=DEV))
    m = s.amax(-1, keepdim=True)
    p = torch.where(visible, torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m)), torch.zeros((), device=DEV))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    out = torch.matmul(p.reshape(B, Hkv, -1, n), v)
    return out.view(B, Hq, T, Dh).to(q.dtype)


def _log_normaliser(x):
    """log sum exp of each row: exponentials in 32 bits, their sum and its logarithm in 64 (KL terms are small differences of these)."""
    m = x.amax(-1)
    return m.double() + torch.log(torch.exp(x - m[:, None]).sum(-1, dtype=torch.float64))


def _policy_plain(state):
    case, w, adv, beta = state["case"], state["mask"], state["advantages"], state["kl_coef"]
    temp = case["temperature"]
    logits, ids = state["logits"].float(), state["ids"][:, None]
    x = logits / temp
    lse = _log_normaliser(x)
    p = torch.exp(x - lse.float()[:, None])
    logp64 = logits.gather(1, ids)[:, 0].double() / temp - lse
    logp = logp64.float()
    ratio = torch.exp(logp64 - state["old_logp"]).float()
    lo, hi = 1 - state["clip"][0], 1 + state["clip"][1]
    plain, clipped = -adv * ratio, -adv * ratio.clamp(lo, hi)
    d_logp = torch.where(plain >= clipped, plain, torch.zeros_like(plain))
    kl, gap = torch.zeros_like(logp), None
    if case["kl"] == "sampled":
        d = state["ref_logp"] - logp64
        kl = (torch.exp(d) - d - 1).float()
        d_logp = d_logp + beta * (1 - torch.exp(d)).float()
    if case["kl"] == "full":
        ref = state["ref_logits"].float()
        gap = (logits - ref) / temp - (lse - _log_normaliser(ref / temp)).float()[:, None]      # logp - log of the reference
        kl = (p * gap).sum(-1)
    total = w.sum()
    loss = ((w * (torch.maximum(plain, clipped) + beta * kl)).sum(dtype=torch.float64) / total).float()
    grad = -d_logp[:, None] * p
    if gap is not None:
        grad = grad + beta * p * (gap - kl[:, None])
    grad.scatter_add_(1, ids, d_logp[:, None])
    grad = grad * (w / (total * temp))[:, None]
    return loss, grad.to(state["logits"].dtype), logp * w, kl * w


def run(state):
    case = state["case"]
    if not own:
        return {"append": _append_plain, "attend": _attend_plain, "policy": _policy_plain}[case["op"]](state)
    _, losses, ops = _framework()
    if case["op"] == "append":
        layer = state["cache"].layer(0)
        ops.kv_cache_append(layer, state["k"], state["v"], start=state["start"], counts=state["counts"])
        return list(ops.kv_cache_read(layer, case["T"], start=state["start"], counts=state["counts"], dtype=state["k"].dtype))
    if case["op"] == "attend":
        return ops.kv_cache_attention(state["q"], state["cache"].layer(0), start=state["start"], counts=state["counts"], max_keys=state["max_keys"])[0]
    loss, logp, kl = losses.clippedPolicyLoss(state["logits"], state["ids"], state["old_logp"], state["advantages"], mask=state["mask"],
                                              refLogProbs=state.get("ref_logp"), refLogits=state.get("ref_logits"), clipRange=state["clip"],
                                              klWeight=state["kl_coef"], temperature=case["temperature"])
    grad, = torch.autograd.grad(loss, state["logits"])
    return loss.detach(), grad, logp, kl


# ---------------------------------------------------------------------------------------------------
# the operators' definitions in 64 bits
# ---------------------------------------------------------------------------------------------------
def _held(x, bits):
    """Each 32 channels share s = max|x| / L, rounded to 32 bits and from there to bf16; a value is held as s * rint(x / s)."""
    top = float(2 ** (bits - 1) - 1)
    y = x.double().reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    s = (y.abs().max(-1, keepdim=True).values / top).to(torch.float32).to(torch.bfloat16).to(torch.float64)
    safe = torch.where(s == 0, 1.0, s)
    return (torch.clip((y / safe).round(), -top, top) * s).reshape(x.shape)


def exact(case, seed):
    gen, dtype = _generator(seed), getattr(torch, case["dtype"])
    if case["op"] == "policy":
        st = prepare(case, seed)
        temp, ids, w = case["temperature"], st["ids"], st["mask"].double()
        lp = torch.log_softmax(st["logits"].detach().double() / temp, -1)
        tok = lp[torch.arange(case["R"], device=DEV), ids]
        r, adv = (tok - st["old_logp"].double()).exp(), st["advantages"].double()
        lo, hi = 1 - st["clip"][0], 1 + st["clip"][1]
        objective = torch.minimum(r * adv, torch.clip(r, lo, hi) * adv)
        moves = torch.where(adv >= 0, r <= hi, r >= lo)
        slope = -(r * adv) * moves
        beta, kl = st["kl_coef"], torch.zeros_like(tok)
        p = lp.exp()
        grad = torch.zeros_like(lp)
        if case["kl"] == "sampled":
            e = (st["ref_logp"].double() - tok)
            kl = torch.expm1(e) - e
            slope = slope - beta * torch.expm1(e)
        if case["kl"] == "full":
            gap = lp - torch.log_softmax(st["ref_logits"].double() / temp, -1)
            kl = (p * gap).sum(-1)
            grad = beta * p * (gap - kl[:, None])
            del gap
        grad -= slope[:, None] * p
        grad[torch.arange(case["R"], device=DEV), ids] += slope
        grad *= (w / w.sum() / temp)[:, None]
        return ((beta * kl - objective) * w).sum() / w.sum(), grad, tok * w, kl * w

    start, counts = _lengths(case)
    B, Dh, T = case["B"], case["Dh"], case["T"]
    if case["op"] == "append":
        k, v = _keys_values(gen, B, case["H"], T, Dh, dtype)
        k, v = _held(k, case["bits"]), _held(v, case["bits"])
        for b, c in enumerate(counts):
            k[b, :, c:], v[b, :, c:] = 0, 0
        return [k, v]
    keys = max(s + c for s, c in zip(start, counts))
    k, v = _keys_values(gen, B, case["Hkv"], keys, Dh, dtype)
    q = torch.randn(B, case["Hq"], T, Dh, generator=gen, device=DEV).to(dtype).double()
    G = case["Hq"] // case["Hkv"]
    out = torch.zeros(B, case["Hq"], T, Dh, dtype=torch.float64, device=DEV)
    for b in range(B):                                                     # one sequence at a time, its visible keys only
        n, c = start[b] + counts[b], counts[b]
        kb = _held(k[b, :, :n], case["bits"]).repeat_interleave(G, 0)
        vb = _held(v[b, :, :n], case["bits"]).repeat_interleave(G, 0)
        s = (q[b, :, :c] @ kb.transpose(1, 2)) / Dh ** 0.5
        last = torch.arange(start[b], n, device=DEV)
        s.masked_fill_(torch.arange(n, device=DEV) > last[:, None], -math.inf)
        out[b, :, :c] = torch.softmax(s, -1) @ vb
    return out
