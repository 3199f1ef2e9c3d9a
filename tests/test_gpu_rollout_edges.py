"""The quantised cache, the attention over it and the clipped policy loss where sums, scales and masks reach their ends; against float64."""
import math

import pytest
import torch

from oracle import kvcache as OK

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("Dh,B,H,G,T", [(32, 32, 16, 1, 1), (64, 32, 16, 1, 1), (128, 16, 16, 2, 1), (32, 16, 16, 16, 2), (128, 16, 16, 4, 8), (32, 1, 2, 1, 3)])
def test_sums_over_many_keys_do_not_lose_digits(Dh, B, H, G, T):
    """4 bits, bf16 queries, 65536 keys, key ranges with and without splits.  Keys of zero give every key the probability 1, scales of
    values are 8-bit numbers in [1, 2), and the values of a turn of 128 keys add up to at most 2 (its halves cancel).  Whatever the
    sums are kept in, a multiple of 2^-7 below 2^17 is exact in fp32: the values of one turn with codes offset by up to 24 reach 128 * 31 *
    2 < 2^13, all turns together without an offset 512 * 2 = 2^10 - so the output is the exact sum over the exact count, divided (2^-22) and
    rounded to bf16 (half a step).  Sums that carry an offset from turn to turn reach 65536 / 4 * 31 * 1.5 > 2^19 and do not pass."""
    from branchgan import kvcache, ops
    gen = torch.Generator().manual_seed(Dh + G)
    n = 65536
    s = (1 + torch.randint(0, 128, (n // 128, 1, 64, Dh // 32), generator=gen) / 128).double().expand(-1, 2, -1, -1).reshape(n, Dh // 32)
    c = torch.randint(-6, 7, (n // 128, 64, Dh), generator=gen).double()
    c[..., ::32] = 7.0                                                       # the largest magnitude of its 32 channels: fixes the scale
    c = torch.stack((c, -c), 1)
    c[:, 1, 0, 1:31] += 1                                                    # a turn leaves one s behind, in most channels
    c = c.view(n, Dh)
    v = c * s.repeat_interleave(32, 1)
    assert torch.equal(v, v.float().double()) and torch.equal(v, OK.held_values(v.float(), 4))
    turns = v.view(-1, 128, Dh)
    assert turns.sum(1).abs().max() < 2 and turns.cumsum(1).abs().max() < 2.0 ** 13
    layer = kvcache.QuantizedKVCache(1, B, H, n, Dh).layer(0)
    ops.kv_cache_append(layer, torch.zeros(1, 1, n, Dh, device="cuda").expand(B, H, n, Dh), v.float().cuda().view(1, 1, n, Dh).expand(B, H, n, Dh))
    q = torch.randn(B, H * G, T, Dh, generator=gen).bfloat16().cuda()
    start = torch.full((B,), n - T, dtype=torch.int32, device="cuda")
    out, lse = ops.kv_cache_attention(q, layer, start=start)
    seen = torch.arange(n - T, n) + 1
    want = (v.cumsum(0)[seen - 1] / seen[:, None]).cuda()
    err = (out.double() - want).abs()
    assert bool((err <= (2.0 ** -8 + 2.0 ** -22) * want.abs()).all()), float((err - 2.0 ** -8 * want.abs()).max() / want.abs().max())
    assert float((lse.double() - torch.log(seen.double()).cuda()).abs().max()) < 2.0 ** -19


def test_saved_tensors_that_come_back_in_a_layout_of_their_own_each_time():
    """Hooks that answer dense, as saved, dense again: the same gradient from every backward."""
    from branchgan import ops
    gen = torch.Generator().manual_seed(85)
    B, T, V = 3, 4, 1031
    full, ref = [torch.randn(B, 9, V, generator=gen).bfloat16().cuda() for _ in range(2)]
    rows = [torch.randint(0, V, (B, T), generator=gen).cuda(), torch.randn(B, T, generator=gen).cuda() - 7, torch.randn(B, T, generator=gen).cuda()]
    x, dense = full.requires_grad_(True), [False]
    unpack = lambda t: t.contiguous().clone() if dense[0] and t.dim() == 3 else t
    def loss():
        return ops.policy_loss(x[:, 2:6], *rows, ref_logits=ref[:, 2:6], kl_coef=0.1)[0]
    plain = loss()
    torch.autograd.grad(plain, x, retain_graph=True)
    want, = torch.autograd.grad(plain, x)                                    # a second backward reads the logits again, as the ones below do
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        hooked = loss()
    torch.autograd.grad(hooked, x, retain_graph=True)
    for dense[0] in (True, False, True):
        assert torch.equal(torch.autograd.grad(hooked, x, retain_graph=True)[0], want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [40, 5003, 120001])
@pytest.mark.parametrize("g", [1.0, 0.5])
@pytest.mark.parametrize("ref", ["masked", "nan", "logp"])
def test_a_kl_that_is_reported_only_stays_out_of_the_update(dtype, V, g, ref):
    """kl_coef 0 with a reference that masks an entry the policy gives weight (an infinite KL), a broken one, or a reference log-prob far
    above the policy's: loss and gradient are those without a reference, to rounding."""
    from branchgan import ops
    gen = torch.Generator().manual_seed(V)
    rows = 5
    x = torch.randn(rows, V, generator=gen).to(dtype)
    ids = torch.randint(2, V, (rows,), generator=gen)
    logp = torch.log_softmax(x.double(), -1).gather(1, ids[:, None])[:, 0]
    old, adv = (logp + torch.tensor([0.1, -0.1, 0.05, 0.5, -0.5])).float(), torch.tensor([1.0, -2.0, 0.5, 1.0, 1.0])
    kw = dict(ref_logp=torch.full((rows,), 150.0, device="cuda"))
    if ref != "logp":
        y = x.clone()
        y[:4, 1] = -math.inf if ref == "masked" else math.nan
        y[4, 0] = -math.inf if ref == "masked" else math.nan
        kw = dict(ref_logits=y.cuda())
    xd = x.double().requires_grad_(True)
    ratio = torch.exp(torch.log_softmax(xd, -1).gather(1, ids[:, None])[:, 0] - old.double())
    want = torch.maximum(-adv.double() * ratio, -adv.double() * ratio.clamp(0.8, 1.2)).mean()
    (want * g).backward()
    leaf = x.cuda().requires_grad_(True)
    loss, got_logp, kl = ops.policy_loss(leaf, ids.cuda(), old.cuda(), adv.cuda(), **kw)
    (loss * g).backward()
    assert bool((kl.isnan() if ref == "nan" else kl == math.inf).all())
    # a p and a log-prob are off by dl at most (34 roundings of an argument below 30, V / 256 + 16 of a sum), a row's term by |A| ratio times
    # twice that, its gradient by four times, then the rounding of the result
    dl = 34 * 2.0 ** -23 + (V / 256 + 16) * 2.0 ** -24
    size = (adv.abs() * ratio.detach())
    assert abs(float(loss.detach()) - float(want.detach())) <= float(size.mean()) * 2 * dl + 2.0 ** -23 * abs(float(want.detach()))
    one = torch.zeros(rows, V, dtype=torch.float64).scatter_(1, ids[:, None], 1.0)
    tol = 4 * dl * size[:, None] / rows * (one + torch.softmax(xd.detach(), -1)) + torch.finfo(dtype).eps / 2 * (1 + 1e-5) * xd.grad.abs() + 1e-38
    assert bool(((leaf.grad.cpu().double() - xd.grad).abs() <= tol).all())


@pytest.mark.parametrize("pad_is_eos", [False, True])
def test_what_fills_up_a_finished_sequence_does_not_train(pad_is_eos):
    """Rollouts with an end of sequence, masked by liveTokens: the padding behind it has no gradient and no part in the loss's mean."""
    from branchgan import configs, generate, losses, models
    torch.manual_seed(9)
    lm = models.make_lm(configs.LMConfig("gpt_neox", 19, 64, 2, 2, 64)).cuda()
    B, P, new, eos = 8, 5, 30, 3
    prompt = torch.randint(0, 19, (B, P), device="cuda")
    seq, old = generate.generate(lm, prompt, max_new_tokens=new, do_sample=True, cache_bits=4, return_logprobs=True, eos_token_id=eos,
                                 pad_token_id=eos if pad_is_eos else 0, generator=torch.Generator(device="cuda").manual_seed(2))
    live = generate.liveTokens(seq[:, P:], eos)
    ends = [row.index(eos) + 1 if eos in row else new for row in seq[:, P:].tolist()]
    assert live.sum(1).tolist() == ends and min(ends) < new and not old[~live].any()
    adv = torch.randn(B, new, generator=torch.Generator().manual_seed(3)).cuda()
    logits = lm(input_ids=seq[:, :-1], returnLmLogits=True).logits
    logits.retain_grad()
    behind = lambda t: torch.nn.functional.pad(t, (P - 1, 0))
    loss, logp, _ = losses.clippedPolicyLoss(logits, seq[:, 1:], behind(old), behind(adv), mask=behind(live.float()))
    loss.backward()
    grad = logits.grad[:, P - 1:]
    assert not grad[~live].any() and not logits.grad[:, :P - 1].any() and not logp[:, P - 1:][~live].any() and bool((grad[live].abs().amax(-1) > 0).any())
    x = logits.detach().cpu().double()[:, P - 1:][live.cpu()].requires_grad_(True)
    tok = torch.log_softmax(x, -1).gather(1, seq[:, P:][live].cpu()[:, None])[:, 0]
    r, a = torch.exp(tok - old[live].cpu().double()), adv[live].cpu().double()
    want = torch.maximum(-a * r, -a * r.clamp(0.8, 1.2)).sum() / sum(ends)
    want.backward()
    # the vocabulary is small: a log-prob is off by 34 * 2^-23 + 17 * 2^-24 < 6e-6, a term by |A| r twice that, a gradient by four times
    size = (a.abs() * r.detach()).max()
    assert abs(float(loss.detach()) - float(want.detach())) <= float(size) * 1.2e-5
    assert float((grad[live].cpu().double() - x.grad).abs().max()) <= float(size) / sum(ends) * 2 * 2.4e-5


@pytest.mark.parametrize("shape,cut,g", [((2500, 40), slice(None), 0.5), ((5000, 1, 33), slice(None), 1.0), ((70000, 2, 17), slice(1, None), 1.0),
                                         ((70000, 2, 17), slice(1, None), -0.25)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("with_ref", [False, True])
def test_more_rows_and_groups_than_a_launch_takes(shape, cut, g, dtype, with_ref):
    """A gradient computed again over more rows than its launch has workgroups, and more groups of rows than a grid's second dimension."""
    from branchgan import ops
    gen = torch.Generator().manual_seed(shape[0] + shape[-1])
    V, view = shape[-1], lambda t: t[:, cut] if len(shape) == 3 else t
    full = [torch.randn(shape, generator=gen).to(dtype) for _ in range(2)]
    x, y = [view(t).reshape(-1, V).double() for t in full]
    rows = x.shape[0]
    lead = view(full[0]).shape[:-1]
    ids = torch.randint(0, V, (rows,), generator=gen)
    lx, ly = torch.log_softmax(x, -1), torch.log_softmax(y, -1)
    logp = lx.gather(1, ids[:, None])[:, 0]
    old, adv = (logp + 0.3 * torch.randn(rows, generator=gen)).float(), torch.randn(rows, generator=gen)
    ratio = torch.exp(logp - old.double())
    for end in (0.8, 1.2):                                                   # off the clip's ends, where the gradient jumps
        old = torch.where((ratio - end).abs() < 1e-3, old + 0.01, old)
    ratio, a, beta = torch.exp(logp - old.double()), adv.double(), 0.1 if with_ref else 0.0
    w = (torch.arange(rows) % 5 > 0).double()
    plain, clipped = -a * ratio, -a * ratio.clamp(0.8, 1.2)
    slope, p, gap = torch.where(plain >= clipped, plain, 0.0), lx.exp(), lx - ly
    kl = (p * gap).sum(-1) if with_ref else torch.zeros(rows, dtype=torch.float64)
    want = (w * (torch.maximum(plain, clipped) + beta * kl)).sum() / w.sum()
    one = torch.zeros_like(p).scatter_(1, ids[:, None], 1.0)
    grad = g / w.sum() * w[:, None] * (slope[:, None] * (one - p) + beta * p * (gap - kl[:, None]))
    leaf = full[0].cuda().requires_grad_(True)
    dev = lambda t: t.cuda().view(lead)
    loss, got_logp, got_kl = ops.policy_loss(view(leaf), dev(ids), dev(old), dev(adv), weights=dev(w.float()), kl_coef=beta,
                                             ref_logits=view(full[1].cuda()) if with_ref else None)
    (loss * g).backward()
    # dl: a p, and a log-prob; the full KL 4 dl of its terms' magnitudes and 4 dl; a row's term 2 dl |A| ratio, its gradient 4 dl of its parts
    dl = 34 * 2.0 ** -23 + (V / 256 + 16) * 2.0 ** -24
    kl_tol = 4 * dl * (p * gap.abs()).sum(-1) + 4 * dl + 2.0 ** -23 * kl.abs()
    near = lambda got, ref, tol: bool((((got.cpu().double().reshape(ref.shape) - ref).abs() <= tol) | (w == 0)).all())
    assert near(got_logp, logp, dl + 2.0 ** -24 * logp.abs()) and near(got_kl, kl, kl_tol)
    term_tol = 2 * dl * (a * ratio).abs() + beta * kl_tol
    assert abs(float(loss.detach()) - float(want)) <= float((w * term_tol).sum() / w.sum()) + 2.0 ** -23 * abs(float(want))
    tol = 4 * dl * (a * ratio).abs()[:, None] * (one + p) + beta * p * (4 * dl * (gap.abs() + kl.abs()[:, None]) + 4 * dl + kl_tol[:, None])
    tol = tol * abs(g) / w.sum() * w[:, None] + torch.finfo(dtype).eps / 2 * (1 + 1e-5) * grad.abs() + 1e-38
    got = leaf.grad.cpu().double()
    assert bool(((view(got).reshape(-1, V) - grad).abs() <= tol).all())
    view(got).zero_()
    assert not got.any()


@pytest.mark.parametrize("family", ["gpt2", "gpt_neox"])
@pytest.mark.parametrize("fused_path", [True, False])
@pytest.mark.parametrize("bits", [4, 8])
def test_a_chunk_through_the_model_is_its_tokens_one_by_one(family, fused_path, bits, monkeypatch):
    """models.CachePast with several new tokens, sequences of uneven length and padding: the logits of each token decoded alone, and nothing
    written behind a sequence's last one."""
    from branchgan import configs, fused, kvcache, models, ops
    monkeypatch.setattr(fused, "ENABLED", fused_path)
    torch.manual_seed(6)
    lm = models.make_lm(configs.LMConfig(family, 211, 128, 2, 4, 128)).cuda()
    B, T, cap, held, counts = 4, 7, 64, (40, 0, 33, 12), (7, 5, 0, 1)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    ids = torch.randint(0, 211, (B, T), device="cuda")
    gen = torch.Generator().manual_seed(bits)
    caches = [kvcache.QuantizedKVCache(2, B, 4, cap, 32, bits=bits) for _ in range(2)]
    for l in range(2):
        k, v = [torch.randn(B, 4, cap, 32, generator=gen).cuda() for _ in range(2)]
        for c in caches:
            ops.kv_cache_append(c.layer(l), k, v)
    before = [ops.kv_cache_read(caches[0].layer(l), cap, dtype=torch.float32) for l in range(2)]
    start = i32(held)
    def forward(cache, tokens, at, n, most):
        pos = at[:, None] + torch.arange(tokens.shape[1], device="cuda", dtype=torch.int32)
        return lm(input_ids=tokens, position_ids=pos, textualPast=models.CachePast(cache, at, n, max_keys=most), returnLmLogits=True).logits.float()
    with torch.no_grad():
        whole = forward(caches[0], ids, start, i32(counts), max(held) + T)
        for t in range(T):
            n = i32([int(t < c) for c in counts])
            one = forward(caches[1], ids[:, t:t + 1], start + t, n, cap)
            # layer 0's keys are the same numbers up to fp32 rounding; a code of layer 1 may flip at its border, a step of 1 / 7 of a key's maximum
            for b in range(B):
                if t < counts[b]:
                    torch.testing.assert_close(whole[b, t], one[b, 0], rtol=0, atol=0.02 * float(whole.abs().max()))
    for l in range(2):
        for was, now in zip(before[l], ops.kv_cache_read(caches[0].layer(l), cap, dtype=torch.float32)):
            for b in range(B):
                new = torch.zeros(cap, dtype=torch.bool)
                new[held[b]:held[b] + counts[b]] = True
                assert torch.equal(was[b][:, ~new], now[b][:, ~new]) and (counts[b] == 0 or not torch.equal(was[b][:, new], now[b][:, new]))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("T", [1, 2])
def test_scales_next_to_a_tie_are_the_documented_product(bits, T):
    """fp32 maxima on, one step below and one above L t, t halfway between two bf16 numbers, where a product with 1 / L and a quotient by L can
    round to different neighbours: the scale is bf16(a * fp32(1 / L)), worked out here in whole numbers, and what a tensor divided by the
    number L gives on the same device.  It is read off the held value of the maximum itself, L s."""
    from branchgan import kvcache, ops
    top = 7 if bits == 4 else 127
    t = torch.arange(257, 512, 2).double() / 256                             # the 128 ties of [1, 2)
    a = torch.cat([torch.nextafter((top * t).float(), torch.tensor(to)) for to in (0.0, math.inf)] + [(top * t).float()])
    a = torch.cat([a * 2.0 ** e for e in (-100, 0, 3, 90)])
    def bf16_of(x):                                                          # fp32 -> bf16, half to even, on the bits
        u = x.view(torch.int32).long()
        return (((u + 0x7FFF + ((u >> 16) & 1)) >> 16) << 16).int().view(torch.float32)
    reciprocal = torch.tensor(1 / top, dtype=torch.float32)
    scale = bf16_of((a.double() * reciprocal.double()).float())             # 48 bits: exact in a double, rounded to fp32 once
    assert not torch.equal(scale, bf16_of((a.double() / top).float()))       # the points tell the two apart
    assert torch.equal(scale, bf16_of((a.cuda() / top).cpu()))
    x = torch.zeros(len(a), 1, T, 64)
    x[:, 0, :, 3], x[:, 0, :, 40] = a[:, None], -a[:, None]
    x[:, 0, :, 50] = 0.37 * a[:, None]
    layer = kvcache.QuantizedKVCache(1, len(a), 1, T, 64, bits=bits).layer(0)
    ops.kv_cache_append(layer, x.cuda(), x.flip(-1).contiguous().cuda())
    k, v = [r.cpu() for r in ops.kv_cache_read(layer, T, dtype=torch.float32)]
    for t in range(T):
        assert torch.equal(k[:, 0, t, 3], top * scale) and torch.equal(k[:, 0, t, 40], -top * scale)
    assert torch.equal(k.double(), OK.held_values(x, bits)) and torch.equal(v.double(), OK.held_values(x.flip(-1), bits))
