"""The clipped policy loss with a KL term against float64 (oracle/policy.py), forward and backward.

Tolerances, derived.  An exponential is off by |z| 2^-23 (the roundings of its argument z = (logit - max) / T, of which only |z| < 30
matters: below it p < 1e-13) + 2^-21 (the instruction); the sum of V of them, V / 256 in a row and a tree of ten, by (V / 256 + 16)
2^-24.  So  del = 34 * 2^-23 + (V / 256 + 16) 2^-24  bounds the relative error of every p and the absolute error of logp (which is then rounded: 2^-24 |logp|)."""
import contextlib
import math

import pytest
import torch

from oracle import policy as O

pytestmark = pytest.mark.gpu


def delta(V):
    return 34 * 2.0 ** -23 + (V / 256 + 16) * 2.0 ** -24


def inputs(rows, V, dtype, seed, ref, scale=2.5):
    g = torch.Generator().manual_seed(seed)
    d = dict(logits=(scale * torch.randn(rows, V, generator=g)).to(dtype), ids=torch.randint(0, V, (rows,), generator=g))
    lp = torch.log_softmax(d["logits"].double(), -1).gather(1, d["ids"][:, None])[:, 0]
    d["old_logp"] = (lp + 0.4 * torch.randn(rows, generator=g)).float()
    d["advantages"] = torch.randn(rows, generator=g)
    if ref == "logits":
        d["ref_logits"] = (d["logits"].float() + 0.5 * torch.randn(rows, V, generator=g)).to(dtype)
    if ref == "logp":
        d["ref_logp"] = (lp + 0.3 * torch.randn(rows, generator=g)).float()
    return d


def off_the_clip(d, temperature, low, high):
    """Rows whose ratio lies within 1e-4 of an end of the clip range (where the gradient jumps) move away from it."""
    ok = (d["ids"] >= 0) & (d["ids"] < d["logits"].shape[1])
    lp = torch.log_softmax(d["logits"].double() / temperature, -1).gather(1, d["ids"].clamp(0, d["logits"].shape[1] - 1)[:, None])[:, 0]
    r = torch.exp(lp - d["old_logp"].double())
    near = ok & (((r - (1 - low)).abs() < 1e-4) | ((r - (1 + high)).abs() < 1e-4))
    d["old_logp"] = torch.where(near, d["old_logp"] + 0.01, d["old_logp"])
    return d


def run(d, g=1.0, place=None, **kw):
    from branchgan import losses
    names = dict(weights="mask", ref_logp="refLogProbs", ref_logits="refLogits")
    dev = {k: v.cuda() for k, v in d.items()}
    if place is not None:
        return run_placed(dev, g, place, names, kw)
    x = dev.pop("logits").requires_grad_(True)
    ids, old, adv = dev.pop("ids"), dev.pop("old_logp"), dev.pop("advantages")
    loss, logp, kl = losses.clippedPolicyLoss(x, ids, old, adv, **{names[k]: v for k, v in dev.items()}, clipRange=(kw.get("clip_low", 0.2), kw.get("clip_high", 0.2)),
                                              klWeight=kw.get("kl_coef", 0.0), temperature=kw.get("temperature", 1.0), denominator=kw.get("denominator"))
    (loss * g).backward()
    return loss.detach().cpu(), logp.cpu(), kl.cpu(), x.grad


def run_placed(dev, g, place, names, kw):
    """place(rows, V) -> (shape of a larger tensor, view(that tensor) holding the rows as (..., V), whether the reference lies alike)."""
    from branchgan import losses
    rows, V = dev["logits"].shape
    shape, view, alike = place(rows, V)
    def lay(t):
        full = torch.full(shape, float("nan"), dtype=t.dtype, device="cuda")
        view(full).copy_(t.view(view(full).shape))
        return full
    leaf = lay(dev.pop("logits")).requires_grad_(True)
    x = view(leaf)
    if "ref_logits" in dev:
        dev["ref_logits"] = view(lay(dev["ref_logits"])) if alike else dev["ref_logits"].view(x.shape)
    dev = {k: t if k == "ref_logits" else t.view(x.shape[:-1]) for k, t in dev.items()}
    ids, old, adv = dev.pop("ids"), dev.pop("old_logp"), dev.pop("advantages")
    loss, logp, kl = losses.clippedPolicyLoss(x, ids, old, adv, **{names[k]: v for k, v in dev.items()}, klWeight=kw.get("kl_coef", 0.0),
                                              temperature=kw.get("temperature", 1.0))
    if x.dim() < 4:
        assert loss.grad_fn.saved_tensors[0].data_ptr() == x.data_ptr()             # read where it lies
    first, = torch.autograd.grad(loss, leaf, retain_graph=True)
    (loss * g).backward()
    grad = view(leaf.grad).reshape(rows, V)
    if g == 1.0:                                                                    # the gradient of the forward's reading, and the one computed again
        torch.testing.assert_close(first, leaf.grad, rtol=2 * torch.finfo(x.dtype).eps if x.dtype == torch.bfloat16 else 1e-4, atol=1e-7)
    outside = leaf.grad.clone()
    view(outside).zero_()
    assert not outside.any()
    return loss.detach().cpu(), logp.reshape(-1).cpu(), kl.reshape(-1).cpu(), grad


def check(d, g=1.0, **kw):
    T, beta = kw.get("temperature", 1.0), kw.get("kl_coef", 0.0)
    x = d["logits"].double().requires_grad_(True)
    ref = {k: v for k, v in d.items() if k != "logits"}
    loss, logp, kl = O.policy_loss(x, **ref, **{k: v for k, v in kw.items() if k != "place"})
    (loss * g).backward()
    got_loss, got_logp, got_kl, grad = run(d, g, **kw)
    rows, V = d["logits"].shape
    dl = delta(V)
    w = torch.ones(rows, dtype=torch.float64) if d.get("weights") is None else d["weights"].double()
    w = torch.where((d["ids"] >= 0) & (d["ids"] < V), w, torch.zeros_like(w))
    n = float(w.sum()) if kw.get("denominator") is None else float(kw["denominator"])
    assert bool(((got_logp.double() - logp).abs() <= dl + 2.0 ** -24 * logp.abs()).all())
    # KL: p off by dl, differences by dl; the sampled form moves by |1 - exp(d)| per unit of logp
    if d.get("ref_logits") is not None:
        lx, ly = torch.log_softmax(d["logits"].double() / T, -1), torch.log_softmax(d["ref_logits"].double() / T, -1)
        far = torch.where(lx.exp() > 0, (lx - ly).abs(), torch.zeros_like(lx))
        kl_tol = 4 * dl * (lx.exp() * torch.where(lx.exp() > 0, far, torch.zeros_like(far))).sum(-1) + 4 * dl + 2.0 ** -23 * kl.abs()
    elif d.get("ref_logp") is not None:
        far = None
        kl_tol = dl * (1 - torch.exp(d["ref_logp"].double() - logp)).abs() * 2 + 2.0 ** -23 * kl.abs() + dl * dl
    else:
        far, kl_tol = None, torch.zeros(rows, dtype=torch.float64)
    assert bool((((got_kl.double() - kl).abs() <= kl_tol) | (w == 0)).all())
    ratio = torch.exp(logp - d["old_logp"].double())
    pg_tol = (d["advantages"].double() * ratio).abs() * 2 * dl
    total = (w.abs() * (pg_tol + abs(beta) * kl_tol))[w != 0].sum() / abs(n) if n else torch.zeros(())
    loss = float(loss.detach())
    assert abs(float(got_loss) - loss) <= float(total) + 2.0 ** -23 * abs(loss), (float(got_loss), loss)
    # gradient: slope (off by 2 dl of its parts) times (1[j = id] - p), p off by dl; KL part p (gap - kl); one rounding at the end
    p = torch.softmax(d["logits"].double() / T, -1)
    one = torch.zeros_like(p)
    inside = (d["ids"] >= 0) & (d["ids"] < V)
    one[inside.nonzero()[:, 0], d["ids"][inside]] = 1
    slope = (d["advantages"].double() * ratio).abs() + (abs(beta) * (1 + torch.exp(d["ref_logp"].double() - logp)) if d.get("ref_logp") is not None else 0)
    tol = 4 * dl * slope[:, None] * (one + p) * (w.abs() * abs(g) / abs(n or 1) / T)[:, None]
    if far is not None:
        tol = tol + (abs(beta) * abs(g) / abs(n or 1) / T * w.abs())[:, None] * p * (4 * dl * (far + kl.abs()[:, None]) + 4 * dl + kl_tol[:, None])
    tol = torch.where((w == 0)[:, None], torch.zeros_like(tol), tol)
    want = x.grad
    err = (grad.cpu().double() - want).abs()
    assert grad.dtype == d["logits"].dtype
    assert bool((err <= tol + torch.finfo(grad.dtype).eps / 2 * want.abs() * (1 + 1e-5) + 1e-38).all()), float((err / (tol + 1e-38)).max())
    return got_loss


@pytest.mark.parametrize("rows,V", [(1, 2), (3, 97), (33, 1031), (5, 50257), (6, 50304), (2, 120001)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("ref", [None, "logp", "logits"])
def test_against_float64(rows, V, dtype, ref):
    d = inputs(rows, V, dtype, rows + V, ref)
    check(off_the_clip(d, 0.8, 0.1, 0.3), clip_low=0.1, clip_high=0.3, kl_coef=0.07, temperature=0.8)


@pytest.mark.parametrize("ref", [None, "logp", "logits"])
def test_weights_padding_and_denominators(ref):
    d = inputs(41, 513, torch.float32, 7, ref)
    d["weights"] = torch.rand(41, generator=torch.Generator().manual_seed(1)) * (torch.arange(41) % 3 > 0)
    d["ids"][::7] = -100                                                    # padding by id
    d["ids"][5], d["ids"][6] = 513, 512                                     # one past the vocabulary, and its last entry
    d["logits"][3], d["logits"][7], d["advantages"][9], d["old_logp"][12] = math.nan, math.inf, math.nan, math.inf     # rows that do not count
    assert not d["weights"][[3, 9, 12]].any() and int(d["ids"][7]) == -100
    d = off_the_clip(d, 1.3, 0.2, 0.2)
    check(d, kl_coef=0.3, temperature=1.3)
    check(d, kl_coef=0.3, temperature=1.3, denominator=1000.0)
    check(d, g=-0.37, kl_coef=0.3, temperature=1.3, denominator=torch.tensor(64.0).cuda())
    d["weights"].zero_()                                                    # nothing counts
    loss, logp, kl, grad = run(d, kl_coef=0.3)
    assert float(loss) == 0 and not logp.any() and not kl.any() and not grad.any()


@pytest.mark.parametrize("lowest", [-math.inf, torch.finfo(torch.bfloat16).min])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masked_vocabulary(lowest, dtype):
    """Entries that both models mask, that only the policy masks, and a whole masked stretch at the row's start."""
    d = inputs(4, 3001, dtype, 17, "logits")
    d["ids"] = torch.tensor([900, 1500, 2999, 700])
    for t in (d["logits"], d["ref_logits"]):
        t[:, :600] = lowest
        t[1, 2000:] = lowest
    d["logits"][2, 1000:1100] = lowest
    lp = torch.log_softmax(d["logits"].double(), -1).gather(1, d["ids"][:, None])[:, 0]
    d["old_logp"] = (lp + torch.tensor([0.3, -0.3, 0.05, -0.05])).float()
    check(d, kl_coef=0.2)


def test_large_logits_and_broken_rows():
    d = inputs(4, 1000, torch.float32, 23, "logits")
    d["logits"][0] += 3000.0
    d["ref_logits"][0] -= 20000.0
    d["old_logp"] = torch.log_softmax(d["logits"].double(), -1).gather(1, d["ids"][:, None])[:, 0].float() + 0.05
    d["logits"][0], d["ref_logits"][0] = d["logits"][0].round(), d["ref_logits"][0].round()      # differences exact
    d["old_logp"][0] = torch.log_softmax(d["logits"][0].double(), -1)[d["ids"][0]].float() + 0.05
    check(d, kl_coef=0.1)
    d["logits"][2, 17] = math.nan                                           # a broken row that counts: the loss shows it
    loss, logp, _, grad = run(d, kl_coef=0.1)
    assert math.isnan(float(loss)) and math.isnan(float(logp[2])) and bool(grad[2].isnan().all()) and bool(grad[0].isfinite().all())


def test_gradient_against_differences():
    d = off_the_clip(inputs(6, 40, torch.float32, 29, "logits", scale=1.0), 0.9, 0.2, 0.2)
    kw = dict(kl_coef=0.5, temperature=0.9)
    _, _, _, grad = run(d, **kw)
    u = torch.randn(6, 40, generator=torch.Generator().manual_seed(2))
    h = 2.0 ** -7
    up, down = [float(O.policy_loss((d["logits"] + s * h * u).double(), **{k: v for k, v in d.items() if k != "logits"}, **kw)[0]) for s in (1, -1)]
    # the kernel's own loss is off by ~1e-6 at most: over 2 h that is 1e-4; the third derivative (|u| ~ 1, slopes of order 1) gives h^2
    own = [float(run({**d, "logits": d["logits"] + s * h * u}, **kw)[0]) for s in (1, -1)]
    slope = float((grad.cpu().double() * u).sum())
    assert abs((up - down) / (2 * h) - slope) < 4 * h * h and abs((own[0] - own[1]) / (2 * h) - slope) < 4 * h * h + 2e-4


def test_strides_leading_dimensions_and_integer_types():
    from branchgan import ops
    d = inputs(12, 777, torch.float32, 31, "logits")
    x = d["logits"].cuda()
    args = lambda s: [d[k].cuda().view(s) for k in ("ids", "old_logp", "advantages")]
    base = ops.policy_loss(x, *args((12,)), ref_logits=d["ref_logits"].cuda(), kl_coef=0.1)
    wide = torch.zeros(12, 800, device="cuda")
    wide[:, 5:782] = x
    shaped = ops.policy_loss(x.view(3, 4, 777), *args((3, 4)), ref_logits=d["ref_logits"].cuda().view(3, 4, 777), kl_coef=0.1)
    assert shaped[1].shape == (3, 4) and torch.equal(base[0], shaped[0]) and torch.equal(base[1], shaped[1].view(-1))
    w = wide.requires_grad_(True)
    strided = ops.policy_loss(w[:, 5:782], *args((12,)), ref_logits=d["ref_logits"].cuda(), kl_coef=0.1)
    torch.testing.assert_close(strided[0], base[0], rtol=1e-6, atol=1e-6)
    strided[0].backward()
    xr = x.clone().requires_grad_(True)
    ops.policy_loss(xr, args((12,))[0].int(), *args((12,))[1:], ref_logits=d["ref_logits"].cuda(), kl_coef=0.1)[0].backward()
    torch.testing.assert_close(w.grad[:, 5:782], xr.grad, rtol=1e-5, atol=1e-9)
    assert not w.grad[:, :5].any() and not w.grad[:, 782:].any()
    # one row of logits for every token (an expanded tensor): the gradient sums over them
    one = x[:1].clone().requires_grad_(True)
    ops.policy_loss(one.expand(12, 777), *args((12,)))[0].backward()
    rep = x[:1].repeat(12, 1).requires_grad_(True)
    ops.policy_loss(rep, *args((12,)))[0].backward()
    torch.testing.assert_close(one.grad[0], rep.grad.sum(0), rtol=1e-5, atol=1e-8)


PLACES = {
    "shifted": lambda R, V: ((3, R // 3 + 1, V), lambda t: t[:, :-1], True),                  # logits[:, :-1]
    "middle": lambda R, V: ((3, R // 3 + 5, V), lambda t: t[:, 2:-3], True),
    "middle_ref_dense": lambda R, V: ((3, R // 3 + 5, V), lambda t: t[:, 2:-3], False),
    "transposed": lambda R, V: ((R // 3, 3, V), lambda t: t.transpose(0, 1), True),
    "one_token": lambda R, V: ((R, 4, V), lambda t: t[:, 1:2], True),
    "one_sequence": lambda R, V: ((2, R + 3, V), lambda t: t[1:, 1:-2], True),
    "rows": lambda R, V: ((R + 4, V), lambda t: t[3:-1], True),
    "wide": lambda R, V: ((3, R // 3 + 1, V + 9), lambda t: t[:, 1:, 4:-5], True),
    "four_dimensions": lambda R, V: ((3, R // 6, 3, V), lambda t: t[:, :, 1:], True),
}


@pytest.mark.parametrize("place", PLACES)
@pytest.mark.parametrize("V,dtype", [(1031, torch.bfloat16), (2048, torch.bfloat16), (1031, torch.float32), (20001, torch.bfloat16), (13, torch.float32)])
@pytest.mark.parametrize("ref,g", [("logits", 1.0), ("logp", 1.0), ("logits", 0.7)])
def test_rows_where_they_lie(place, V, dtype, ref, g):
    """Slices and transpositions of (B, T, V), against float64; what lies around the rows is NaN and gets no gradient."""
    d = off_the_clip(inputs(12, V, dtype, 83, ref), 0.8, 0.2, 0.2)
    check(d, g, place=PLACES[place], kl_coef=0.1, temperature=0.8)


@pytest.mark.parametrize("g", [1.0, 0.5])
def test_saved_tensors_that_come_back_in_another_layout(g):
    """Hooks that keep a copy of the saved logits (off-loading to the host does) return them dense, whatever they were."""
    from branchgan import ops
    d = inputs(12, 1031, torch.bfloat16, 85, "logits")
    full, ref = [torch.zeros(3, 9, 1031, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    full[:, 2:6], ref[:, 2:6] = d["logits"].view(3, 4, 1031).cuda(), d["ref_logits"].view(3, 4, 1031).cuda()
    rest = [d[k].view(3, 4).cuda() for k in ("ids", "old_logp", "advantages")]
    grads = []
    for hooked in (False, True):
        x = full.clone().requires_grad_(True)
        hooks = torch.autograd.graph.saved_tensors_hooks(lambda t: t.contiguous().clone(), lambda t: t) if hooked else contextlib.nullcontext()
        with hooks:
            loss = ops.policy_loss(x[:, 2:6], *rest, ref_logits=ref[:, 2:6], kl_coef=0.1)[0]
        torch.autograd.grad(loss, x, retain_graph=True)                             # the second backward reads the logits again
        (loss * g).backward()
        grads.append(x.grad)
    assert torch.equal(*grads)


def test_backward_twice_and_without_grad():
    from branchgan import ops
    d = inputs(9, 333, torch.bfloat16, 37, "logp")
    args = [d[k].cuda() for k in ("ids", "old_logp", "advantages")]
    x = d["logits"].cuda().requires_grad_(True)
    loss, _, _ = ops.policy_loss(x, *args, ref_logp=d["ref_logp"].cuda(), kl_coef=0.1)
    g1, = torch.autograd.grad(loss, x, retain_graph=True)
    g1 = g1.clone()
    g3, = torch.autograd.grad(3 * loss, x, retain_graph=True)
    g1b, = torch.autograd.grad(loss, x)
    assert torch.equal(g1, g1b)
    torch.testing.assert_close(g3.float(), 3 * g1.float(), rtol=2.0 ** -7, atol=1e-12)
    with torch.no_grad():
        assert torch.equal(ops.policy_loss(x, *args, ref_logp=d["ref_logp"].cuda(), kl_coef=0.1)[0], loss)


@pytest.mark.parametrize("ref", [None, "logp", "logits"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_for_every_size_of_workgroup(dtype, ref):
    """Vocabularies on both sides of every limit in the choice of kernel (whole vectors per thread and workgroup), and rows whose
    16-byte grid differs between logits, reference and gradient."""
    n = 4 if dtype == torch.float32 else 8
    for V in (2 * n - 1, 2 * n, 2 * n + 1, 512 * n - n - 1, 512 * n, 2048 * n - 1, 2048 * n + 1, 6656 * n - n - 1, 6656 * n - 1, 6656 * n + 1):
        check(off_the_clip(inputs(2, V, dtype, V, ref), 1.0, 0.2, 0.2), kl_coef=0.1)
    if ref == "logits":
        from branchgan import ops
        d = off_the_clip(inputs(5, 1001, dtype, 3, ref), 1.0, 0.2, 0.2)
        wide = torch.zeros(5, 1003, dtype=dtype, device="cuda")
        wide[:, 1:1002] = d["logits"].cuda()
        want, _, _, grad = run(d, kl_coef=0.1)
        x = wide.requires_grad_(True)
        loss, _, _ = ops.policy_loss(x[:, 1:1002], *[d[k].cuda() for k in ("ids", "old_logp", "advantages")], ref_logits=d["ref_logits"].cuda(), kl_coef=0.1)
        loss.backward()
        torch.testing.assert_close(loss.detach().cpu(), want, rtol=1e-6, atol=1e-7)
        torch.testing.assert_close(x.grad[:, 1:1002], grad, rtol=2 * torch.finfo(dtype).eps, atol=1e-9)


def test_many_rows_and_the_largest_vocabulary_are_one_answer():
    """More rows than the workgroups sum weights for themselves; the loss equals the mean of the rows' own losses."""
    from branchgan import ops
    d = off_the_clip(inputs(1500, 300, torch.float32, 61, "logp"), 1.0, 0.2, 0.2)
    d["weights"] = (torch.arange(1500) % 5 > 0).float()
    check(d, kl_coef=0.1)
    args = [d[k].cuda() for k in ("logits", "ids", "old_logp", "advantages")]
    whole, _, _ = ops.policy_loss(*args, weights=d["weights"].cuda(), ref_logp=d["ref_logp"].cuda(), kl_coef=0.1)
    parts = [float(ops.policy_loss(*[a[i:i + 300] for a in args], weights=d["weights"][i:i + 300].cuda(), ref_logp=d["ref_logp"][i:i + 300].cuda(),
                                   kl_coef=0.1, denominator=1200)[0]) for i in range(0, 1500, 300)]
    assert abs(float(whole) - sum(parts)) <= 6 * 2.0 ** -23 * sum(abs(p) for p in parts)


def test_captured_step_replays():
    """Forward and backward captured once, replayed on new inputs with eager work in between."""
    from branchgan import ops
    first = inputs(64, 5003, torch.bfloat16, 41, "logits")
    bufs = {k: v.cuda() for k, v in first.items()}
    def step(b, x):
        loss, logp, kl = ops.policy_loss(x, b["ids"], b["old_logp"], b["advantages"], ref_logits=b["ref_logits"], kl_coef=0.1)
        return (loss.detach(), logp, kl, torch.autograd.grad(loss, x)[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(bufs, bufs["logits"].detach().requires_grad_(True))
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step(bufs, bufs["logits"].detach().requires_grad_(True))
    for seed in (42, 43, 44):
        new = inputs(64, 5003, torch.bfloat16, seed, "logits")
        for k, v in new.items():
            bufs[k].copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        fresh = {k: v.cuda() for k, v in new.items()}
        for a, b in zip(out, step(fresh, fresh["logits"].requires_grad_(True))):
            assert torch.equal(a, b)


def test_rollouts_over_a_quantised_cache_and_the_update_on_them():
    """The operators as they are used together: sample over a 4-bit cache with log-probs, score the rollouts with the full model and a
    reference, clipped update with the KL over the vocabulary; loss and the gradient of the head against float64 on the same logits."""
    from branchgan import configs, generate, losses, models
    torch.manual_seed(9)
    lm, ref = [models.make_lm(configs.LMConfig("gpt_neox", 211, 128, 2, 4, 128)).cuda() for _ in range(2)]
    prompt = torch.randint(0, 211, (4, 11), device="cuda")
    seq, old = generate.generate(lm, prompt, max_new_tokens=21, do_sample=True, temperature=0.9, cache_bits=4, return_logprobs=True,
                                 generator=torch.Generator(device="cuda").manual_seed(1))
    adv = torch.randn(4, 1, generator=torch.Generator().manual_seed(3)).expand(4, 21).cuda()
    out = lm(input_ids=seq, returnLmLogits=True).logits[:, 10:-1]
    with torch.no_grad():
        ref_logits = ref(input_ids=seq, returnLmLogits=True).logits[:, 10:-1]
    out.retain_grad()
    loss, logp, kl = losses.clippedPolicyLoss(out, seq[:, 11:], old, adv, refLogits=ref_logits, klWeight=0.1, temperature=0.9)
    loss.backward()
    assert float((logp - old).abs().max()) < 1.0 and bool((kl > 0).all())    # the rollout policy is near the model's, the reference another
    flat = lambda t: t.detach().cpu().reshape(-1, *t.shape[2:])
    d = dict(logits=flat(out).contiguous(), ids=flat(seq[:, 11:]), old_logp=flat(old), advantages=flat(adv), ref_logits=flat(ref_logits).contiguous())
    x = d["logits"].double().requires_grad_(True)
    want, _, _ = O.policy_loss(x, **{k: v for k, v in d.items() if k != "logits"}, kl_coef=0.1, temperature=0.9)
    want.backward()
    torch.testing.assert_close(loss.detach().cpu().double(), want.detach(), rtol=1e-5, atol=1e-6)
    torch.testing.assert_close(flat(out.grad).double(), x.grad, rtol=1e-4, atol=1e-7)
    assert lm.embed_out.weight.grad is not None and bool(lm.embed_out.weight.grad.isfinite().all()) and bool(lm.embed_out.weight.grad.any())


def test_prompt_positions_left_out_by_weight_or_by_slice():
    """The logits of a whole sequence with weight 0 on its prompt, or their slice: the same rows, the same value and gradient; what the
    rows left out hold does not matter."""
    from branchgan import losses
    g = torch.Generator().manual_seed(71)
    B, S, P, V = 3, 9, 4, 1003
    logits, ref = [torch.randn((B, S, V), generator=g).to(torch.bfloat16).cuda() for _ in range(2)]
    ids = torch.randint(0, V, (B, S), generator=g).cuda()
    old, adv = [(torch.randn((B, S - P), generator=g) - c).cuda() for c in (7.0, 0.0)]
    behind = lambda t: torch.nn.functional.pad(t, (P, 0))
    x = logits.clone().requires_grad_(True)
    want = losses.clippedPolicyLoss(x[:, P:], ids[:, P:], old, adv, refLogits=ref[:, P:], klWeight=0.1)
    want[0].backward()
    broken = [t.clone() for t in (logits, ref)]
    for t in broken:
        t[:, :P] = float("nan")
    y = broken[0].requires_grad_(True)
    got = losses.clippedPolicyLoss(y, ids, behind(old), behind(adv), mask=behind(torch.ones_like(old)), refLogits=broken[1], klWeight=0.1)
    got[0].backward()
    # Not bit for bit: V is odd, so a row lies elsewhere on the 16-byte grid in the copy that the slice becomes, and its elements fall to
    # other threads.  A thread adds at most 17 terms in fp32 (two vectors of 8 and a single one), so each of the three sums s, s', t is off
    # by at most 17 u of its terms' magnitudes, u = 2^-24, in either call; everything behind them is fp64 or the same operation.
    #   log s: 17 u.   logp: that, and its rounding (|logp| < 16).   kl = t / s - (log s - log s'): with |difference of two logits| <= D
    #   in every term, 17 u D from t, 17 u D from s, 34 u from the logs, rounding u |kl|.
    u, D = 2.0 ** -24, float((logits - ref).float().abs().max() + (logits.float().amax(-1) - ref.float().amax(-1)).abs().max())
    e_logp, e_kl = 2 * (17 + 16) * u, 2 * (34 * D + 34 + 2) * u
    assert float((got[1][:, P:] - want[1]).abs().max()) <= e_logp and float((got[2][:, P:] - want[2]).abs().max()) <= e_kl
    # a row's term A ratio moves by ratio (e_logp + 4 u) (expf, the product, the ratio's argument rounded to fp32: |argument| < 8)
    A_r = (adv.abs() * (want[1] - old).exp()).max()
    assert abs(float((got[0] - want[0]).detach())) <= float(A_r) * (e_logp + 12 * u) + 0.1 * e_kl + abs(float(want[0].detach())) * u
    # a logit's gradient is p / N (slope and 0.1 (difference - off)), then bf16: neighbours at most (2^-7 of the value), and where the parts cancel,
    # p / N times what slope, off (both e_kl and e_logp at most, as above) and p (relative 17 u, 3 more operations) moved
    p_max = float(torch.softmax(logits.float(), -1).max())
    moved = p_max / (B * (S - P)) * (float(A_r) * (e_logp + 32 * u) + 0.1 * (e_kl + D * 40 * u))
    torch.testing.assert_close(y.grad.float(), x.grad.float(), rtol=2.0 ** -7, atol=moved)
    assert not y.grad[:, :P].any()


def test_refusals():
    from branchgan import ops
    d = inputs(4, 50, torch.float32, 53, "logits")
    x, ids, old, adv = [d[k].cuda() for k in ("logits", "ids", "old_logp", "advantages")]
    ref = d["ref_logits"].cuda()
    for args, kw in (((x, ids[:3], old, adv), {}), ((x, ids, old[:, None], adv), {}), ((x, ids, old, adv), dict(weights=adv[:2])),
                     ((x, ids, old, adv), dict(ref_logits=ref[:, :40])), ((x, ids, old, adv), dict(ref_logits=ref.bfloat16())),
                     ((x, ids, old, adv), dict(ref_logits=ref, ref_logp=old)), ((x, ids, old, adv), dict(temperature=0.0)),
                     ((x, ids, old, adv), dict(temperature=math.nan)), ((x, ids, old, adv), dict(clip_low=-0.1)),
                     ((x[:0], ids[:0], old[:0], adv[:0]), {}), ((x, ids, old, adv), dict(denominator=torch.ones(2, device="cuda")))):
        with pytest.raises(ValueError):
            ops.policy_loss(*args, **kw)
    for bad in ((x.half(), ids, old, adv), (x, ids.float(), old, adv)):
        with pytest.raises(TypeError):
            ops.policy_loss(*bad)
    with pytest.raises(RuntimeError):
        ops.policy_loss(x, ids, old, adv, temperature=1e9)
