"""The quantised key / value cache and attention over it, against float64 on the CPU (oracle/kvcache.py).

What the cache holds is compared exactly (codes are those of the real quotients, see csrc/kv_cache.hip).  Tolerances of the
attention, derived: a score is a sum of Dh products whose factors are exact in the kernel; with fp32 sums in any order it is off by at
most (Dh + 8) 2^-23 sum |q k| scale =: ds (twice the textbook (n - 1) u, for the exponent's own rounding).  A probability is then off by a
factor of 2 ds, its products and sums over n keys by n 2^-24, and bf16 queries' probabilities are carried in two bf16 pieces
(2^-16), fp32 queries' in three (2^-23): |out - ref| <= max|v| (2 ds + n 2^-24 + piece) + half a step of the output type."""
import math

import pytest
import torch

from oracle import kvcache as O

pytestmark = pytest.mark.gpu


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def bound(q, k, v, scale, dtype, ref):
    """Per-element bound of the docstring (k, v: held values, float64)."""
    Dh, n = q.shape[-1], k.shape[2]
    G = q.shape[1] // k.shape[1]
    mags = torch.matmul(q.double().abs(), k.abs().repeat_interleave(G, 1).transpose(-1, -2).contiguous()).amax(-1) * scale     # (B, Hq, T)
    rel = 2 * (Dh + 8) * 2.0 ** -23 * mags + n * 2.0 ** -24 + (2.0 ** -16 if dtype == torch.bfloat16 else 2.0 ** -23)
    vmax = v.abs().amax(2).repeat_interleave(G, 1)[:, :, None]                                                              # (B, Hq, 1, Dh)
    return rel[..., None] * vmax + half_step(dtype) * ref.abs() + 1e-30, rel


def make(gen, B, H, n, Dh, dtype, spread=0.7):
    gain = torch.exp(spread * torch.randn(1, H, 1, Dh, generator=gen))
    return [(torch.randn(B, H, n, Dh, generator=gen) * g).to(dtype) for g in (gain, 1.0)]


def new_cache(B, H, capacity, Dh, bits, fill=None):
    from branchgan import kvcache
    c = kvcache.QuantizedKVCache(1, B, H, capacity, Dh, bits=bits)
    if fill is not None:
        c.data.copy_(torch.randint(0, 256, c.data.shape, dtype=torch.uint8, generator=torch.Generator().manual_seed(fill)))
    return c.layer(0)


def within(err, tol):
    return bool((err.abs() <= tol).all())


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def same(a, b):
    """Equal bit for bit up to the sign of zero and NaN payloads."""
    a, b = a.cpu().float(), b.cpu().float()
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


@pytest.mark.parametrize("Dh", [32, 64, 128, 256])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T", [1, 2, 33, 100])
def test_append_and_read_hold_the_definition(bits, Dh, dtype, T):
    from branchgan import ops
    gen = torch.Generator().manual_seed(bits * Dh + T)
    B, H, cap = 3, 2, 150
    layer = new_cache(B, H, cap, Dh, bits, fill=5)
    before_k, before_v = ops.kv_cache_read(layer, cap, dtype=torch.float32)
    k, v = make(gen, B, H, T, Dh, dtype)
    k[0, 0, 0], v[1, 1, 0, :32] = 0, 0                                        # groups of zeros
    start, counts = i32(0, 31, 45), i32(T, max(T - 1, 1), T // 2)
    ops.kv_cache_append(layer, k.cuda(), v.cuda(), start=start, counts=counts)
    got = ops.kv_cache_read(layer, cap, dtype=torch.float32)
    for was, x, now in ((before_k, k, got[0]), (before_v, v, got[1])):
        want = was.cpu().double()
        held = O.held_values(x, bits)
        for b in range(B):
            s, c = int(start[b]), int(counts[b])
            want[b, :, s:s + c] = held[b, :, :c]
        assert same(now, want)                                               # what was written, and everything else as it was
    rk, rv = ops.kv_cache_read(layer, T + 3, start=start, counts=counts, dtype=dtype)
    for x, r in ((k, rk), (v, rv)):
        want = torch.zeros(B, H, T + 3, Dh, dtype=torch.float64)
        held = O.held_values(x, bits)
        for b in range(B):
            want[b, :, :int(counts[b])] = held[b, :, :int(counts[b])]
        assert same(r, want.to(dtype))


@pytest.mark.parametrize("bits", [4, 8])
def test_codes_at_their_borders(bits):
    """fp32 inputs on, one step below and one step above every border (k + 1/2) s: the code is the real quotient's."""
    from branchgan import ops
    top = 7 if bits == 4 else 127
    rows = []
    for s in (0.37109375, 1.0, 3.0, 2.0 ** -40 * 1.5078125):                 # bf16 numbers
        s = torch.tensor(s).bfloat16().float()
        half = ((torch.arange(top).float() + 0.5) * s)                       # exact in fp32
        pts = torch.cat((half, torch.nextafter(half, torch.tensor(math.inf)), torch.nextafter(half, torch.tensor(-math.inf))))
        pts = torch.cat((pts, -pts))
        pts = torch.cat((pts, torch.zeros(-len(pts) % 31)))
        rows += [torch.cat((p, top * s.view(1))) for p in pts.view(-1, 31)]
    x = torch.stack(rows)                                                    # each row: 31 points and the value that fixes the scale
    x = x[: len(x) // 2 * 2].reshape(1, 1, -1, 32)
    layer = new_cache(1, 1, x.shape[2], 32, bits)
    ops.kv_cache_append(layer, x.cuda(), x.flip(2).contiguous().cuda())
    k, v = ops.kv_cache_read(layer, x.shape[2], dtype=torch.float32)
    assert same(k, O.held_values(x, bits)) and same(v, O.held_values(x.flip(2), bits))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("T", [1, 40])
def test_extreme_values(bits, T):
    from branchgan import ops
    x = torch.randn(1, 1, T, 128, generator=torch.Generator().manual_seed(1))
    x[0, 0, 0, 5], x[0, 0, 0, 40], x[0, 0, T - 1, 70], x[0, 0, T - 1, 99] = math.inf, math.nan, -3.3e38, 2.0 ** 126
    y = torch.full((1, 1, T, 128), 1e-38)
    y[..., 32:64], y[..., 64:96], y[..., 96:] = 1e-44, -2.0 ** -119, torch.finfo(torch.bfloat16).tiny * 7
    layer = new_cache(1, 1, T, 128, bits)
    ops.kv_cache_append(layer, x.cuda(), y.cuda())
    k, v = ops.kv_cache_read(layer, T, dtype=torch.float32)
    assert same(k, O.held_values(x, bits)) and same(v, O.held_values(y, bits))
    assert bool(k[0, 0, 0, :64].isnan().all()) and bool(k[0, 0, T - 1, 64:96].isnan().all()) and bool(k[0, 0, T - 1, 96:].isfinite().all())


def test_strided_and_unaligned_inputs():
    from branchgan import ops
    gen = torch.Generator().manual_seed(3)
    B, H, T, Dh = 2, 3, 37, 64
    packed = torch.randn(B, T, 3, H, Dh, generator=gen).bfloat16()           # slices of a packed projection
    odd = torch.randn(B, H, T, Dh + 3, generator=gen).bfloat16()             # rows off the 16-byte grid
    for base, cut in ((packed, lambda t: (t[:, :, 1].permute(0, 2, 1, 3), t[:, :, 2].permute(0, 2, 1, 3))),
                      (odd, lambda t: (t[..., 1:Dh + 1], t[..., 2:Dh + 2]))):
        (k, v), (kd, vd) = cut(base), cut(base.cuda())
        for n in (T, 1):
            layer = new_cache(B, H, T, Dh, 4)
            ops.kv_cache_append(layer, kd[:, :, :n], vd[:, :, :n])
            rk, rv = ops.kv_cache_read(layer, n, dtype=torch.bfloat16)
            assert same(rk, O.held_values(k[:, :, :n], 4).bfloat16()) and same(rv, O.held_values(v[:, :, :n], 4).bfloat16())
    # an expanded key (one row for every head) and a transposed one (last dimension not dense)
    one = torch.randn(B, 1, T, Dh, generator=gen)
    tr = torch.randn(B, H, Dh, T, generator=gen)
    layer = new_cache(B, H, T, Dh, 8)
    ops.kv_cache_append(layer, one.cuda().expand(B, H, T, Dh), tr.cuda().transpose(-1, -2))
    rk, rv = ops.kv_cache_read(layer, T, dtype=torch.float32)
    assert same(rk, O.held_values(one, 8).expand(B, H, T, Dh)) and same(rv, O.held_values(tr.transpose(-1, -2), 8))


def test_positions_outside_the_cache_are_dropped():
    from branchgan import ops
    gen = torch.Generator().manual_seed(4)
    for T in (1, 50):
        k, v = make(gen, 5, 1, T, 64, torch.float32)
        layer = new_cache(5, 1, 70, 64, 4, fill=7)
        want = [x.cpu().double() for x in ops.kv_cache_read(layer, 70, dtype=torch.float32)]
        start = i32(69, 70, -20, 2 ** 31 - 3, -2 ** 31)
        ops.kv_cache_append(layer, k.cuda(), v.cuda(), start=start, counts=i32(T, T, T, T, T + 100))
        got = ops.kv_cache_read(layer, 70, dtype=torch.float32)
        for w, x, g in zip(want, (k, v), got):
            held = O.held_values(x, 4)
            for b in range(3):
                for t in range(T):
                    p = int(start[b]) + t
                    if 0 <= p < 70:
                        w[b, :, p] = held[b, :, t]
            assert same(g, w)
        rk, _ = ops.kv_cache_read(layer, 9, start=start, dtype=torch.float32)
        assert same(rk[0, :, :1], got[0][0, :, 69:]) and not rk[0, :, 1:].any() and not rk[1].any() and not rk[3:].any()


ATTN = [  # B, Hq, H, Dh, T, starts, counts, capacity
    (1, 2, 2, 64, 1, (0,), None, 1),                                        # one key
    (2, 3, 3, 64, 1, (256, 31), None, 300),
    (3, 4, 4, 32, 1, (0, 1, 127), (1, 0, 1), 130),                          # a padded row
    (2, 8, 2, 128, 1, (1000, 517), None, 1001),                             # four query heads to a cache head
    (1, 16, 2, 256, 1, (4000,), None, 4099),
    (1, 40, 2, 64, 1, (333,), None, 400),                                   # twenty of them
    (2, 2, 2, 128, 5, (0, 60), (5, 3), 70),                                 # a first chunk and a later, padded one
    (2, 4, 2, 64, 67, (130, -3), None, 200),                                # rows before the first key see nothing
    (1, 1, 1, 256, 33, (700,), (20,), 733),
    (1, 6, 1, 32, 19, (2 ** 20,), None, 90),                                # a start past the capacity: the whole cache is seen
]


@pytest.mark.parametrize("case", ATTN, ids=[str(i) for i in range(len(ATTN))])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_against_float64(case, bits, dtype):
    from branchgan import ops
    B, Hq, H, Dh, T, starts, counts, cap = case
    gen = torch.Generator().manual_seed(Dh + T + bits)
    k, v = make(gen, B, H, cap, Dh, dtype)
    layer = new_cache(B, H, cap, Dh, bits, fill=9)                          # codes and scales behind the last key: anything
    ops.kv_cache_append(layer, k.cuda(), v.cuda())
    q = torch.randn(B, Hq, T, Dh, generator=gen).to(dtype)
    kh, vh = O.held_values(k, bits), O.held_values(v, bits)
    ref, ref_lse = O.attention(q, kh, vh, starts, counts)
    out, lse = ops.kv_cache_attention(q.cuda(), layer, start=i32(*starts), counts=None if counts is None else i32(*counts))
    tol, rel = bound(q, kh, vh, 1 / math.sqrt(Dh), dtype, ref)
    assert out.dtype == dtype and out.shape == q.shape
    err = (out.cpu().double() - ref).abs()
    assert bool((err <= tol).all()), float((err / tol).max())
    seen = ref_lse > -math.inf
    assert bool((lse.cpu()[~seen] == -math.inf).all()) and not out.cpu()[~seen].any()
    assert bool(((lse.cpu().double() - ref_lse).abs()[seen] <= (rel + 2.0 ** -23 * (ref_lse.abs() + 8))[seen]).all())


FEW = [(1, 1), (2, 1), (1, 3), (3, 2), (8, 1), (1, 10), (16, 1), (4, 5)]     # query heads per cache head, new tokens


@pytest.mark.parametrize("G,T", FEW)
@pytest.mark.parametrize("Dh", [32, 64, 128, 256])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_few_rows_around_the_turns(G, T, Dh, bits, dtype):
    """Every shape of few-row tile, with sequences that end on, before and after a wave's 128 keys and a workgroup's 512."""
    from branchgan import ops
    gen = torch.Generator().manual_seed(G * 100 + T * 10 + Dh + bits)
    held = (1, 127, 128, 129, 512, 641)
    B, H = len(held), 1
    n = max(held) + T
    k, v = make(gen, B, H, n, Dh, dtype)
    layer = new_cache(B, H, n + 3, Dh, bits, fill=21)
    ops.kv_cache_append(layer, k.cuda(), v.cuda())
    q = torch.randn(B, G * H, T, Dh, generator=gen).to(dtype)
    kh, vh = O.held_values(k, bits), O.held_values(v, bits)
    start = tuple(x - 1 for x in held)
    ref, ref_lse = O.attention(q, kh, vh, start)
    tol, rel = bound(q, kh, vh, 1 / math.sqrt(Dh), dtype, ref)
    out, lse = ops.kv_cache_attention(q.cuda(), layer, start=i32(*start))
    assert within(out.cpu().double() - ref, tol) and within(lse.cpu().double() - ref_lse, rel + 2.0 ** -23 * (ref_lse.abs() + 8))
    # one sequence at a time: other splits of the key range, the same numbers within the bound
    for b in (0, 3, 5):
        one = ops.KVCacheLayer(layer.data[b:b + 1], bits, Dh, n + 3)
        o1, _ = ops.kv_cache_attention(q[b:b + 1].cuda(), one, start=i32(start[b]), max_keys=start[b] + T)
        assert within(o1.cpu().double() - ref[b:b + 1], tol[b:b + 1])


def test_scales_of_any_sign():
    from branchgan import ops
    gen = torch.Generator().manual_seed(23)
    for G, T in ((1, 1), (2, 20)):
        k, v = make(gen, 2, 2, 300, 64, torch.float32)
        layer = new_cache(2, 2, 300, 64, 4)
        ops.kv_cache_append(layer, k.cuda(), v.cuda())
        q = torch.randn(2, 2 * G, T, 64, generator=gen)
        kh, vh = O.held_values(k, 4), O.held_values(v, 4)
        for scale in (-0.2, 0.0, 1.0):
            ref, _ = O.attention(q, kh, vh, (150, 280), scale=scale)
            tol, _ = bound(q, kh, vh, abs(scale), torch.float32, ref)
            out, _ = ops.kv_cache_attention(q.cuda(), layer, start=i32(150, 280), scale=scale)
            assert within(out.cpu().double() - ref, tol), scale


def test_on_another_stream():
    """Append, read and attend on a side stream, ordered by events with the tensors' own: the same bits as on theirs."""
    from branchgan import ops
    gen = torch.Generator().manual_seed(24)
    k, v = [t.cuda() for t in make(gen, 2, 2, 1500, 64, torch.bfloat16)]
    q = torch.randn(2, 2, 1, 64, generator=gen).bfloat16().cuda()
    res = []
    for side in (None, torch.cuda.Stream()):
        layer = new_cache(2, 2, 1600, 64, 4)
        if side is not None:
            side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side or torch.cuda.current_stream()):
            ops.kv_cache_append(layer, k, v)
            res.append([*ops.kv_cache_attention(q, layer, start=i32(1499, 1203)), *ops.kv_cache_read(layer, 1500)])
        if side is not None:
            torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(*res))


def test_keys_behind_the_last_one_do_not_matter():
    """Stale scales of NaN and infinity behind the visible keys (an earlier, longer sequence) change nothing."""
    from branchgan import ops
    gen = torch.Generator().manual_seed(11)
    for bits, n in ((4, 77), (8, 128), (4, 400)):
        k, v = make(gen, 1, 2, 512, 64, torch.bfloat16)
        q = torch.randn(1, 2, 3, 64, generator=gen).bfloat16().cuda()
        clean, dirty = new_cache(1, 2, 512, 64, bits), new_cache(1, 2, 512, 64, bits)
        bad = k.clone()
        bad[:, :, n:] = math.nan
        ops.kv_cache_append(clean, k[:, :, :n].cuda(), v[:, :, :n].cuda())
        ops.kv_cache_append(dirty, bad.cuda(), bad.cuda())
        ops.kv_cache_append(dirty, k[:, :, :n].cuda(), v[:, :, :n].cuda())
        a, b = [ops.kv_cache_attention(q, c, start=i32(n - 3))[0] for c in (clean, dirty)]
        assert torch.equal(a, b) and bool(a.isfinite().all())


def test_nan_and_large_values_behave_as_in_the_plain_form():
    from branchgan import ops
    gen = torch.Generator().manual_seed(12)
    k, v = make(gen, 2, 1, 200, 64, torch.float32)
    k[0, 0, 50, 3], v[1, 0, 60, 40] = math.nan, math.inf                    # a broken key; a broken value (its 32 channels)
    layer = new_cache(2, 1, 200, 64, 4)
    ops.kv_cache_append(layer, k.cuda(), v.cuda())
    q = torch.randn(2, 1, 1, 64, generator=gen).cuda()
    out, _ = ops.kv_cache_attention(q, layer, start=i32(199, 199))
    assert bool(out[0].isnan().all()) and bool(out[1, ..., 32:].isnan().all()) and bool(out[1, ..., :32].isfinite().all())
    out, _ = ops.kv_cache_attention(q, layer, start=i32(49, 59))
    assert bool(out.isfinite().all())
    # scores far apart: only the largest counts; and huge equal scores
    k = torch.zeros(1, 1, 96, 32)
    k[0, 0, 70], k[0, 0, 10] = 3e4, -3e4
    v = torch.randn(1, 1, 96, 32, generator=gen)
    layer = new_cache(1, 1, 96, 32, 8)
    ops.kv_cache_append(layer, k.cuda(), v.cuda())
    out, _ = ops.kv_cache_attention(torch.ones(1, 1, 1, 32).cuda(), layer, start=i32(95), scale=1.0)
    assert torch.allclose(out[0, 0, 0].cpu().double(), O.held_values(v, 8)[0, 0, 70], rtol=2.0 ** -20)


def test_long_cache_past_32_bit_offsets():
    """One layer whose bytes pass 2^32: the last sequence is written and read where it belongs."""
    from branchgan import ops
    B, H, Dh, cap = 16, 16, 256, 64 * 1024
    gen = torch.Generator().manual_seed(13)
    layer = new_cache(B, H, cap, Dh, 4)
    nbytes = layer.data.numel()
    assert nbytes > 2 ** 32
    n = 300
    k, v = make(gen, 1, H, n, Dh, torch.bfloat16)
    kd, vd = k.cuda().expand(B, H, n, Dh), v.cuda().expand(B, H, n, Dh)
    s = cap - n
    ops.kv_cache_append(layer, kd, vd, start=i32(*[s] * B))
    rk, rv = ops.kv_cache_read(layer, n, start=i32(*[s] * B), dtype=torch.bfloat16)
    for b in (0, B - 1):
        assert same(rk[b], O.held_values(k[0], 4).bfloat16()) and same(rv[b], O.held_values(v[0], 4).bfloat16())
    # the keys before it are zeros: uniform weights over the zeros, and the values' share is exact arithmetic away
    q = torch.zeros(B, H, 1, Dh, device="cuda", dtype=torch.bfloat16)
    out, lse = ops.kv_cache_attention(q, layer, start=i32(*[cap - 1] * B))
    want = O.held_values(v, 4).sum(2) / cap
    tol = (cap * 2.0 ** -24 + 2.0 ** -16) * O.held_values(v, 4).abs().sum(2) / cap + 2.0 ** -8 * want.abs()
    assert within(out[B - 1, :, 0].cpu().double() - want[0], tol[0])
    assert torch.allclose(lse.cpu(), torch.full_like(lse.cpu(), math.log(cap)), rtol=1e-6)


def test_max_keys_and_strided_queries():
    from branchgan import ops
    gen = torch.Generator().manual_seed(14)
    B, H, T, Dh, n = 2, 4, 3, 64, 900
    k, v = make(gen, B, H, n, Dh, torch.bfloat16)
    layer = new_cache(B, H, 2048, Dh, 4)
    ops.kv_cache_append(layer, k.cuda(), v.cuda())
    kh, vh = O.held_values(k, 4), O.held_values(v, 4)
    packed = torch.randn(B, T, 3, H, Dh, generator=gen).bfloat16()
    q = packed[:, :, 0].permute(0, 2, 1, 3)
    starts = (n - T, 400)
    ref, _ = O.attention(q, kh, vh, starts)
    qd = packed.cuda()[:, :, 0].permute(0, 2, 1, 3)
    odd = torch.zeros(B, H, T, Dh + 1, dtype=torch.bfloat16)
    odd[..., 1:] = q
    tol, _ = bound(q, kh, vh, 0.125, torch.bfloat16, ref)
    for qq in (qd, odd.cuda()[..., 1:], qd.transpose(-1, -2).contiguous().transpose(-1, -2)):
        for mk in (None, n, 1024, 2048):
            out, _ = ops.kv_cache_attention(qq, layer, start=i32(*starts), max_keys=mk)
            assert within(out.cpu().double() - ref, tol)
    # keys past max_keys are not read
    out, _ = ops.kv_cache_attention(qd, layer, start=i32(*starts), max_keys=402)
    ref, _ = O.attention(q, kh[:, :, :402], vh[:, :, :402], (401, 400))
    assert within(out.cpu().double() - ref, tol + 2.0 ** -8 * ref.abs())


def test_streams_and_graph_replay():
    """Append and attend captured once, replayed as the sequence grows (start moves inside the graph), two graphs side by side."""
    from branchgan import kvcache, ops
    gen = torch.Generator().manual_seed(15)
    B, H, Dh, n0, steps = 2, 2, 128, 700, 5
    k, v = make(gen, B, H, n0 + steps, Dh, torch.bfloat16)
    q = torch.randn(B, H, steps, Dh, generator=gen).bfloat16()
    graphs = []
    for _ in range(2):
        layer = kvcache.QuantizedKVCache(1, B, H, 2048, Dh).layer(0)
        ops.kv_cache_append(layer, k[:, :, :n0].cuda(), v[:, :, :n0].cuda())
        io = [torch.zeros(B, H, 1, Dh, dtype=torch.bfloat16, device="cuda") for _ in range(3)]
        start = torch.full((B,), n0, dtype=torch.int32, device="cuda")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            ops.kv_cache_append(layer, io[1], io[2], start=start)
            out, lse = ops.kv_cache_attention(io[0], layer, start=start)
            start.add_(1)
        graphs.append((g, io, out, torch.cuda.Stream(), layer, start))      # the graph reads layer and start: they live as long as it
    kh, vh = O.held_values(k, 4), O.held_values(v, 4)
    ref, _ = O.attention(q, kh, vh, (n0, n0))
    tol, _ = bound(q, kh, vh, 1 / math.sqrt(Dh), torch.bfloat16, ref)
    for t in range(steps):
        for g, io, out, s, *_ in graphs:
            for dst, src in zip(io, (q, k[:, :, n0:], v[:, :, n0:])):
                dst.copy_(src[:, :, t:t + 1])
        torch.cuda.synchronize()
        for g, io, out, s, *_ in graphs:
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        torch.randn(1000, device="cuda").sum().item()                       # the program's own work in between
        for g, io, out, s, *_ in graphs:
            assert within(out[:, :, 0].cpu().double() - ref[:, :, t], tol[:, :, t]), t


def small_lm(family, seed=6):
    from branchgan import configs, models
    torch.manual_seed(seed)
    lm = models.make_lm(configs.LMConfig(family, 211, 128, 2, 4, 128)).cuda()
    with torch.no_grad():
        for p in lm.parameters():
            p.mul_(4.0) if p.dim() > 1 else None
    return lm


@pytest.mark.parametrize("family", ["gpt2", "gpt_neox"])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("fused_path", [True, False])
def test_generate_decodes_over_the_held_values(family, bits, fused_path, monkeypatch):
    """The tokens and log-probs of generate(cache_bits=) against forwards of the same model whose text keys / values are what the cache
    holds (read back in fp32, exact), attended by the branch attention kernel: the same numbers up to fp32 rounding."""
    from branchgan import fused, generate, kvcache, models, ops
    monkeypatch.setattr(fused, "ENABLED", fused_path)
    lm = small_lm(family)
    B, S, new = 3, 9, 40
    prompt = torch.randint(0, 211, (B, S), device="cuda")
    out, logp = generate.generate(lm, prompt, max_new_tokens=new, cache_bits=bits, return_logprobs=True)
    assert out.shape == (B, S + new) and logp.shape == (B, new) and logp.dtype == torch.float32 and torch.equal(out[:, :S], prompt)
    with torch.no_grad():
        first = lm(input_ids=prompt, use_cache=True, returnLmLogits=True)
        cache = kvcache.QuantizedKVCache(2, B, 4, S + new, 32, bits=bits)
        for l in range(2):
            ops.kv_cache_append(cache.layer(l), *first.past_key_values[l])
        logits, decisive_seen = first.logits[:, -1].float(), 0
        for t in range(new):
            tok = out[:, S + t:S + t + 1]
            lp = torch.log_softmax(logits, -1)
            torch.testing.assert_close(logp[:, t], lp.gather(1, tok)[:, 0], rtol=1e-3, atol=1e-3)
            top2 = logits.topk(2, dim=-1).values
            decisive = (top2[:, 0] - top2[:, 1]) > 1e-2
            decisive_seen += int(decisive.sum())
            assert torch.equal(tok[decisive, 0], logits.argmax(-1)[decisive]), t
            if t == new - 1:
                break
            start = torch.full((B,), S + t, dtype=torch.int32, device="cuda")
            over_cache = lm(input_ids=tok, position_ids=start.view(B, 1), textualPast=models.CachePast(cache, start, max_keys=S + t + 1),
                            returnLmLogits=True).logits[:, -1].float()
            text = [ops.kv_cache_read(cache.layer(l), S + t + 1, dtype=torch.float32) for l in range(2)]
            past = models.BranchPast(text=text, ancestors=[[], []], ctx_len=i32(S + t + 1), paths=[[]], n_query_nodes=1)
            logits = lm(input_ids=tok, position_ids=start.view(B, 1), textualPast=past, returnLmLogits=True).logits[:, -1].float()
            torch.testing.assert_close(over_cache, logits, rtol=1e-3, atol=1e-3 * float(logits.abs().max()))
    assert decisive_seen > B * new // 2
    # eight bits stay close to the unquantised decode's log-probs of the same tokens
    if bits == 8:
        with torch.no_grad():
            full = torch.log_softmax(lm(input_ids=out, returnLmLogits=True).logits[:, S - 1:-1].float(), -1).gather(-1, out[:, S:, None])[..., 0]
        assert float((full - logp).abs().mean()) < 0.1


def test_generate_with_cache_bits_keeps_its_options():
    from branchgan import generate
    lm = small_lm("gpt_neox")
    prompt = torch.randint(0, 211, (3, 9), device="cuda")
    g = lambda: torch.Generator(device="cuda").manual_seed(5)
    a, la = generate.generate(lm, prompt, max_new_tokens=12, do_sample=True, temperature=0.7, generator=g(), cache_bits=4, return_logprobs=True)
    b = generate.generate(lm, prompt, max_new_tokens=12, do_sample=True, temperature=0.7, generator=g(), cache_bits=4)
    assert torch.equal(a, b) and bool((la <= 0).all())
    # log-probs of the plain cache: the policy's own at the sampling temperature
    a, la = generate.generate(lm, prompt, max_new_tokens=12, do_sample=True, temperature=0.7, generator=g(), return_logprobs=True)
    assert torch.equal(a, generate.generate(lm, prompt, max_new_tokens=12, do_sample=True, temperature=0.7, generator=g()))
    with torch.no_grad():
        lp = torch.log_softmax(lm(input_ids=a, returnLmLogits=True).logits[:, 8:-1].float() / 0.7, -1).gather(-1, a[:, 9:, None])[..., 0]
    torch.testing.assert_close(la, lp, rtol=1e-3, atol=1e-3)
    # end of sequence: the tail is padding with log-prob 0
    greedy = generate.generate(lm, prompt, max_new_tokens=20, cache_bits=4)
    eos = int(greedy[0, 12])
    out, lp = generate.generate(lm, prompt, max_new_tokens=20, cache_bits=4, eos_token_id=eos, pad_token_id=0, return_logprobs=True)
    end = out[0, 9:].tolist().index(eos)
    assert not out[0, 9 + end + 1:].any() and not lp[0, end + 1:].any() and bool((lp[0, :end + 1] < 0).all())


def test_refusals():
    from branchgan import configs, generate, kvcache, models, ops
    for kw in (dict(bits=3), dict(head_dim=48), dict(capacity=0)):
        with pytest.raises(ValueError):
            kvcache.QuantizedKVCache(**{**dict(n_layers=1, batch=1, heads=1, capacity=8, head_dim=64), **kw})
    layer = new_cache(2, 2, 64, 64, 4)
    k = torch.zeros(2, 2, 5, 64, device="cuda")
    bad = [dict(k=k[:1], v=k[:1]), dict(k=k[..., :32], v=k[..., :32]), dict(k=k, v=k[:, :, :4]), dict(k=k, v=k.bfloat16()),
           dict(k=k, v=k, start=torch.zeros(2, dtype=torch.int64, device="cuda")), dict(k=k, v=k, counts=i32(1))]
    for kw in bad:
        with pytest.raises(ValueError):
            ops.kv_cache_append(layer, **kw)
    with pytest.raises(TypeError):
        ops.kv_cache_append(layer, k.half(), k.half())
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.kv_cache_append(layer, k.requires_grad_(), k)
    k = k.detach()
    for q, kw in ((k[..., :32], {}), (torch.zeros(2, 3, 1, 64, device="cuda"), {}), (k, dict(max_keys=65)), (k, dict(max_keys=0))):
        with pytest.raises(ValueError):
            ops.kv_cache_attention(q, layer, **kw)
    with pytest.raises(TypeError):
        ops.kv_cache_attention(k.half(), layer)
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.kv_cache_attention(k.clone().requires_grad_(), layer)
    with pytest.raises(ValueError):
        ops.KVCacheLayer(layer.data, 4, 64, 128)
    ops.kv_cache_append(layer, k[:, :, :0], k[:, :, :0])                     # nothing to write, nothing to attend: fine
    assert ops.kv_cache_attention(k[:, :, :0], layer)[0].shape == (2, 2, 0, 64)
    cfg = configs.LMConfig("gpt2", 64, 64, 1, 2, 32, attn_pdrop=0.1)
    with pytest.raises(NotImplementedError, match="dropout"):
        generate.generate(models.make_lm(cfg).cuda(), torch.zeros(1, 4, dtype=torch.long, device="cuda"), max_new_tokens=2, cache_bits=4)
