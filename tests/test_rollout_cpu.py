"""No-GPU checks of the quantised cache and the policy loss: the library's refusals before any launch, the size query, the oracles
against independent forms and differences, and the Python entry points' refusal of CPU tensors."""
import ctypes
import math

import pytest
import torch

from oracle import kvcache as OK
from oracle import policy as OP


def cache_struct(**kw):
    from branchgan import _capi
    c = _capi.KvCache()
    d = dict(bits=4, B=1, H=2, Dh=64, capacity=100)
    d.update(kw)
    tile = _capi.lib().bg_kv_cache_tile_bytes(d["bits"], d["Dh"])
    c.c_sh, c.c_sb = 4 * tile, 8 * tile
    for k, v in d.items():
        setattr(c, k, v)
    return c


def test_tile_bytes():
    from branchgan import _capi
    f = _capi.lib().bg_kv_cache_tile_bytes
    for Dh in (32, 64, 128, 256):
        assert f(4, Dh) == 2 * 32 * (Dh // 2 + Dh // 32 * 2) and f(8, Dh) == 2 * 32 * (Dh + Dh // 32 * 2)
    assert f(3, 64) == 0 and f(4, 48) == 0 and f(16, 64) == 0 and f(4, 0) == 0


def test_cache_calls_refuse_before_any_launch():
    from branchgan import _capi
    lib = _capi.lib()
    p = ctypes.c_void_p(1 << 20)                      # never dereferenced on the host; the calls are refused before a launch
    def append(c, data=p, k=p, v=p, dtype=1, T=3):
        return lib.bg_kv_cache_append(ctypes.byref(c), data, k, v, dtype, T, 0, 0, 64, 0, 0, 64, None, None, None)
    def read(c, data=p, k=p, v=p, dtype=1, T=3):
        return lib.bg_kv_cache_read(ctypes.byref(c), data, k, v, dtype, T, 0, 0, 64, None, None, None)
    def attn(c, data=p, q=p, dtype=1, Hq=2, T=1, max_keys=100, out=p):
        return lib.bg_kv_cache_attn_fwd(ctypes.byref(c), data, q, dtype, Hq, T, 0, 0, 64, None, None, max_keys, 1.0, out, 0, 0, 64, None, None, 0, None)
    for f in (append, read, attn):
        for bad, word in ((dict(bits=5), b"bits=5"), (dict(Dh=96), b"Dh=96"), (dict(B=0), b"B=0"), (dict(capacity=0), b"capacity=0"),
                          (dict(capacity=1 << 30), b"capacity"), (dict(c_sh=16), b"overlap"), (dict(c_sb=8), b"16-byte")):
            assert f(cache_struct(**bad)) == 1 and word in lib.bg_last_error(), (f, bad, lib.bg_last_error())
        assert f(cache_struct(), data=None) == 1 and b"null" in lib.bg_last_error()
        assert f(cache_struct(), data=ctypes.c_void_p(8)) == 1 and b"16-byte" in lib.bg_last_error()
        assert f(cache_struct(), dtype=2) == 1 and b"dtype" in lib.bg_last_error()
        assert f(cache_struct(), T=0) == 1
    assert append(cache_struct(), k=None) == 1 and read(cache_struct(), v=None) == 1 and attn(cache_struct(), q=None) == 1
    assert attn(cache_struct(), Hq=3) == 1 and b"Hq=3" in lib.bg_last_error()
    assert attn(cache_struct(), max_keys=101) == 1 and b"max_keys=101" in lib.bg_last_error()
    assert attn(cache_struct(), max_keys=0) == 1


def test_caches_whose_heads_and_sequences_interleave_are_refused():
    """Strides that keep neighbours apart and still let (1, 0) and (0, 1) share bytes; the two orders that do not are taken (as far
    as the next check, here a missing output)."""
    from branchgan import _capi
    lib = _capi.lib()
    p = ctypes.c_void_p(1 << 20)
    bytes_ = -(-100 // 32) * lib.bg_kv_cache_tile_bytes(4, 64)
    def read(c_sb, c_sh):
        c = cache_struct(B=3, H=4, c_sb=c_sb, c_sh=c_sh)
        rc = lib.bg_kv_cache_read(ctypes.byref(c), p, None, None, 1, 3, 0, 0, 64, None, None, None)
        assert rc == 1
        return lib.bg_last_error()
    for sb, sh in ((bytes_, bytes_), (2 * bytes_, bytes_), (4 * bytes_ - 16, bytes_), (bytes_, 3 * bytes_ - 16), (5 * bytes_, 2 * bytes_)):
        assert b"overlap" in read(sb, sh), (sb, sh)
    for sb, sh in ((4 * bytes_, bytes_), (bytes_, 3 * bytes_), (7 * bytes_, 2 * bytes_), (4 * bytes_ + 64, bytes_)):
        assert b"null k / v" in read(sb, sh), (sb, sh)


def test_policy_calls_refuse_before_any_launch():
    from branchgan import _capi
    lib = _capi.lib()
    p = ctypes.c_void_p(1 << 20)
    def shape(**kw):
        s = _capi.PolicyShape()
        d = dict(dtype=0, rows=4, V=50, x_stride=50, ref_stride=50, temperature=1.0, clip_low=0.2, clip_high=0.2, kl_coef=0.0)
        d.update(kw)
        for k, v in d.items():
            setattr(s, k, v)
        return s
    def fwd(s, logits=p, ref=None, ref_logp=None, stats=p):
        return lib.bg_policy_loss_fwd(ctypes.byref(s), logits, ref, p, p, ref_logp, p, None, None, p, p, p, stats, None, None, None)
    def bwd(s, logits=p, ref=None, stats=p):
        return lib.bg_policy_loss_bwd(ctypes.byref(s), logits, ref, p, stats, p, p, 0, None)
    for f in (fwd, bwd):
        for bad, word in ((dict(dtype=3), b"dtype 3"), (dict(rows=0), b"rows=0"), (dict(V=0), b"V=0"), (dict(x_stride=49), b"stride=49"),
                          (dict(temperature=0.0), b"temperature"), (dict(temperature=math.nan), b"temperature"), (dict(clip_low=-1.0), b"clip range"),
                          (dict(clip_high=math.nan), b"clip range")):
            assert f(shape(**bad)) == 1 and word in lib.bg_last_error(), (bad, lib.bg_last_error())
        assert f(shape(), logits=None) == 1 and b"null" in lib.bg_last_error()
        assert f(shape(), stats=ctypes.c_void_p(4)) == 1
        assert f(shape(ref_stride=10), ref=p) == 1 and b"reference stride" in lib.bg_last_error()
    assert fwd(shape(), ref=p, ref_logp=p) == 1 and b"exclude" in lib.bg_last_error()


def test_python_entry_points_refuse_cpu_tensors():
    from branchgan import ops
    layer = ops.KVCacheLayer(torch.zeros(1, 2, 4 * 32 * 72, dtype=torch.uint8), 4, 64, 128)
    x = torch.zeros(1, 2, 1, 64)
    for call in (lambda: ops.kv_cache_append(layer, x, x), lambda: ops.kv_cache_read(layer, 1), lambda: ops.kv_cache_attention(x, layer),
                 lambda: ops.policy_loss(torch.zeros(2, 5), torch.zeros(2, dtype=torch.long), torch.zeros(2), torch.zeros(2))):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
    for kw in (dict(bits=2), dict(head_dim=80), dict(capacity=0), dict(capacity=200)):
        with pytest.raises(ValueError):
            ops.KVCacheLayer(**{**dict(data=layer.data, bits=4, head_dim=64, capacity=128), **kw})


@pytest.mark.parametrize("bits", [4, 8])
def test_held_values_are_close_and_repeatable(bits):
    x = torch.randn(3, 5, 64, generator=torch.Generator().manual_seed(bits))
    y = OK.held_values(x, bits)
    top = 7 if bits == 4 else 127
    a = x.abs().unflatten(-1, (2, 32)).amax(-1, keepdim=True).double()
    step = a / top * (1 + 2.0 ** -8)                                         # the scale's own rounding included
    # at most half a step off, the largest magnitude by what the scale's rounding takes off it
    assert bool(((y - x.double()).abs().unflatten(-1, (2, 32)) <= torch.maximum(step / 2, a * 2.0 ** -8) * (1 + 1e-9)).all())
    again = OK.held_values(y, bits)                                          # what is held is held again as the same numbers, or its scale moved by one rounding
    assert bool(((again - y).abs() <= 2.0 ** -7 * a.expand(3, 5, 2, 32).flatten(-2)).all())


def test_policy_oracle_gradient_against_differences():
    g = torch.Generator().manual_seed(0)
    rows, V = 5, 7
    x = torch.randn(rows, V, dtype=torch.float64, generator=g).requires_grad_(True)
    ids = torch.tensor([0, 6, 3, -1, 2])
    old = torch.log_softmax(x.detach(), -1).gather(1, ids.clamp(min=0)[:, None])[:, 0] + torch.tensor([0.1, -0.5, 0.5, 0.0, -0.1])
    adv = torch.tensor([1.0, 2.0, -1.5, 1.0, -0.3])
    ref = torch.randn(rows, V, dtype=torch.float64, generator=g)
    for kw in (dict(), dict(ref_logits=ref), dict(ref_logp=old - 0.2)):
        assert torch.autograd.gradcheck(lambda t: OP.policy_loss(t, ids, old, adv, kl_coef=0.3, temperature=0.8, **kw)[0], (x,))


def test_policy_row_groups_refuse_before_any_launch():
    from branchgan import _capi
    lib = _capi.lib()
    p = ctypes.c_void_p(1 << 20)
    def fwd(ref=None, **kw):
        sh = _capi.PolicyShape(1, 0, 12, 100, 100, 100 if ref else 0, 1.0, 0.2, 0.2, 0.1, 4, 500, 500 if ref else 0, 400)
        for k, v in kw.items():
            setattr(sh, k, v)
        # a missing output is what a shape that is accepted stumbles over
        rc = lib.bg_policy_loss_fwd(ctypes.byref(sh), p, ref, p, p, None, p, None, None, None, p, p, p, None, None, None)
        assert rc == 1
        return lib.bg_last_error()
    for kw in (dict(inner=5), dict(inner=-1), dict(x_outer=-1), dict(ref=p, ref_outer=-1), dict(d_outer=399)):
        assert b"group" in fwd(**kw), (kw, lib.bg_last_error())
    for kw in (dict(), dict(inner=0, d_outer=0, x_outer=-1), dict(inner=12, d_outer=0, x_outer=-1), dict(x_outer=0), dict(ref=p)):
        assert b"null argument" in fwd(**kw), (kw, lib.bg_last_error())


def test_calls_of_more_threads_than_a_launch_has_are_refused():
    from branchgan import _capi
    lib = _capi.lib()
    p = ctypes.c_void_p(1 << 20)
    sh = _capi.PolicyShape(1, 0, 1 << 22, 16, 16, 0, 1.0, 0.2, 0.2, 0.1, 0, 0, 0, 0)
    assert lib.bg_policy_loss_fwd(ctypes.byref(sh), p, None, p, p, None, p, None, None, p, p, p, p, None, None, None) == 1 and b"rows" in lib.bg_last_error()
    tile = lib.bg_kv_cache_tile_bytes(4, 32)
    wide = cache_struct(B=60000, H=60000, Dh=32, capacity=1, c_sh=tile, c_sb=60000 * tile)
    for T in (1, 2):
        assert lib.bg_kv_cache_append(ctypes.byref(wide), p, p, p, 1, T, 0, 0, 32, 0, 0, 32, None, None, None) == 1 and b"blocks" in lib.bg_last_error()
        assert lib.bg_kv_cache_read(ctypes.byref(wide), p, p, p, 1, T, 0, 0, 32, None, None, None) == 1 and b"blocks" in lib.bg_last_error()
    c = cache_struct(H=1, capacity=1)
    assert lib.bg_kv_cache_attn_fwd(ctypes.byref(c), p, p, 1, 1, (1 << 28) + 1, 0, 0, 64, None, None, 1, 1.0, p, 0, 0, 64, None, None, 0, None) == 1
    assert b"rows" in lib.bg_last_error()
