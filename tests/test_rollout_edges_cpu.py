"""No-GPU checks of the quantised cache and the policy loss at their edges: what the wrappers hand to the library."""
import pytest
import torch

B, T, V = 3, 4, 1031


def test_live_tokens():
    from branchgan import generate
    ids = torch.tensor([[5, 2, 0, 0, 0], [2, 2, 2, 2, 2], [1, 3, 4, 5, 6], [0, 0, 7, 2, 9], [1, 1, 1, 1, 2]])
    want = torch.tensor([[1, 1, 0, 0, 0], [1, 0, 0, 0, 0], [1, 1, 1, 1, 1], [1, 1, 1, 1, 0], [1, 1, 1, 1, 1]]).bool()
    assert torch.equal(generate.liveTokens(ids, 2), want) and generate.liveTokens(ids, None).all() and generate.liveTokens(ids[:, :0], 2).shape == (5, 0)


def policy_calls(monkeypatch):
    """ops.policy_loss without its launches: the shape structs that the calls got, copied."""
    from branchgan import _capi, ops
    calls = []
    def record(name, device, entry, sh, x, y, *rest):
        calls.append((name, _capi.PolicyShape.from_buffer_copy(sh._obj), x))
    monkeypatch.setattr(ops, "_launch", record)
    monkeypatch.setattr(ops.C, "require_cuda", lambda *t: None)
    return calls


def test_a_kl_weight_without_a_reference_is_told(monkeypatch, recwarn):
    from branchgan import ops
    policy_calls(monkeypatch)
    x = [torch.zeros(4, V), torch.zeros(4, dtype=torch.long), torch.zeros(4), torch.zeros(4)]
    ops.policy_loss(*x)
    ops.policy_loss(*x, ref_logp=torch.zeros(4), kl_coef=0.1)
    ops.policy_loss(*x, ref_logits=x[0], kl_coef=0.1)
    assert not [w for w in recwarn if "KL" in str(w.message)]
    with pytest.warns(UserWarning, match="no KL term"):
        ops.policy_loss(*x, kl_coef=0.1)


@pytest.mark.parametrize("with_ref", [False, True])
def test_each_backward_walks_the_layout_that_the_hooks_returned(monkeypatch, with_ref):
    """Saved-tensor hooks that answer dense, as saved, dense again: every call's strides are those of the tensors it was given."""
    from branchgan import ops
    calls = policy_calls(monkeypatch)
    full, ref = [torch.zeros(B, 9, V) for _ in range(2)]
    x = full.requires_grad_(True)
    rows = [torch.zeros(B, T, dtype=torch.long), torch.zeros(B, T), torch.zeros(B, T)]
    returned, dense = [], [False]
    def unpack(t):
        t = t.contiguous().clone() if dense[0] and t.dim() == 3 else t
        returned.append(t)
        return t
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        loss = ops.policy_loss(x[:, 2:6], *rows, ref_logits=ref[:, 2:6] if with_ref else None)[0]
    for dense[0] in (True, False, True):
        returned.clear()
        torch.autograd.grad(loss, x, retain_graph=True)
        name, sh, address = calls[-1]
        logits = [t for t in returned if t.dim() == 3]
        assert name == "bg_policy_loss_bwd" and address == logits[0].data_ptr()
        assert (sh.x_stride, sh.x_outer) == (V, (T if dense[0] else 9) * V) == (logits[0].stride(1), logits[0].stride(0))
        if with_ref:
            assert (sh.ref_stride, sh.ref_outer) == (logits[1].stride(1), logits[1].stride(0))
        assert (sh.inner, sh.d_outer, sh.rows) == (calls[0][1].inner, calls[0][1].d_outer, B * T)
