"""Oracle: the clipped policy loss with a KL term, float64, differentiable (test infrastructure; no counterpart in the reference)."""
import torch


def policy_loss(logits, ids, old_logp, advantages, weights=None, ref_logp=None, ref_logits=None, clip_low=0.2, clip_high=0.2, kl_coef=0.0,
                temperature=1.0, denominator=None):
    """-> (loss, logp (rows), kl (rows)); logits (rows, V) float64.  Rows of weight 0 or with an id outside the vocabulary do not count."""
    V = logits.shape[-1]
    w = torch.ones(logits.shape[0], dtype=torch.float64) if weights is None else weights.double()
    w = torch.where((ids >= 0) & (ids < V), w, torch.zeros_like(w))
    rows = (w != 0).nonzero()[:, 0]
    logp, kl = torch.zeros_like(w), torch.zeros_like(w)
    total = logits.sum() * 0 if rows.numel() == 0 else 0
    for r in rows.tolist():
        lp = torch.log_softmax(logits[r] / temperature, -1)
        tok = lp[ids[r]]
        ratio = torch.exp(tok - old_logp[r].double())
        a = advantages[r].double()
        term = torch.maximum(-a * ratio, -a * ratio.clamp(1 - clip_low, 1 + clip_high))
        if ref_logits is not None:
            lq = torch.log_softmax(ref_logits[r].double() / temperature, -1)
            seen = lp > -torch.inf
            k = (lp[seen].exp() * (lp[seen] - lq[seen])).sum()
        elif ref_logp is not None:
            d = ref_logp[r].double() - tok
            k = torch.exp(d) - d - 1
        else:
            k = torch.zeros((), dtype=torch.float64)
        total = total + w[r] * (term + kl_coef * k)
        logp[r], kl[r] = tok.detach(), k.detach()
    n = float(w.sum()) if denominator is None else float(denominator)
    return (total / n if n != 0 else total * 0), logp, kl
