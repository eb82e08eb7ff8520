"""The classifier losses in 64 bits, from their definitions (torch float64, on whatever device the inputs are).

Test infrastructure only.  With every result comes a bound of what a computation may be off that sums products in float32
in any order, takes exponentials in float32 to a few units in the last place and rounds its results, and the logits' gradient
before the gradients' products, to the operands' type."""
import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiniest(dtype):
    """Half the spacing of the type's smallest numbers."""
    return torch.finfo(dtype).smallest_normal * half_step(dtype)


def head(hidden, weight, labels, scale=1.0, smoothing=0.0, grad_loss=None, most=None, links=None):
    """loss, grad_hidden, grad_weight and a bound of each one's error (same shapes).  Of some rows of a longer batch, the bounds
    take the largest |grad_loss| of its counted rows (most) and the additions in a sum over its rows (links)."""
    dtype = hidden.dtype
    h, w = hidden.double(), weight.double()
    n, v, dim = h.shape[0], w.shape[0], h.shape[1]
    counted = (labels >= 0) & (labels < v)
    h = torch.where(counted[:, None], h, torch.zeros_like(h))
    at = labels.long().clamp(0, v - 1)[:, None]
    z = scale * (h @ w.t())
    off_z = (dim + 4) * U * scale * (h.abs() @ w.abs().t()) + 2 * U * z.abs()
    one = torch.zeros_like(z).scatter_(1, at, 1.0)
    # -log p of the label, and 1 - p, from the other classes: 1 - p itself would keep nothing of a sure row in 64 bits
    lse = torch.logsumexp(z, 1, keepdim=True)
    others = torch.logsumexp(torch.where(one > 0, -float("inf"), z), 1, keepdim=True)
    nll = torch.nn.functional.softplus(others - z.gather(1, at), threshold=1e300)
    p = (z - lse).exp()
    minus_target = torch.where(one > 0, -(others - lse).exp() + smoothing, p) - smoothing / v
    loss = ((1 - smoothing) * nll + smoothing * (lse - z.mean(1, keepdim=True)))[:, 0]
    # d loss = sum (p - target) dz, and the sums' own rounding
    off = (minus_target.abs() * off_z).sum(1) + off_z.amax(1) + 8 * U * (1 + loss.abs() + smoothing * z.abs().amax(1))
    loss = torch.where(counted, loss, torch.where(labels < 0, 0.0, float("nan")).double())
    g = torch.full((n,), 1.0 / max(n, 1), dtype=torch.float64, device=h.device) if grad_loss is None else grad_loss.double()
    c = (g * scale * counted)[:, None]
    d = minus_target * c
    # where p is the label's it is known by 1 - p; elsewhere by its logarithm
    spread = off_z.amax(1, keepdim=True)
    off_p = torch.where(one > 0, (1 - p), p) * (3 * spread + off_z + 16 * U).expm1() + 4 * U * smoothing
    off_d = off_p * c.abs()
    if dtype != torch.float32:
        off_d = off_d * (1 + 2 * half_step(dtype)) + half_step(dtype) * d.abs() + 2.0 ** -38 * (c.abs().amax() if most is None else most * scale)
    else:
        off_d = off_d + 4 * U * d.abs()
    gh, gw = d @ w, d.t() @ h
    off_h = off_d @ w.abs() + (v + 8) * U * ((d.abs() + off_d) @ w.abs())
    off_w = off_d.t() @ h.abs() + (n + 8 if links is None else links) * U * ((d.abs() + off_d).t() @ h.abs())
    off_h = off_h * (1 + 2 * half_step(dtype)) + half_step(dtype) * gh.abs() + tiniest(dtype)
    off_w = off_w * (1 + 2 * half_step(dtype)) + half_step(dtype) * gw.abs() + tiniest(dtype)
    return (loss, gh, gw), (off, off_h, off_w)


def distill(logits, values, index, tau=1.0, lse=None, grad_loss=None):
    """loss, grad and a bound of each one's error."""
    dtype = logits.dtype
    n, v = logits.shape
    u = logits.double() / tau
    entry = (index >= 0) & (index < v) & (values != -float("inf"))
    has = entry.any(1)
    at = torch.where(entry, index.long(), 0)
    t = torch.where(entry, values.double() / tau, -float("inf"))
    logp = torch.log_softmax(u, 1)
    if lse is None:
        whole = torch.logsumexp(torch.where(has[:, None], t, 0.0), 1)
    else:
        whole = lse.double()
    logq = t - whole[:, None]
    q = torch.where(entry, logq.exp(), 0.0)
    lq, lp = torch.where(q > 0, logq, 0.0), torch.where(q > 0, logp.gather(1, at), 0.0)
    terms = q * (lq - lp)
    loss, size = terms.sum(1), (q * (1 + lq.abs() + lp.abs())).sum(1)
    p = logp.exp()
    away = torch.zeros_like(p).scatter_add_(1, at, q)
    inside = torch.zeros_like(p).scatter_add_(1, at, entry.double()) > 0
    total = q.sum(1, keepdim=True)
    d = p * total - away
    part = p * total + away
    if lse is not None:
        other = torch.where(inside, 0.0, p)
        rest_q = (1 - total).clamp(min=0)
        ln_p = torch.logsumexp(torch.where(inside, -float("inf"), logp), 1)[:, None]
        # a float32 log-sum-exp says no more of 1 - Q than this; where the student has nothing either, that is nothing
        empty = (ln_p < -104) & (rest_q <= 2.0 ** -20 * (1 + whole.abs()[:, None]))
        use = (~inside).any(1, keepdim=True) & ~empty
        rest = torch.where(use & (rest_q > 0), rest_q * (torch.log(rest_q.clamp(min=1e-300)) - ln_p), 0.0)
        loss, size = loss + rest[:, 0], size + (rest.abs() + 2 * rest_q * use)[:, 0]
        # the classes' shares of the bucket; where the student has none of it, none
        share = torch.softmax(torch.where(inside, -float("inf"), u), 1)
        share = torch.where(inside | (ln_p == -float("inf")) | ~use, 0.0, share)
        d = p * (total + rest_q * use) - away - share * rest_q
        # q_r = 1 - Q is off by what Q is: by 2^-23 of the share at most, which the bucket's classes pass on
        part = p * (total + rest_q * use) + away + share * (1 + rest_q)
    g = torch.full((n,), 1.0 / max(n, 1), dtype=torch.float64, device=u.device) if grad_loss is None else grad_loss.double()
    loss = torch.where(has, loss, 0.0) * tau ** 2
    d = torch.where(has[:, None], d, 0.0) * (g * tau)[:, None]
    # exponentials of (z - max) log2(e) / tau: the product is rounded, so a value is off by its exponent times U
    far = (u.amax(1, keepdim=True) - u).clamp(max=200)
    far = torch.where(torch.isfinite(far), far, 200.0)
    off_d = part * (g.abs() * tau)[:, None] * U * (24 + 4 * far) + half_step(dtype) * d.abs() + tiniest(dtype)
    deep = torch.where(q > 0, (whole[:, None] - t).abs().clamp(max=200), 0.0).amax(1)
    off = tau ** 2 * U * (40 + 4 * deep) * (size + 1)
    return (loss, d), (off, torch.where(has[:, None], off_d, tiniest(dtype)))
