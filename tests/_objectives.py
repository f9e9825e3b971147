"""Plain 64-bit forms of the policy objectives, and the error bounds their kernels are held to."""
import math

import torch

U = 2.0 ** -24                      # half a step of float32, relative
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25}


def log_softmax(x):
    """64-bit log-softmax; a segment with every category closed gives -inf everywhere"""
    y = torch.log_softmax(x.double(), -1)
    return torch.where(torch.isneginf(x.double()).all(-1, keepdim=True), torch.full_like(y, -math.inf), y)


def softmax(x):
    p = torch.softmax(x.double(), -1)
    return torch.where(torch.isneginf(x.double()).all(-1, keepdim=True), torch.zeros_like(p), p)


def spread(x):
    """largest finite distance of a segment's logits from its maximum (the exponent's argument), [..., 1]"""
    d = x.double().amax(-1, keepdim=True) - x.double()
    return torch.where(torch.isfinite(d), d, torch.zeros_like(d)).amax(-1, keepdim=True)


def segment_bound(x):
    """Bound on the relative error of sum exp(x - max), and of one exp, in 32 bits.  exp(x - m): the difference and its product
    with log2(e) are rounded once each (2 u |x - m|), the instruction is off by at most a step (2 u).  The sum: at most 24 terms
    by one lane of a short axis and 7 additions across lanes; on a long axis (N > 1024) N / 256 terms by a thread and 18 steps
    of joins, each of them an addition, a product and an exp (counted 5 u)."""
    N = x.shape[-1]
    chain = 31 if N <= 1024 else N / 256 + 5 * 18 + 2 * N / 256
    one = 2 * spread(x) + 3
    return (one + chain) * U, one * U


def logprob(x, k):
    """-> logp [B], bound [B]"""
    N = x.shape[-1]
    inside = (k >= 0) & (k < N)
    lp = log_softmax(x).gather(-1, k.long().clamp(0, N - 1).unsqueeze(-1)).squeeze(-1)
    lp = torch.where(inside, lp, torch.zeros_like(lp))
    tot = lp.sum(-1)
    err = torch.where(inside, segment_bound(x)[0].squeeze(-1), torch.zeros_like(lp)).sum(-1)
    return tot, err + U * tot.abs() + 1e-37


def gradient(x, k, dlogp, derr=None):
    """-> gradient and its bound before the rounding to the logits' type.  dlogp (1[n = k] - p): p is off by the exp, the sum, the
    division and the product (3 u), the difference and the product with dlogp by u each."""
    N = x.shape[-1]
    inside = ((k >= 0) & (k < N) & ~torch.isneginf(x.double()).all(-1)).unsqueeze(-1)
    one = torch.zeros(x.shape, dtype=torch.float64, device=x.device).scatter_(-1, k.long().clamp(0, N - 1).unsqueeze(-1), 1.0)
    p = softmax(x)
    g = dlogp.double().view(-1, 1, 1)
    out = torch.where(inside, g * (one - p), torch.zeros_like(p))
    s_err, e_err = segment_bound(x)
    bound = g.abs() * (p * (s_err + e_err + 3 * U) + 2 * U * (one - p).abs())
    if derr is not None:
        bound = bound + derr.view(-1, 1, 1) * (one - p).abs()
    return out, torch.where(inside, bound, torch.zeros_like(bound))


def rounded(value, bound, dtype):
    """the bound after one rounding to `dtype`"""
    return bound + HALF_STEP[dtype] * (value.abs() + bound) + TINY[dtype]


def head(logp, old, adv, ref, w, lo, hi, c, stats=None, err=None):
    """-> dlogp, its bound for log-probs off by `err`, loss4 (64 bits).  The kernels take the differences of log-probs in 64 bits and
    round them once, the exponentials in 32: exp is off by |argument| u and a step (2 u), its product with the advantage by u;
    exp(d) - 1 by (|d| + 2) u exp(d) + u (|d| < 1: by its series, under 8 u of itself)."""
    a = adv.double()
    if stats is not None:
        s = stats.double()
        a = ((a - s[0]) * s[1]).clamp(s[2].item(), s[3].item())
    w = w.double() if w is not None else torch.full_like(logp, 1.0 / logp.shape[0])
    live = w != 0
    r = torch.exp(logp - old.double())
    sur, held = r * a, r.clamp(1 - lo, 1 + hi) * a
    clipped = held < sur
    pol = torch.where(clipped, -held, -sur)
    g = torch.where(clipped, torch.zeros_like(sur), -sur)
    kl = torch.zeros_like(r)
    lip = sur.abs()
    own = sur.abs() * ((logp - old.double()).abs() + 4) * U
    if ref is not None:
        d = ref.double() - logp
        kl = torch.expm1(d) - d
        g = g - c * torch.expm1(d)
        lip = lip + c * torch.exp(d)
        own = own + c * ((d.abs() + 3) * torch.exp(d) + 8 * torch.expm1(d).abs()) * U
    zero = torch.zeros_like(g)
    sums = [torch.where(live, w * t, zero).sum() for t in (pol + c * kl, pol, kl, clipped.double())]
    dlogp = torch.where(live, w * g, zero)
    bound = U * dlogp.abs() + torch.where(live, w.abs() * own, zero)
    if stats is not None:
        bound = bound + 3 * U * torch.where(live, w.abs() * sur.abs() * (1 + adv.double().abs() + stats.double()[0].abs()), zero)
    if err is not None:
        bound = bound + torch.where(live, 2 * w.abs() * lip * err, zero)
    return dlogp, bound, torch.stack(sums)


def preference(logp, offsets, ref, w, beta, smoothing, kind):
    T, P = logp.shape[0], offsets.shape[0] // 2
    gap = logp.double() - (ref.double() if ref is not None else 0.0)
    ww = w.double() if w is not None else torch.ones_like(gap)
    gap = torch.where(ww == 0, torch.zeros_like(gap), gap * ww)
    at = offsets.clamp(0, T).tolist()
    sums = torch.stack([gap[a:b].sum() for a, b in zip(at[:-1], at[1:])])
    delta = sums[0::2] - sums[1::2]
    m = beta * delta
    if kind == "logistic":
        loss = -(1 - smoothing) * torch.nn.functional.logsigmoid(m) - smoothing * torch.nn.functional.logsigmoid(-m)
        slope = beta * (smoothing * torch.sigmoid(m) - (1 - smoothing) * torch.sigmoid(-m))
    else:
        loss = (delta - 0.5 / beta) ** 2
        slope = 2 * (delta - 0.5 / beta)
    dlogp = torch.zeros_like(gap)
    for i in range(P):
        dlogp[at[2 * i]:at[2 * i + 1]] = slope[i] / P
        dlogp[at[2 * i + 1]:at[2 * i + 2]] = -slope[i] / P
    dlogp = torch.where(ww == 0, torch.zeros_like(dlogp), dlogp * ww)
    return dlogp, m, torch.stack([loss.mean(), (m > 0).double().mean(), m.mean()])


def balance(x, K, coef, mask=None):
    """-> loss, counts, mean_prob, gradient, bound of the gradient (before the rounding to the logits' type)"""
    R, A, N = x.shape
    keep = torch.ones(R, dtype=torch.bool, device=x.device) if mask is None else mask.bool()
    v = keep.view(-1, 1, 1)
    V = int(keep.sum())
    xd = torch.where(v, x.double(), torch.zeros((), dtype=torch.float64, device=x.device))
    order = torch.sort(xd, dim=-1, descending=True, stable=True)
    took = torch.zeros(R, A, N, dtype=torch.bool, device=x.device)
    took.scatter_(-1, order.indices[..., :K], torch.isfinite(order.values[..., :K]))
    counts = (took & v).sum(0)
    p = softmax(xd) * v
    share = counts.double() / (K * V) if V else torch.zeros(A, N, dtype=torch.float64, device=x.device)
    mean = p.sum(0) / max(V, 1)
    loss = coef * N / A * (share * mean).sum()
    scale = coef * N / (A * V) if V else 0.0
    dot = (share * p).sum(-1, keepdim=True)
    grad = scale * p * (share - dot)
    s_err, e_err = segment_bound(xd)
    rel = s_err + e_err + 6 * U
    # f and the dot are off by their own rounding each, the product by the error of p
    bound = abs(scale) * p * (rel * (share - dot).abs() + 2 * (rel + 34 * U) * dot + 2 * U * share)
    return loss, counts, mean, grad, bound
