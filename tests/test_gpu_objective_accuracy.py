"""GPU: the policy objectives where terms cancel or grow large, against 64-bit forms, within bounds derived from the arithmetic."""
import math

import pytest
import torch

from _objectives import U, balance, gradient, head, logprob, preference, rounded, segment_bound, softmax
from test_gpu_objectives import SHAPES, close, make_logits, objective

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def between(got, want, bound):
    """one rounding to the type of `got` of a value within `bound` of `want`: rounding keeps order, so it lies between the roundings
    of the two ends"""
    lo, hi = (want - bound).to(got.dtype), (want + bound).to(got.dtype)
    return (got >= lo) & (got <= hi)


# ---- balance loss: shares that are nearly equal -----------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,A,N,K", [(64003, 1, 8, 1), (30011, 3, 35, 1), (20007, 1, 128, 8), (9001, 2, 300, 4)])
def test_balance_gradient_of_nearly_equal_counts(dev, R, A, N, K, dtype):
    """every category is chosen by as many rows as the next, one or two apart: the gradient is what is left of shares that agree in
    all their leading digits"""
    from pfpn_amd import kernels
    g = torch.Generator(device=dev)
    g.manual_seed(N)
    x = (0.5 * torch.randn(R, A, N, device=dev, generator=g)).clamp(-2, 2)
    r, a = torch.arange(R, device=dev).view(R, 1, 1), torch.arange(A, device=dev).view(1, A, 1)
    x.scatter_add_(-1, (r * K + a + torch.arange(K, device=dev).view(1, 1, K)) % N, torch.full((R, A, K), 5.0, device=dev))
    x = x.to(dtype)
    coef = 1e7                  # (a float16 gradient stays above that type's smallest step)
    _, counts, _, grad, _ = balance(x, K, coef)
    assert 0 < int(counts.max() - counts.min()) <= 2
    got = kernels.balance_loss(x, topk=K, coef=coef)
    assert torch.equal(got[1].long(), counts.long())
    # f less its least entry is whole numbers of coef N / (A K R^2): rounded once (u).  p is off by s_err + e_err and 6 u (division,
    # product, difference), the dot by that and 34 roundings of its sum: no term in u times the share itself
    p, f = softmax(x), coef * N / (A * K) / R / R * (counts - counts.amin(-1, keepdim=True)).double()
    dot = (p * f).sum(-1, keepdim=True)
    s_err, e_err = segment_bound(x)
    rel = s_err + e_err + 6 * U
    bound = p * (rel * (f - dot).abs() + (rel + 36 * U) * dot + 2 * U * f)
    assert float((p * (f - dot) - grad).abs().max()) < 1e-9 * float(grad.abs().max())       # (the two 64-bit forms agree)
    ok = between(got[3], grad, bound)
    assert bool(ok.all()), "%d of %d entries, off by up to %.3g of the bound" % (
        int((~ok).sum()), ok.numel(), float(((got[3].double() - grad).abs() / bound).masked_fill(ok, 0).max()))


def test_balance_means_of_many_equal_rows(dev):
    """2^24 rows of one fresh policy: equal weights, whose 32-bit sums round to one side"""
    from pfpn_amd import kernels
    gap = torch.tensor([0.125, 0.296875, 0.5, 0.703125, 1.296875, 1.5, 1.703125, 2.296875], device=dev)
    row = torch.stack([gap, torch.zeros_like(gap)], -1).bfloat16()
    x = row.expand(1 << 24, 8, 2).contiguous()
    loss, counts, mean, _ = kernels.balance_loss(x)
    want = torch.softmax(row.double(), -1)
    assert counts[:, 0].tolist() == [1 << 24] * 8 and not counts[:, 1].any()
    # a weight is off by its exponential, sum and quotient (12 u at these gaps); a lane adds 257 of them at most, a block its 18 rows
    # of lanes; the chunks are added in 64 bits and rounded once
    bound = (12 + 257 + 18 + 1) * U
    assert float(((mean.double() - want).abs() / want).max()) <= bound
    assert abs(float(loss) - float(2 / 8 * want[:, 0].sum())) <= bound * float(loss)


def test_balance_loss_can_be_less_than_its_coefficient(dev):
    """three rows of five at weights (0.51, 0.49), two at (0, 1): shares (0.6, 0.4) of means (0.306, 0.694), 2 (0.6 x 0.306 + 0.4 x 0.694)"""
    from pfpn_amd import kernels
    x = torch.tensor([[math.log(0.51), math.log(0.49)]] * 3 + [[-math.inf, 0.0]] * 2, device=dev).unsqueeze(1)
    loss, counts, mean, _ = kernels.balance_loss(x, coef=0.5)
    assert counts.tolist() == [[3, 2]] and abs(float(loss) - 0.5 * 0.9224) < 1e-6
    # equal shares, or equal mean weights: the coefficient
    assert abs(float(kernels.balance_loss(x[[0, 3]], coef=0.5)[0]) - 0.5) < 1e-6
    even = torch.tensor([[0.9, 0.1], [0.45, 0.55], [0.15, 0.85]], device=dev).log().unsqueeze(1)
    assert abs(float(kernels.balance_loss(even, coef=0.5)[0]) - 0.5) < 1e-6


# ---- clipped loss with a KL term: log-probs that lie far apart ------------------------------------------------------------------------
def far_head(logp, old, adv, ref, w, eps, c, err=0.0):
    """-> dlogp, its bound, loss4 and its bound, in 64 bits.  The kernels' differences, exponentials and products are 64-bit; the series of
    the KL term (|d| < 1) has a 32-bit sum: 4 u of itself.  `err`: what the log-prob itself is off by.  A row of advantage 0 has no
    surrogate, however large its ratio."""
    a, w = adv.double(), w.double()
    r = torch.exp(logp - old.double())
    sur = torch.where(a == 0, torch.zeros_like(r), r * a)
    held = r.clamp(1 - eps, 1 + eps) * a
    clipped = held < sur
    d = ref.double() - logp
    em1, kl = torch.expm1(d), torch.expm1(d) - d
    pol, g = torch.where(clipped, -held, -sur), torch.where(clipped, torch.zeros_like(sur), -sur)
    dlogp = w * (g - c * em1)
    series = torch.where(d.abs() < 1, kl, torch.zeros_like(kl)).abs()
    slack = w * ((g.abs() + c * (em1.abs() + 1)) * (1.01 * err) + 4 * U * c * series) + 1e-14 * w * (g.abs() + c * em1.abs())
    loss4 = torch.stack([(w * t).sum() for t in (pol + c * kl, pol, kl, clipped.double())])
    part = w * (g.abs() * (1.01 * err) + 4 * U * series) + w * (1.01 * err) * em1.abs() + 1e-14 * w * (pol.abs() + kl)
    off = torch.stack([part.sum() * (1 + c), part.sum(), part.sum(), 1e-14 * w.sum()])
    return dlogp, U * dlogp.abs() + slack + 1e-45, loss4, U * loss4.abs() + off + 1e-45


GAPS = [-100.0, -88.0, -3.0, -0.25, 0.0, 2.0 ** -7, 0.25, 3.0, 60.0, 88.0, 90.0, 100.0]


def test_far_log_probs(dev):
    """every gap to the old policy with every gap to the reference, under advantages of both signs and none; weights small enough
    that ratios of e^100 leave finite sums"""
    from pfpn_amd import kernels
    gap, ref, adv = [t.reshape(-1) for t in torch.meshgrid(torch.tensor(GAPS), torch.tensor(GAPS), torch.tensor([0.0, 1.5, -0.7]),
                                                          indexing="ij")]
    logp = torch.full_like(gap, -256.0)
    old, ref, w = logp - gap, logp + ref, torch.full_like(gap, 1e-20)
    # ... and gaps whose ratio no 64-bit number holds, or that are infinite: clipped, or without an advantage
    extra = torch.tensor([[-256.0, -2000.0, -256.0, 0.0, 1e-20], [-256.0, -2000.0, -256.0, 2.0, 1e-20],
                          [-256.0, -math.inf, -256.0, 0.0, 1e-20], [-256.0, -math.inf, -256.0, 2.0, 1e-20],
                          [-256.0, 1000.0, -256.0, -1.0, 1e-20], [-256.0, -256.0, -2000.0, 1.0, 1e-20]]).t()
    logp, old, ref, adv, w = [torch.cat([t, e]).to(dev) for t, e in zip((logp, old, ref, adv, w), extra)]
    for n in (logp.shape[0], 5000):            # (one block, which finishes the sums itself, and many)
        args = [t.repeat(n // logp.shape[0] + 1)[:n].contiguous() for t in (logp, old, adv, ref, w)]
        want, bound, loss4, off = far_head(args[0].double(), args[1], args[2], args[3], args[4], 0.2, 0.05)
        assert torch.isfinite(want).all() and torch.isfinite(loss4).all()
        dlogp, l4 = kernels.policy_kl_loss(args[0], args[1], args[2], logp_ref=args[3], weight=args[4], kl_coef=0.05)
        assert bool(((dlogp.double() - want).abs() <= bound).all())
        assert bool(((l4.double() - loss4).abs() <= off).all())
    # a NaN is not covered up by an advantage of zero
    bad = torch.tensor([math.nan, -1.0], device=dev)
    d, l4 = kernels.policy_kl_loss(bad, torch.zeros(2, device=dev), torch.zeros(2, device=dev))
    assert d[0].isnan() and d[1] == 0 and l4[0].isnan()


def test_rows_without_advantage_under_a_one_sided_clip(dev):
    """no upper bound on the ratio, an impossible old choice, no advantage: nothing, not inf * 0"""
    from pfpn_amd import kernels
    old, adv = torch.tensor([-math.inf, -2000.0, -1.0, -1.0], device=dev), torch.tensor([0.0, 0.0, 0.0, 2.0], device=dev)
    d, l4 = kernels.policy_kl_loss(torch.full((4,), -1.0, device=dev), old, adv, clip_eps=(0.2, math.inf))
    assert d.tolist() == [0.0, 0.0, 0.0, -0.5] and l4.tolist() == [-0.5, -0.5, 0.0, 0.0]


@pytest.mark.parametrize("shape", [(36, 40, 8), (36, 2, 300), (36, 1, 5000), (600, 1, 1500), (5, 3, 1100), (3, 1, 70001)])
def test_far_log_probs_from_logits(dev, shape):
    from pfpn_amd import kernels
    B, A, N = shape
    g = torch.Generator(device=dev)
    g.manual_seed(N)
    x = torch.randn(B, A, N, device=dev, generator=g)
    k = torch.randint(0, N, (B, A), device=dev, generator=g)
    gap = torch.tensor(GAPS, device=dev).repeat(B // len(GAPS) + 1)[:B] if B > 5 else torch.tensor([100.0, 90.0, 95.0, -90.0, 0.0], device=dev)[:B]
    adv = torch.tensor([0.0, 1.5, -0.7], device=dev).repeat(B)[:B].roll(1) * (torch.arange(B, device=dev) % 7 != 0)
    base = kernels.categorical_logprob_fwd(x, k)
    old, ref, w = base - gap, base + gap.flip(0), torch.full((B,), 1e-20, device=dev)
    logp, err = logprob(x, k)
    got = kernels.categorical_ppo_fwd_bwd(x, k, old, adv, logp_ref=ref, weight=w, kl_coef=0.05)
    dlogp, derr, loss4, off = far_head(logp, old, adv, ref, w, 0.2, 0.05, err)
    assert torch.isfinite(dlogp).all()
    want, bound = gradient(x, k, dlogp, derr)
    assert bool(((got["dlogits"].double() - want).abs() <= rounded(want, bound, torch.float32)).all())
    assert bool(((got["loss4"].double() - loss4).abs() <= off).all())


# ---- preference loss: pairs that are won or lost by far, and slopes that cancel ----------------------------------------------------------
# P pairs of 2 L steps: the one-block form, groups of 16 and 64 lanes, a block a pair (held and not), pieces of a pair
@pytest.mark.parametrize("P,L", [(12, 3), (2000, 8), (1500, 200), (300, 300), (400, 1000), (2, 20000)])
@pytest.mark.parametrize("kind,smoothing", [("logistic", 0.0), ("logistic", 0.02), ("logistic", 0.5), ("squared", 0.0)])
def test_preference_of_far_margins(dev, P, L, kind, smoothing):
    """the slope -(1 - e) sigma(-m) + e sigma(m) where it is e^-|m| and where it is a small difference: beside its rounding nothing of 32
    bits is in it"""
    from pfpn_amd import kernels
    margins = torch.tensor([-80.0, -20.0, -3.0, -1e-3, 0.0, 1e-6, 0.4, 3.8918202981106265, 12.0, 30.0, 60.0, 85.0])
    g = torch.Generator()
    g.manual_seed(P)
    beta, T = 0.5, 2 * P * L
    ref = (-8 + torch.randn(T, generator=g)).float()
    first = margins.repeat(P // len(margins) + 1)[:P] / beta
    gap = torch.zeros(P, 2, L)
    gap[:, 0, L // 2] = first
    gap = gap + torch.randn(P, 2, L, generator=g) * 1e-6
    logp = (ref.double() + gap.view(-1).double()).float()
    offsets = torch.arange(2 * P + 1) * L
    d = (logp.double() - ref.double()).view(P, 2, L).sum(-1)
    delta = d[:, 0] - d[:, 1]
    m = beta * delta
    if kind == "logistic":
        # (e sigma(m) - (1 - e) sigma(-m) = sigma(-m) (e (1 + e^m) - 1), without a difference of the two)
        s = torch.where(m < 30, torch.sigmoid(-m) * (smoothing * torch.expm1(m) + (2 * smoothing - 1)),
                        smoothing * torch.sigmoid(m) - (1 - smoothing) * torch.exp(-m) / (1 + torch.exp(-m)))
        slope, part = beta * s, beta * (smoothing * torch.sigmoid(m) + (1 - smoothing) * torch.sigmoid(-m))
        loss = -(1 - smoothing) * torch.nn.functional.logsigmoid(m) - smoothing * torch.nn.functional.logsigmoid(-m)
    else:
        slope, loss = 2 * (delta - 0.5 / beta), (delta - 0.5 / beta) ** 2
        part = slope.abs() + 1 / beta
    # 64-bit sums of 2 L terms of about 10, their effect on the slope (Lipschitz beta part, or 2), and 64-bit rounding of its parts
    noise = 2.0 ** -51 * (40 + 2 * L)
    off = ((beta * part * noise if kind == "logistic" else 2 * noise) + 2.0 ** -48 * part) / P
    want = slope / P
    got, margin, l3 = kernels.preference_loss(logp.to(dev), offsets.to(dev), logp_ref=ref.to(dev), beta=beta, label_smoothing=smoothing,
                                              kind=kind)
    got = got.double().cpu().view(P, 2, L)
    bound = (U * want.abs() + off + 1e-45).view(P, 1, 1)
    assert bool(((got[:, :1] - want.view(P, 1, 1)).abs() <= bound).all()) and bool(((got[:, 1:] + want.view(P, 1, 1)).abs() <= bound).all())
    assert bool(((margin.double().cpu() - m).abs() <= U * m.abs() + beta * noise).all())
    mean = loss.mean()
    assert abs(float(l3[0]) - float(mean)) <= float((U + 2.0 ** -40) * mean + noise * part.mean() * (1 if kind == "logistic" else 200))


@pytest.mark.parametrize("T", [50, 20001])          # (one block; pieces of a pair)
def test_preference_bounds_out_of_order(dev, T):
    """bounds beyond the vector or below the one before: as if clamped to [0, T] and to ascend, the same in every call, and nothing
    beside the vectors is read (NaN there) or written"""
    from pfpn_amd import kernels
    g = torch.Generator(device=dev)
    g.manual_seed(T)
    held = [torch.full((T + 64,), math.nan, device=dev) for _ in range(3)]
    logp, ref, w = [t[32:32 + T] for t in held]
    logp.normal_(generator=g)
    ref.normal_(generator=g)
    w.uniform_(generator=g)
    s = T // 50
    for bounds, clamped in (([0, 40, 10], [0, 40, 40]), ([-7, 20, 1 << 40], [0, 20, 50]), ([60, 70, 80], [50, 50, 50]), ([30, 10, 40], [30, 30, 40]),
                            ([-9, -5, -1], [0, 0, 0]), ([45, 20, 3], [45, 45, 45]), ([1 << 62, -(1 << 62), 0], [50, 50, 50]),
                            ([0, 10, 30, 45, 20], [0, 10, 30, 45, 45])):
        scale = lambda v: T if v == 50 else v * s if abs(v) < 1000 else v
        at = torch.tensor([scale(v) for v in bounds], device=dev)
        want, margin, _ = preference(logp, torch.tensor([scale(v) for v in clamped], device=dev), ref, w, 0.1, 0.0, "logistic")
        for _ in range(5):
            d, m, l3 = kernels.preference_loss(logp, at, logp_ref=ref, weight=w)
            assert bool(((d.double() - want).abs() <= U * want.abs() + 1e-9 / (len(bounds) // 2) + 1e-37).all()), bounds
            assert bool(((m.double() - margin).abs() <= U * margin.abs() + 1e-9).all()) and bool(torch.isfinite(l3).all())
        assert all(bool(t[:32].isnan().all()) and bool(t[-32:].isnan().all()) for t in held)


def test_outputs_given_lie_apart_from_what_is_read(dev):
    """an output on memory that other blocks still read (its own old log-probs, a piece of the weights) is refused before the launch"""
    from pfpn_amd import kernels
    x, k = torch.randn(8, 2, 5, device=dev), torch.zeros(8, 2, dtype=torch.int32, device=dev)
    old, adv, ref, w = [torch.rand(8, device=dev) for _ in range(4)]
    pool = torch.rand(64, device=dev)

    def ppo(logp=None, loss4=None, dlogits=None, **kw):
        out = {"logp": pool[:8] if logp is None else logp, "loss4": pool[8:12] if loss4 is None else loss4,
               "dlogits": torch.zeros_like(x) if dlogits is None else dlogits}
        a = dict(logp_old=old, adv=adv, logp_ref=ref, weight=w, kl_coef=0.1, out=out)
        a.update(kw)
        return kernels.categorical_ppo_fwd_bwd(x, k, a.pop("logp_old"), a.pop("adv"), **a)
    want = kernels.categorical_ppo_fwd_bwd(x, k, old, adv, logp_ref=ref, weight=w, kl_coef=0.1)
    got = ppo()
    assert all(torch.equal(got[n], want[n]) for n in want)
    for kw in (dict(logp=old), dict(logp=adv), dict(logp=ref), dict(logp=w), dict(logp=x.view(-1)[8:16]), dict(loss4=w[2:6]), dict(loss4=pool[6:10]),
               dict(logp=pool[4:12], weight=pool[11:19]), dict(loss4=k.view(torch.float32).view(-1)[:4])):
        with pytest.raises(ValueError, match="overlaps"):
            ppo(**kw)
    with pytest.raises(ValueError, match="overlaps"):
        kernels.categorical_logprob_fwd(x, k, out=x.view(-1)[40:48])
    assert torch.equal(kernels.categorical_logprob_fwd(x, k, out=pool[20:28]), kernels.categorical_logprob_fwd(x, k))
    rows = dict(logp_ref=ref, weight=w, kl_coef=0.1)
    want = kernels.policy_kl_loss(old, adv, ref, **rows)
    got = kernels.policy_kl_loss(old, adv, ref, **rows, dlogp=pool[:8], loss4=pool[8:12])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for kw in (dict(dlogp=w), dict(dlogp=adv), dict(loss4=old[:4]), dict(dlogp=pool[:8], loss4=pool[7:11]), dict(dlogp=pool[4:12], stats=pool[11:15])):
        with pytest.raises(ValueError, match="overlaps"):
            kernels.policy_kl_loss(old, adv, ref, **dict(rows, **kw))


# ---- float16 logits in the clipped loss -------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("shape", SHAPES)
def test_policy_loss_from_float16_logits(dev, shape):
    """the shapes of the float32 and bfloat16 test, under its bounds; weights of about one, so that gradients stay above float16's
    smallest step"""
    from pfpn_amd import kernels
    B, A, N = shape
    x, k, g = make_logits(dev, B, A, N, torch.float16, pad=N % 3, seed=2 * N + A, closed=0.05 if N % 2 else 0.0)
    logp, err = logprob(x, k)
    old, adv, ref, w = objective(dev, logp, g, True)
    w[0] = 0.7
    for ref_, c, stats in ((ref, 0.05, None), (None, 0.0, torch.tensor([0.1, 1.7, -1.0, 1.5], device=dev))):
        got = kernels.categorical_ppo_fwd_bwd(x, k.int(), old, adv, logp_ref=ref_, weight=w, stats=stats, clip_eps=(0.2, 0.3), kl_coef=c)
        dlogp, derr, loss4 = head(logp, old, adv, ref_, w, 0.2, 0.3, c, stats, err)
        close(got["logp"], torch.where(w != 0, logp, torch.zeros_like(logp)), err, "logp")
        wg, bg = gradient(x, k, dlogp, derr)
        assert got["dlogits"].dtype == torch.float16
        close(got["dlogits"], wg, rounded(wg, bg, torch.float16), "dlogits")
        lsum = derr.sum() + U * loss4.abs().sum() + 1e-30
        close(got["loss4"], loss4, torch.full((4,), float(lsum), device=dev, dtype=torch.float64), "loss4")


# ---- more rows than one launch has blocks -----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("shape", [((1 << 22) + 5, 1, 1025), ((1 << 22) + 2, 20, 3), ((1 << 21) + 3, 2, 1030)])
def test_more_rows_than_a_launch_has_blocks(dev, shape):
    """the rows on both sides of where a launch ends against the same rows alone (row weights small powers of two: the same bits), the
    loss against the sum over parts"""
    from pfpn_amd import kernels
    B, A, N = shape
    g = torch.Generator(device=dev)
    g.manual_seed(N)
    x = torch.empty(B, A, N, dtype=torch.float16, device=dev)
    for lo in range(0, B, 1 << 18):
        x[lo:lo + (1 << 18)].normal_(generator=g)
    k = torch.randint(0, N, (B, A), device=dev, generator=g)
    adv, w = torch.randn(B, device=dev, generator=g), torch.full((B,), 2.0 ** -4, device=dev)
    logp = kernels.categorical_logprob_fwd(x, k)
    old = logp + 0.1 * torch.randn(B, device=dev, generator=g)
    got = kernels.categorical_ppo_fwd_bwd(x, k, old, adv, logp_ref=logp, weight=w, kl_coef=0.1)
    d = kernels.categorical_logprob_bwd(x, k, adv)
    edge = ((1 << 22) - 1) // (1 if N <= 1024 else A)
    for lo in (0, edge - 30, B - 40):
        part = slice(lo, lo + 40)
        assert torch.equal(logp[part], kernels.categorical_logprob_fwd(x[part], k[part]))
        assert torch.equal(d[part], kernels.categorical_logprob_bwd(x[part], k[part], adv[part]))
        alone = kernels.categorical_ppo_fwd_bwd(x[part], k[part], old[part], adv[part], logp_ref=logp[part], weight=w[part], kl_coef=0.1)
        assert torch.equal(got["dlogits"][part], alone["dlogits"]) and torch.equal(got["logp"][part], alone["logp"])
    half = B // 2
    parts = [kernels.categorical_ppo_fwd_bwd(x[s], k[s], old[s], adv[s], logp_ref=logp[s], weight=w[s], kl_coef=0.1)["loss4"].double()
             for s in (slice(0, half), slice(half, B))]
    total = parts[0] + parts[1]
    scale = 2.0 ** -4 * torch.tensor([2.0, 2.0, 1.0, 1.0], device=dev, dtype=torch.float64) * B
    assert bool(((got["loss4"].double() - total).abs() <= U * (parts[0].abs() + parts[1].abs() + total.abs()) + 1e-14 * scale).all())
