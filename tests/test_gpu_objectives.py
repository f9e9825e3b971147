"""GPU: the policy objectives (categorical log-probs, clipped loss with a KL term, preference loss, balance loss) against plain
64-bit forms, within bounds derived from the arithmetic (tests/_objectives.py)."""
import math

import pytest
import torch

from _objectives import U, balance, gradient, head, logprob, preference, rounded

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
SHAPES = [(1, 1, 1), (1, 1, 2), (3, 2, 1), (1, 36, 35), (33, 36, 35), (257, 5, 8), (64, 3, 9), (33, 2, 17), (20, 7, 25), (19, 7, 33),
          (5, 130, 41), (7, 13, 64), (5, 3, 65), (5, 3, 96), (9, 4, 97), (9, 4, 128), (6, 2, 129), (6, 2, 192), (5, 3, 193), (5, 128, 256),
          (4, 2, 257), (4, 2, 512), (3, 2, 513), (3, 2, 1024), (2, 3, 1025), (5, 1, 4097), (1, 3, 8191), (3, 1, 50021), (1, 1, 128000),
          (1, 1, 8191), (2, 1, 32768), (2, 2, 32769), (2, 1, 65536), (128, 1, 65536), (130, 1, 65541),
          (700, 1, 1500), (9001, 1, 1100), (8193, 1, 2050), (2, 4096, 3), (1025, 1, 37), (4, 36, 35), (9, 7, 1100), (2, 600, 1030), (3, 700, 300), (2100, 1, 300)]


def make_logits(dev, B, A, N, dtype, pad=0, seed=0, closed=0.0, width=1.5):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    x = torch.randn(B, A, N, device=dev, generator=g) * width * (0.3 + torch.rand(B, A, 1, device=dev, generator=g))
    if closed:
        shut = torch.rand(B, A, N, device=dev, generator=g) < closed
        shut[..., 0] = False
        x = x.masked_fill(shut, -math.inf)
    row = torch.full((B, A * N + pad), 7.0, device=dev, dtype=dtype)
    row[:, :A * N] = x.view(B, A * N).to(dtype)
    k = torch.randint(0, N, (B, A), device=dev, generator=g)
    k = torch.where(torch.isneginf(x.gather(-1, k.unsqueeze(-1)).squeeze(-1)), torch.zeros_like(k), k)
    return row[:, :A * N].unflatten(1, (A, N)), k, g


def close(got, want, bound, what=""):
    got, want = got.double(), want.double()
    assert got.shape == want.shape, what
    same = (got == want) | (got.isnan() & want.isnan())
    off = torch.where(same, torch.zeros_like(got), (got - want).abs() - bound)
    assert not off.isnan().any(), what
    assert float(off.max()) <= 0.0 if off.numel() else True, "%s: off by %.3g over its bound" % (what, float(off.max()))


def objective(dev, logp, g, weighted=False):
    B = logp.shape[0]
    r = torch.exp(0.15 * torch.randn(B, device=dev, dtype=torch.float64, generator=g))
    for border in (0.8, 1.3):           # ratios that rounding could carry over a border of the clip are not drawn
        r = torch.where((r - border).abs() < 2e-3, r + 5e-3, r)
    lp = torch.where(torch.isfinite(logp), logp, torch.full_like(logp, -5.0))
    old, ref = (lp - r.log()).float(), (lp + 0.3 * torch.randn(B, device=dev, dtype=torch.float64, generator=g)).float()
    w = None
    if weighted:
        w = torch.rand(B, device=dev, generator=g)
        w[torch.rand(B, device=dev, generator=g) < 0.3] = 0.0
    return old, torch.randn(B, device=dev, generator=g), ref, w


# ---- categorical log-probs --------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_logprob_and_gradient(dev, shape, dtype):
    from pfpn_amd import kernels
    B, A, N = shape
    pad = (B * 7 + N) % 4
    x, k, g = make_logits(dev, B, A, N, dtype, pad, seed=N + A, closed=0.1 if N % 2 else 0.0)
    k = torch.where(torch.rand(B, A, device=dev, generator=g) < 0.1, torch.full_like(k, -100 if N % 3 else N), k)
    index = k.int() if A % 2 else k
    want, bound = logprob(x, k)
    got = kernels.categorical_logprob_fwd(x, index)
    assert got.dtype == torch.float32
    close(got, want, bound, "logp")
    dlogp = torch.randn(B, device=dev, generator=g)
    if B > 2:
        dlogp[1] = 0.0
    wg, bg = gradient(x, k, dlogp)
    d = kernels.categorical_logprob_bwd(x, index, dlogp)
    assert d.dtype == dtype and d.is_contiguous()
    close(d, wg, rounded(wg, bg, dtype), "dlogits")
    # added to what is there, into padded rows whose padding is left alone
    row = torch.full((B, A * N + 3), 0.5, device=dev, dtype=dtype)
    into = row[:, :A * N].unflatten(1, (A, N))
    kernels.categorical_logprob_bwd(x, index, dlogp, dlogits=into)
    close(into, wg + 0.5, rounded(wg + 0.5, bg + U, dtype), "accumulated")
    assert bool((row[:, A * N:] == 0.5).all())


def test_logprob_two_dimensional_rows_and_repeatability(dev):
    from pfpn_amd import kernels
    x, k, g = make_logits(dev, 40, 1, 3001, torch.bfloat16, 3, seed=3)
    x2, k2 = x.squeeze(1), k.squeeze(1)
    assert x2.stride() == (3004, 1)
    a, b = kernels.categorical_logprob_fwd(x2, k2), kernels.categorical_logprob_fwd(x, k)
    assert torch.equal(a, b) and torch.equal(a, kernels.categorical_logprob_fwd(x2, k2))
    d = torch.randn(40, device=dev, generator=g)
    assert torch.equal(kernels.categorical_logprob_bwd(x2, k2, d), kernels.categorical_logprob_bwd(x, k, d).squeeze(1))


@pytest.mark.parametrize("N", [35, 300, 5000])
def test_closed_and_extreme_logits(dev, N):
    from pfpn_amd import kernels
    low = torch.finfo(torch.float32).min
    x = torch.zeros(6, 2, N, device=dev)
    x[0, 0] = -math.inf                             # nothing open
    x[1, 0] = -math.inf
    x[1, 0, N - 1] = 3.0                            # one open
    x[2, 0] = low                                   # a mask of the type's lowest value everywhere: uniform
    x[3, 0, 1:] = low                               # all but one
    x[4, 0, 0] = -math.inf                          # the choice itself closed
    x[5] = 1e30                                     # large and equal
    k = torch.zeros(6, 2, dtype=torch.int32, device=dev)
    k[1, 0] = N - 1
    want, bound = logprob(x, k)
    got = kernels.categorical_logprob_fwd(x, k)
    assert got[0] == -math.inf and got[4] == -math.inf
    close(got, want, bound)
    dlogp = torch.ones(6, device=dev)
    d = kernels.categorical_logprob_bwd(x, k, dlogp)
    assert bool(torch.isfinite(d).all()) and not d[0, 0].any()
    wg, bg = gradient(x, k, dlogp)
    close(d, wg, rounded(wg, bg, torch.float32))


@pytest.mark.parametrize("N", [35, 5000])
def test_nan_logits_stay_in_their_row(dev, N):
    from pfpn_amd import kernels
    x, k, g = make_logits(dev, 5, 2, N, torch.float32, seed=1)
    x[2, 1, N // 2] = math.nan
    lp = kernels.categorical_logprob_fwd(x, k)
    assert lp.isnan().tolist() == [False, False, True, False, False]
    d = kernels.categorical_logprob_bwd(x, k, torch.ones(5, device=dev))
    assert not d[[0, 1, 3, 4]].isnan().any() and d[2, 1].isnan().all()
    # ... and a row with no upstream gradient, or no weight, is not read at all
    up = torch.tensor([1.0, 1, 0, 1, 1], device=dev)
    assert not kernels.categorical_logprob_bwd(x, k, up).isnan().any()
    v = torch.zeros(5, device=dev)
    bad = v.clone()
    bad[2] = math.nan
    out = kernels.categorical_ppo_fwd_bwd(x, k, bad, bad, logp_ref=bad, weight=up, kl_coef=0.1)
    assert not any(t.isnan().any() for t in out.values()) and out["logp"][2] == 0 and not out["dlogits"][2].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,N", [(520, 1500), (513, 9000), (512, 20001), (3, 6000)])
def test_long_rows_of_every_kind(dev, B, N, dtype):
    """the rows a chip full of long ones may hold: nothing open, one open, all at the type's lowest value, large and equal, far from
    zero, a NaN, no upstream gradient -- none of them touches another"""
    from pfpn_amd import kernels
    x, k, g = make_logits(dev, B, 1, N, dtype, pad=1, seed=N)
    info = torch.finfo(dtype)
    x[0] = -math.inf
    x[1] = -math.inf
    x[1, 0, N - 1], k[1] = 2.0, N - 1
    x[2] = info.min
    if B > 8:
        x[3] = info.max
        x[4] += 300.0                               # (beyond the near range of the exponent; 16-bit steps of 1/4 .. 2)
        x[5] -= 2000.0
        x[6, 0, 1:] = info.min
        x[7, 0, N // 3] = math.nan
        x[8, 0, N // 3], k[8] = -math.inf, N // 3
    dlogp = torch.randn(B, device=dev, generator=g)
    finite = torch.ones(B, dtype=torch.bool, device=dev)
    want, bound = logprob(x, k)
    got = kernels.categorical_logprob_fwd(x, k)
    wg, bg = gradient(x, k, dlogp)
    d = kernels.categorical_logprob_bwd(x, k, dlogp)
    assert got[0] == -math.inf and not d[0].any()
    if B > 8:
        assert got[7].isnan() and d[7].isnan().all() and got[8] == -math.inf
        finite[7] = False
        off = dlogp.clone()
        off[7] = 0.0
        d0 = kernels.categorical_logprob_bwd(x, k, off)
        assert not d0[7].any() and torch.equal(d0[finite], d[finite])
    close(got[finite], want[finite], bound[finite], "logp")
    close(d[finite], wg[finite], rounded(wg, bg, dtype)[finite], "dlogits")


@pytest.mark.parametrize("shape", [(600, 1, 1500), (40, 1, 3000), (700, 2, 1100), (30, 5, 2000)])
def test_rows_without_weight_may_hold_anything(dev, shape):
    from pfpn_amd import kernels
    x, k, g = make_logits(dev, *shape, torch.bfloat16, seed=2)
    old, adv, ref, w = objective(dev, logprob(x, k)[0], g, True)
    w[:3] = torch.tensor([0.5, 0.0, 0.25], device=dev)
    a = kernels.categorical_ppo_fwd_bwd(x, k, old, adv, logp_ref=ref, weight=w, kl_coef=0.1)
    gone = w == 0
    x[gone], old[gone], adv[gone], ref[gone] = math.nan, math.nan, math.inf, -math.inf
    b = kernels.categorical_ppo_fwd_bwd(x, k, old, adv, logp_ref=ref, weight=w, kl_coef=0.1)
    assert all(torch.equal(a[n], b[n]) for n in a) and not a["dlogits"][gone].any() and not a["logp"][gone].any()
    nothing = kernels.categorical_ppo_fwd_bwd(x, k, old, adv, logp_ref=ref, weight=torch.zeros_like(w), kl_coef=0.1)
    assert not any(t.any() for t in nothing.values())


def test_impossible_choice(dev):
    """probability zero: log-prob -inf, ratio 0; without a KL term a finite loss, with one an infinite one"""
    from pfpn_amd import kernels
    x, k = torch.zeros(4, 2, 6, device=dev), torch.zeros(4, 2, dtype=torch.int32, device=dev)
    x[1, 0, 0] = -math.inf
    v = torch.full((4,), -3.5, device=dev)
    out = kernels.categorical_ppo_fwd_bwd(x, k, v, torch.ones(4, device=dev))
    assert out["logp"][1] == -math.inf and bool(torch.isfinite(out["loss4"]).all()) and not out["dlogits"][1].any()
    out = kernels.categorical_ppo_fwd_bwd(x, k, v, torch.ones(4, device=dev), logp_ref=v, kl_coef=0.1)
    assert out["loss4"][0] == math.inf and out["loss4"][2] == math.inf and bool(torch.isfinite(out["dlogits"][[0, 2, 3]]).all())


# ---- clipped loss with a KL term ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_policy_loss_from_logits(dev, shape, dtype):
    from pfpn_amd import kernels
    B, A, N = shape
    x, k, g = make_logits(dev, B, A, N, dtype, pad=N % 3, seed=2 * N + A, closed=0.05 if N % 2 else 0.0)
    logp, err = logprob(x, k)
    weighted = bool(B % 2)
    old, adv, ref, w = objective(dev, logp, g, weighted)
    if w is not None and B > 1:
        w[0] = 0.7
    for ref_, c, stats in ((ref, 0.05, None), (None, 0.0, torch.tensor([0.1, 1.7, -1.0, 1.5], device=dev))):
        got = kernels.categorical_ppo_fwd_bwd(x, k.int(), old, adv, logp_ref=ref_, weight=w, stats=stats, clip_eps=(0.2, 0.3),
                                              kl_coef=c)
        dlogp, derr, loss4 = head(logp, old, adv, ref_, w, 0.2, 0.3, c, stats, err)
        live = torch.ones_like(logp, dtype=torch.bool) if w is None else w != 0
        close(got["logp"], torch.where(live, logp, torch.zeros_like(logp)), err, "logp")
        wg, bg = gradient(x, k, dlogp, derr)
        close(got["dlogits"], wg, rounded(wg, bg, dtype), "dlogits")
        lsum = (derr.sum() + U * loss4.abs().sum() + 1e-30)
        close(got["loss4"], loss4, torch.full((4,), float(lsum), device=dev, dtype=torch.float64), "loss4")


def test_policy_gradient_against_differences(dev):
    """central differences of the 64-bit loss itself, entry by entry: h = 1e-5, off by h^2 |f'''| / 6 + 2^-52 |loss| / h, under 1e-9"""
    from pfpn_amd import kernels
    x, k, g = make_logits(dev, 6, 3, 7, torch.float32, seed=5)
    logp, _ = logprob(x, k)
    old, adv, ref, w = objective(dev, logp, g, True)
    w[0] = 0.5
    got = kernels.categorical_ppo_fwd_bwd(x, k, old, adv, logp_ref=ref, weight=w, clip_eps=(0.2, 0.3), kl_coef=0.4)["dlogits"]
    xd, kc = x.double().cpu(), k.cpu()
    args = [t.cpu() for t in (old, adv, ref, w)]

    def loss(z):
        lp = torch.log_softmax(z, -1).gather(-1, kc.unsqueeze(-1)).squeeze(-1).sum(-1)
        return float(head(lp, *args, 0.2, 0.3, 0.4)[2][0])
    h, num = 1e-5, torch.zeros_like(xd)
    for i in range(xd.numel()):
        up, dn = xd.clone(), xd.clone()
        up.view(-1)[i] += h
        dn.view(-1)[i] -= h
        num.view(-1)[i] = (loss(up) - loss(dn)) / (2 * h)
    assert float((got.double().cpu() - num).abs().max()) < 2e-6 * float(num.abs().max())


@pytest.mark.parametrize("n", [1, 2, 255, 1025, 70001])
@pytest.mark.parametrize("weighted", [False, True])
def test_policy_loss_from_log_probs(dev, n, weighted):
    from pfpn_amd import kernels
    g = torch.Generator(device=dev)
    g.manual_seed(n)
    logp = (-700 + 3 * torch.randn(n, device=dev, generator=g))
    old, adv, ref, w = objective(dev, logp.double(), g, weighted)
    want, bound, loss4 = head(logp.double(), old, adv, ref, w, 0.2, 0.3, 0.05)
    dlogp, l4 = kernels.policy_kl_loss(logp, old, adv, logp_ref=ref, weight=w, clip_eps=(0.2, 0.3), kl_coef=0.05)
    close(dlogp, want, bound + U * want.abs() + 1e-37)
    # a row's term is off by at most what bounds its gradient (|held a| and kl by their exponentials too), summed over the rows
    close(l4, loss4, 1e-12 + 2 * U * loss4.abs() + 4 * float(bound.sum()) + 4 * U * float(l4.abs().sum()))
    none = torch.zeros(n, device=dev)
    dlogp, l4 = kernels.policy_kl_loss(logp, old, adv, weight=none)
    assert not dlogp.any() and not l4.any()


# ---- preference loss ---------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kind", ["logistic", "squared"])
@pytest.mark.parametrize("T,lengths", [(0, [0, 0]), (1, [1, 0]), (5, [0, 0, 2, 1]), (100, [40, 50]), (1000, [0, 300, 64, 65, 255, 257]),
                                       (60001, [1, 30000, 20000, 5000]), (300, [1] * 256), (400000, [150000, 150000, 3, 90000])])
def test_preference_loss(dev, T, lengths, kind):
    from pfpn_amd import kernels
    g = torch.Generator(device=dev)
    g.manual_seed(T + len(lengths))
    start = min(3, T - sum(lengths))
    offsets = torch.tensor([start] + lengths, device=dev).cumsum(0)
    logp = -30 + 3 * torch.randn(T, device=dev, generator=g)
    ref = logp + 0.1 * torch.randn(T, device=dev, generator=g)
    w = torch.rand(T, device=dev, generator=g)
    w[torch.rand(T, device=dev, generator=g) < 0.2] = 0.0
    eps = 0.1 if kind == "logistic" else 0.0
    for ref_, w_ in ((ref, None), (ref, w), (None, w)):
        want, margin, loss3 = preference(logp, offsets, ref_, w_, 0.1, eps, kind)
        if w_ is not None:      # what stands in a step without weight does not matter
            lp, rf = logp.clone(), ref.clone()
            lp[w_ == 0], rf[w_ == 0] = math.nan, math.inf
        else:
            lp, rf = logp, ref
        d, m, l3 = kernels.preference_loss(lp, offsets, logp_ref=rf if ref_ is not None else None, weight=w_, beta=0.1,
                                           label_smoothing=eps, kind=kind)
        # sums in 64 bits: the outputs' own rounding is left, and 64-bit noise of sums of up to T terms of size 30; the logistic
        # loss's exponential, logarithm and quotient are 32-bit: expf, log1pf and 1 / (1 + z) a step or two each, the argument's
        # rounding |m| u, two products and a sum: 16 u and |m| u; its slope is a difference of two such: of the larger one
        noise = 2.0 ** -50 * 40 * (T + 1)
        per = 16 * U + U * float(margin.abs().max())
        slope = 0.1 / len(margin) * per if kind == "logistic" else 0.0
        close(d, want, U * want.abs() + slope + (noise if kind == "squared" else 0.1 * noise) + 1e-37, "dlogp")
        close(m, margin, U * margin.abs() + noise, "margin")
        size = loss3.abs() + noise * (1 + 2 * loss3.abs().max().sqrt() * 10)
        close(l3, loss3, 2 * U * size + per * float(loss3.abs().max()) + noise * (1 + 20 * float(loss3.abs().max()) ** 0.5), "loss3")


@pytest.mark.parametrize("P,longest", [(700, 5), (40000, 4), (2000, 60), (9000, 400), (1100, 350), (8300, 1100), (200, 1000), (200, 3000), (150, 4095)])
def test_many_ragged_pairs(dev, P, longest):
    """every form of the launch by the mean length of a pair; segments of no step among them"""
    from pfpn_amd import kernels
    g = torch.Generator()
    g.manual_seed(P)
    lengths = torch.randint(0, longest + 1, (2 * P,), generator=g)
    offsets = torch.cat([torch.tensor([2]), 2 + lengths.cumsum(0)])
    T = int(offsets[-1]) + 5
    logp, w = -30 + 3 * torch.randn(T, generator=g), torch.rand(T, generator=g)
    ref = logp + 0.1 * torch.randn(T, generator=g)
    w[torch.rand(T, generator=g) < 0.2] = 0.0
    of = torch.repeat_interleave(torch.arange(2 * P), lengths)
    gap = ((logp.double() - ref.double()) * w.double())[2:-5]
    sums = torch.zeros(2 * P, dtype=torch.float64).index_add_(0, of, gap)
    m = 0.1 * (sums[0::2] - sums[1::2])
    loss3 = torch.stack([-torch.nn.functional.logsigmoid(m).mean(), (m > 0).double().mean(), m.mean()])
    want = torch.zeros(T, dtype=torch.float64)
    want[2:-5] = (-0.1 * torch.sigmoid(-m) / P).repeat_interleave(2)[of] * torch.where(of % 2 == 0, 1.0, -1.0) * w[2:-5].double()
    d, got, l3 = kernels.preference_loss(*[t.to(dev) for t in (logp, offsets)], logp_ref=ref.to(dev), weight=w.to(dev), beta=0.1)
    # (bounds as above: sums in 64 bits, the head's 32-bit exponential, logarithm and quotient 16 u, its argument |m| u)
    noise, per = 2.0 ** -50 * 40 * (2 * longest + 1), 16 * U + U * float(m.abs().max())
    close(d.cpu(), want, U * want.abs() + 0.1 / P * per + 0.1 * noise + 1e-37, "dlogp")
    close(got.cpu(), m, U * m.abs() + noise, "margin")
    close(l3.cpu(), loss3, 2 * U * loss3.abs() + per * float(loss3.abs().max()) + noise + 1e-12, "loss3")
    again = kernels.preference_loss(*[t.to(dev) for t in (logp, offsets)], logp_ref=ref.to(dev), weight=w.to(dev), beta=0.1)
    assert torch.equal(d, again[0]) and torch.equal(l3, again[2])


def test_preference_gradient_against_differences(dev):
    """central differences of the 64-bit loss, h = 1e-4: off by h^2 beta^3 and 2^-52 / h, under 1e-9"""
    from pfpn_amd import kernels
    g = torch.Generator(device=dev)
    g.manual_seed(4)
    logp, ref = torch.randn(30, device=dev, generator=g), torch.randn(30, device=dev, generator=g)
    w = torch.rand(30, device=dev, generator=g)
    offsets = torch.tensor([0, 4, 11, 11, 29], device=dev)
    d, _, _ = kernels.preference_loss(logp, offsets, logp_ref=ref, weight=w, beta=0.5, label_smoothing=0.05)
    base, args = logp.double().cpu(), [t.cpu() for t in (offsets, ref, w)]
    num, h = torch.zeros(30, dtype=torch.float64), 1e-4
    for i in range(30):
        e = torch.zeros(30, dtype=torch.float64)
        e[i] = h
        num[i] = (preference(base + e, *args, 0.5, 0.05, "logistic")[2][0] - preference(base - e, *args, 0.5, 0.05, "logistic")[2][0]) / (2 * h)
    assert float((d.double().cpu() - num).abs().max()) < 1e-6       # (the slope, under 0.25, is off by 16 steps of 2^-24 at most)


def test_reported_kl_of_an_impossible_choice_stays_out_of_the_loss(dev):
    """kl_coef = 0 with a reference: the KL term is reported (infinite here), loss and gradient are those without it"""
    from pfpn_amd import kernels
    for B, A, N in ((6, 3, 7), (3, 1, 5000), (2, 1, 70001)):
        x, k, g = make_logits(dev, B, A, N, torch.float32, seed=9)
        x, k = x.contiguous(), k.clamp(min=1)
        x[0].scatter_(-1, k[0].unsqueeze(-1), -math.inf)
        old, adv, ref = torch.full((B,), -5.0, device=dev), torch.randn(B, device=dev, generator=g), torch.full((B,), -5.0, device=dev)
        want = kernels.categorical_ppo_fwd_bwd(x, k, old, adv)
        got = kernels.categorical_ppo_fwd_bwd(x, k, old, adv, logp_ref=ref)
        assert got["loss4"][2] == math.inf and torch.isfinite(got["loss4"][:2]).all()
        assert torch.equal(got["dlogits"], want["dlogits"]) and torch.equal(got["loss4"][[0, 1, 3]], want["loss4"][[0, 1, 3]])
    logp = torch.tensor([-math.inf, -3.0], device=dev)
    d, l4 = kernels.policy_kl_loss(logp, logp.clamp(min=-4), torch.ones(2, device=dev), logp_ref=torch.zeros(2, device=dev))
    assert torch.isfinite(d).all() and l4[2] == math.inf and torch.isfinite(l4[:2]).all()


@pytest.mark.parametrize("T,lengths", [(6, [3, 3]), (60000, [30000, 30000]), (40000, [20, 20] * 1000)])
def test_preference_for_an_impossible_segment(dev, T, lengths):
    """an infinite margin: won pairs have no loss and no gradient, lost ones an infinite loss and the steepest gradient"""
    from pfpn_amd import kernels
    P, offsets = len(lengths) // 2, torch.tensor([0] + lengths, device=dev).cumsum(0)
    for at, loss, slope in ((lengths[0], 0.0, 0.0), (0, math.inf, 0.1)):       # first step of the pair's second / first segment
        logp = torch.full((T,), -1.0, device=dev)
        starts = offsets[:-1].view(P, 2)[:, 0] + at
        logp[starts] = -math.inf
        d, m, l3 = kernels.preference_loss(logp, offsets, beta=0.1)
        assert bool(torch.isinf(m).all()) and l3[0] == loss
        want = torch.full((T,), slope / P, device=dev)
        sign = torch.repeat_interleave(torch.tensor([-1.0, 1.0] * P, device=dev), torch.tensor(lengths, device=dev))
        close(d, want * sign, 4 * U * want.abs())                   # (products and a quotient of 32 bits)


def test_preference_bad_bounds_stay_inside(dev):
    """bounds outside [0, T] are clamped, descending ones make an empty segment: nothing outside the vectors is touched"""
    from pfpn_amd import kernels
    T = 50
    logp, ref = torch.randn(T, device=dev), torch.zeros(T, device=dev)
    for bounds in ([-7, 20, 1 << 40], [60, 70, 80], [30, 10, 40], [-9, -5, -1]):
        d, m, l3 = kernels.preference_loss(logp, torch.tensor(bounds, device=dev), logp_ref=ref)
        assert d.shape == (T,) and bool(torch.isfinite(m).all()) and bool(torch.isfinite(l3).all())
    d, m, _ = kernels.preference_loss(logp, torch.tensor([-7, 20, 1 << 40], device=dev), logp_ref=ref)
    want, margin, _ = preference(logp, torch.tensor([0, 20, 50], device=dev), ref, None, 0.1, 0.0, "logistic")
    close(d, want, (U * want.abs() + 0.1 * 20 * U) + 1e-14)


# ---- balance loss --------------------------------------------------------------------------------------------------------------
BAL = [(1, 1, 1, 1), (1, 1, 2, 2), (2, 3, 8, 3), (33, 36, 35, 1), (700, 36, 35, 2), (300, 5, 16, 16), (64, 7, 24, 1), (64, 7, 32, 4),
       (50, 130, 40, 1), (129, 1, 64, 8), (1000, 1, 96, 6), (4099, 1, 128, 8), (40, 3, 192, 2), (37, 128, 256, 1), (20, 2, 500, 8),
       (9, 3, 1024, 64), (5, 4096, 3, 1), (70001, 1, 8, 2)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,A,N,K", BAL)
def test_balance_loss(dev, R, A, N, K, dtype):
    from pfpn_amd import kernels
    # (few distinct values: equal logits, which the lowest index settles)
    x, _, g = make_logits(dev, R, A, N, dtype, pad=(R + N) % 3, seed=R + N, closed=0.15 if R % 2 else 0.0)
    if N % 2 == 0:
        x.copy_((x * 2).round() / 2)
    coef = 1000.0               # (a float16 gradient stays above that type's smallest step)
    for masked in (False, True):
        mask = (torch.rand(R, device=dev, generator=g) < 0.7) if masked else None
        y = x
        if masked and R > 1:
            mask[0], mask[-1] = True, False
            y = torch.empty_strided(x.shape, x.stride(), dtype=dtype, device=dev).copy_(x)
            y[-1] = math.nan
        loss, counts, mean, grad, bound = balance(x, K, coef, mask)
        got = kernels.balance_loss(y, topk=K, coef=coef, mask=mask)
        assert got[1].dtype == torch.int32 and torch.equal(got[1].long(), counts.long()), "counts"
        # mean_prob: a softmax's bound and up to 1024 32-bit additions of a chunk's rows (measured chunks are far shorter)
        soft = 2 * float((x.double().masked_fill(torch.isneginf(x.double()), 0)).abs().max()) * 2 + 60 + 1024
        close(got[2], mean, soft * U * mean + 1e-37, "mean_prob")
        close(got[0], loss.view(1), soft * U * loss.abs().view(1) + 1e-37, "loss")
        close(got[3], grad, rounded(grad, bound, dtype), "dlogits")
        into = torch.full_like(grad, 0.25, dtype=dtype)
        kernels.balance_loss(y, topk=K, coef=coef, mask=mask, dlogits=into)
        close(into, grad + 0.25, rounded(grad + 0.25, bound + U * (grad.abs() + 0.25), dtype), "accumulated")


def test_balance_nothing_valid_and_nothing_open(dev):
    from pfpn_amd import kernels
    x = torch.randn(12, 3, 9, device=dev)
    loss, counts, mean, d = kernels.balance_loss(x, topk=2, mask=torch.zeros(12, dtype=torch.bool, device=dev))
    assert not loss.any() and not counts.any() and not mean.any() and not d.any()
    x[5, 1] = -math.inf
    loss, counts, mean, d = kernels.balance_loss(x, topk=2)
    assert bool(torch.isfinite(d).all()) and not d[5, 1].any() and counts.sum(-1).tolist() == [24, 22, 24]
    flat = torch.zeros(8, 1, 4, device=dev)
    for r in range(8):
        flat[r, 0, r % 4] = 1e-3
    loss, counts, mean, d = kernels.balance_loss(flat, coef=0.5)
    assert counts.tolist() == [[2, 2, 2, 2]] and abs(float(loss) - 0.5) < 1e-6


def test_balance_gradient_against_differences(dev):
    """the counts are held: central differences of coef N / A sum f P over the logits, h = 1e-5, off by under 1e-9"""
    from pfpn_amd import kernels
    x, _, _ = make_logits(dev, 7, 2, 5, torch.float32, seed=9)
    _, counts, _, d = kernels.balance_loss(x, topk=2, coef=3.0)
    f, xd, h = counts.double().cpu() / 14, x.double().cpu(), 1e-5
    num = torch.zeros_like(xd)
    for i in range(xd.numel()):
        v = []
        for sgn in (h, -h):
            z = xd.clone()
            z.view(-1)[i] += sgn
            v.append(float(3.0 * 5 / 2 * (f * torch.softmax(z, -1).mean(0)).sum()))
        num.view(-1)[i] = (v[0] - v[1]) / (2 * h)
    assert float((d.double().cpu() - num).abs().max()) < 2e-6 * float(num.abs().max()) + 1e-9


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("R,A,N", [(7, 1, 1), (40, 3, 8), (33, 36, 35), (9, 2, 64)])
def test_equal_counts_leave_no_gradient(dev, R, A, N, dtype):
    """every category counts in every row: the gradient is zero, not the rounding of two equal terms"""
    from pfpn_amd import kernels
    x, _, _ = make_logits(dev, R, A, N, dtype, seed=N)
    for coef in (0.01, -2.0):
        loss, counts, _, d = kernels.balance_loss(x, topk=N, coef=coef)
        assert not d.any() and bool((counts == R).all()) and abs(float(loss) - coef) < 1e-5 * abs(coef)


# ---- refusals, empty batches, streams, graphs -------------------------------------------------------------------------------------
def test_refusals_on_the_device(dev):
    from pfpn_amd import kernels
    x, k = torch.randn(4, 3, 5, device=dev), torch.zeros(4, 3, dtype=torch.int32, device=dev)
    b = torch.zeros(4, device=dev)
    for bad in (x.double(), x.transpose(1, 2), x.transpose(0, 1), x[:, :, ::2], x[:, :2], x[0, 0], x[:, :, :0], x.expand(4, 3, 5)[:, :1].expand(4, 3, 5)):
        with pytest.raises(ValueError):
            kernels.categorical_logprob_fwd(bad, k)
    for bad in (k.float(), k[:3], k.t().contiguous(), k.cpu(), k.to(torch.int16)):
        with pytest.raises(ValueError):
            kernels.categorical_logprob_fwd(x, bad)
    for bad in (x, x.bfloat16(), torch.empty(4, 3, 6, device=dev), x.view(-1)[:59]):
        with pytest.raises(ValueError):
            kernels.categorical_logprob_bwd(x, k, b, dlogits=bad)
    wide = torch.randn(4, 40, device=dev)
    with pytest.raises(ValueError, match="overlap"):
        kernels.categorical_logprob_bwd(wide[:, :15].unflatten(1, (3, 5)), k, b, dlogits=wide[:, 15:30].unflatten(1, (3, 5)))
    with pytest.raises(ValueError, match="logp_ref"):
        kernels.categorical_ppo_fwd_bwd(x, k, b, b, kl_coef=0.1)
    for bad in (b[:3], b.double(), b.cpu(), torch.zeros(8, device=dev)[::2]):
        with pytest.raises(ValueError):
            kernels.policy_kl_loss(b, bad, b)
    for bad in (torch.tensor([0, 4], device=dev), torch.tensor([0, 1, 2, 3], device=dev), torch.tensor([0, 1, 2]),
                torch.tensor([0, 1, 2], device=dev, dtype=torch.int32)):
        with pytest.raises(ValueError):
            kernels.preference_loss(b, bad)
    off = torch.tensor([0, 2, 4], device=dev)
    with pytest.raises(ValueError, match="overlap"):
        kernels.policy_kl_loss(wide.view(-1)[:20], *[torch.zeros(20, device=dev)] * 2, dlogp=wide.view(-1)[10:30])
    with pytest.raises(ValueError, match="2\\^31"):        # (the C entry takes the number of rows in 32 bits)
        kernels.categorical_logprob_fwd(torch.empty((1 << 31) + 8, 1, dtype=torch.float16, device=dev), k)
    for kw in ({"beta": 0.0}, {"beta": math.inf}, {"beta": -1.0}, {"kind": "hinge"}, {"label_smoothing": 0.7}, {"kind": "squared", "label_smoothing": 0.1}):
        with pytest.raises(ValueError):
            kernels.preference_loss(b, off, **kw)
    for kw in ({"topk": 0}, {"topk": 6}, {"mask": torch.ones(3, dtype=torch.bool, device=dev)}, {"mask": torch.ones(4, device=dev)},
               {"dlogits": x}):
        with pytest.raises(ValueError):
            kernels.balance_loss(x, **kw)
    with pytest.raises(ValueError):
        kernels.balance_loss(torch.zeros(2, 1, 1025, device=dev))


def test_empty_batches(dev):
    from pfpn_amd import kernels
    x, k, b = torch.empty(0, 3, 5, device=dev), torch.empty(0, 3, dtype=torch.int64, device=dev), torch.empty(0, device=dev)
    assert kernels.categorical_logprob_fwd(x, k).shape == (0,)
    assert kernels.categorical_logprob_bwd(x, k, b).shape == x.shape
    out = kernels.categorical_ppo_fwd_bwd(x, k, b, b, logp_ref=b, kl_coef=0.1)
    assert out["dlogits"].shape == x.shape and out["loss4"].tolist() == [0, 0, 0, 0]
    d, l4 = kernels.policy_kl_loss(b, b, b)
    assert d.shape == (0,) and l4.tolist() == [0, 0, 0, 0]
    loss, counts, mean, d = kernels.balance_loss(x)
    assert not loss.any() and counts.shape == (3, 5) and not counts.any() and d.shape == x.shape


def _together(kernels, x, k, old, adv, ref, w, offsets, mask):
    """a policy's objectives as a step runs them: clipped loss + balance on one gradient, preference on its log-probs"""
    out = kernels.categorical_ppo_fwd_bwd(x, k, old, adv, logp_ref=ref, weight=w, kl_coef=0.05)
    bal = kernels.balance_loss(x, coef=0.1, mask=mask, dlogits=out["dlogits"])
    logp = kernels.categorical_logprob_fwd(x, k)
    dlogp, margin, l3 = kernels.preference_loss(logp, offsets, logp_ref=ref)
    d2 = kernels.categorical_logprob_bwd(x, k, dlogp)
    d3, l4 = kernels.policy_kl_loss(logp, old, adv, logp_ref=ref, weight=w, kl_coef=0.05)
    return [out["logp"], out["dlogits"], out["loss4"], bal[0], bal[1], bal[2], margin, l3, d2, d3, l4]


@pytest.mark.parametrize("shape", [(64, 36, 35), (12, 128, 256), (300, 1, 64), (12, 1, 5000), (530, 1, 2100), (11, 3, 1300)])
def test_together_on_a_side_stream_and_replayed(dev, shape):
    from pfpn_amd import kernels
    B, A, N = shape
    sets = []
    for seed in (1, 2, 3):
        x, k, g = make_logits(dev, B, A, N, torch.float32, seed=seed)
        old, adv, ref, w = objective(dev, logprob(x, k)[0], g, True)
        w[0] = 0.5
        sets.append([x.contiguous(), k, old, adv, ref, w, torch.tensor([0, 3, 5, 5, 11], device=dev),
                     torch.rand(B, device=dev, generator=g) < 0.8])
    run = _together if N <= 1024 else _together_long
    want = [[t.clone() for t in run(kernels, *s)] for s in sets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(kernels, *sets[1])
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want[1]))
    static = [t.clone() for t in sets[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run(kernels, *static)
    for i in (0, 1, 2, 1, 0):
        for s, t in zip(static, sets[i]):
            s.copy_(t)
        graph.replay()
        eager = run(kernels, *sets[(i + 1) % 3])            # the program's own work between replays
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want[i])), i
        assert all(torch.equal(a, b) for a, b in zip(eager, want[(i + 1) % 3])), i


def _together_long(kernels, x, k, old, adv, ref, w, offsets, mask):
    out = kernels.categorical_ppo_fwd_bwd(x, k, old, adv, logp_ref=ref, weight=w, kl_coef=0.05)
    logp = kernels.categorical_logprob_fwd(x, k)
    dlogp, margin, l3 = kernels.preference_loss(logp, offsets, logp_ref=ref)
    return [out["logp"], out["dlogits"], out["loss4"], logp, margin, l3,
            kernels.categorical_logprob_bwd(x, k, dlogp, dlogits=out["dlogits"].clone())]
