"""GPU: the policy objectives where terms cancel or grow large, against 64-bit forms, within bounds derived from the arithmetic."""
import math

import pytest
import torch

from _objectives import U, balance, segment_bound, softmax

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
