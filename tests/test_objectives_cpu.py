"""CPU: what the policy objectives refuse, through the package and through the C ABI (before any launch)."""
import math

import pytest
import torch

from pfpn_amd import _lib, kernels

P = 64          # a non-null address that no refused call reads


def test_package_refuses_host_tensors():
    x, k, b = torch.zeros(4, 3, 5), torch.zeros(4, 3, dtype=torch.int32), torch.zeros(4)
    for call in (lambda: kernels.categorical_logprob_fwd(x, k), lambda: kernels.categorical_logprob_bwd(x, k, b),
                 lambda: kernels.categorical_ppo_fwd_bwd(x, k, b, b), lambda: kernels.policy_kl_loss(b, b, b),
                 lambda: kernels.preference_loss(b, torch.tensor([0, 2, 4])), lambda: kernels.balance_loss(x)):
        with pytest.raises(ValueError, match="CUDA|device"):
            call()


@pytest.mark.parametrize("bad", [-0.1, (0.2, -0.1), (1.5, 0.2), float("nan"), (0.2, float("nan"))])
def test_clip_bounds(bad):
    with pytest.raises(ValueError, match="clip_eps"):
        kernels._clip_bounds(bad)


def test_clip_bounds_forms():
    assert kernels._clip_bounds(0.2) == (0.2, 0.2) and kernels._clip_bounds((0.1, 0.3)) == (0.1, 0.3)


def test_categorical_entry_points_refuse():
    lib = _lib.load()
    ok = dict(logits=P, dtype=0, ld=180, index=P, i64=0, B=4, A=36, N=5)
    bad = [dict(logits=None), dict(index=None), dict(dtype=3), dict(dtype=-1), dict(B=0), dict(A=0), dict(N=0), dict(ld=179),
           dict(A=4097, N=1, ld=1 << 20), dict(N=(1 << 30) + 1, A=1, ld=1 << 40)]
    for change in bad:
        a = dict(ok, **change)
        lead = (a["logits"], a["dtype"], a["ld"], a["index"], a["i64"])
        shape = (a["B"], a["A"], a["N"])
        assert lib.pfpn_categorical_logprob_fwd(*lead, *shape, P, None, 0, None) == 1, change
        assert lib.pfpn_categorical_logprob_bwd(*lead, P, *shape, 0, P, 1 << 41, None, 0, None) == 1, change
        assert lib.pfpn_categorical_ppo_fwd_bwd(*lead, P, P, None, None, None, *shape, 0.2, 0.2, 0.0, P, P, 1 << 41, P,
                                                P, 1 << 30, None) == 1, change
    lead, shape = (P, 0, 180, P, 0), (4, 36, 5)
    assert lib.pfpn_categorical_logprob_fwd(*lead, *shape, None, None, 0, None) == 1
    assert lib.pfpn_categorical_logprob_bwd(*lead, None, *shape, 0, P, 180, None, 0, None) == 1
    assert lib.pfpn_categorical_logprob_bwd(*lead, P, *shape, 0, P, 179, None, 0, None) == 1
    for old, adv, ref, lo, hi, c in ((None, P, None, .2, .2, 0.), (P, None, None, .2, .2, 0.), (P, P, None, .2, .2, .1),
                                     (P, P, None, -.2, .2, 0.), (P, P, None, .2, -.2, 0.), (P, P, None, float("nan"), .2, 0.)):
        assert lib.pfpn_categorical_ppo_fwd_bwd(*lead, old, adv, ref, None, None, *shape, lo, hi, c, P, P, 180, P, P, 1 << 30,
                                                None) == 1
        assert lib.pfpn_policy_kl_loss(P, old, adv, ref, None, None, 10, lo, hi, c, P, P, P, 1 << 30, None) == 1
    assert lib.pfpn_policy_kl_loss(P, P, P, None, None, None, 0, .2, .2, 0., P, P, P, 1 << 30, None) == 1
    # a missing or short workspace
    need = lib.pfpn_categorical_workspace_bytes(4, 36, 5)
    for ws, n in ((None, 0), (P, need - 1)):
        assert lib.pfpn_categorical_ppo_fwd_bwd(*lead, P, P, None, None, None, *shape, .2, .2, 0., P, P, 180, P, ws, n, None) == 3
    long_need = lib.pfpn_categorical_workspace_bytes(4, 1, 5000)
    for ws, n in ((None, 0), (P, 7)):
        assert lib.pfpn_categorical_logprob_fwd(P, 1, 5000, P, 1, 4, 1, 5000, P, ws, n, None) == 3
    assert long_need > 8 and lib.pfpn_categorical_workspace_bytes(0, 1, 5) == 0
    assert lib.pfpn_policy_kl_loss(P, P, P, None, None, None, 10, .2, .2, 0., P, P, P, 8, None) == 3


def test_preference_entry_point_refuses():
    lib = _lib.load()
    need = lib.pfpn_preference_workspace_bytes(3, 100)
    good = dict(logp=P, off=P, P=3, T=100, beta=.1, eps=0., kind=0, d=P, m=P, l=P, ws=P, n=need)

    def call(**change):
        a = dict(good, **change)
        return lib.pfpn_preference_loss(a["logp"], None, None, a["off"], a["P"], a["T"], a["beta"], a["eps"], a["kind"], a["d"],
                                        a["m"], a["l"], a["ws"], a["n"], None)
    for change in (dict(logp=None), dict(off=None), dict(P=0), dict(P=(1 << 22) + 1), dict(T=-1), dict(beta=0.), dict(beta=-1.),
                   dict(beta=float("nan")), dict(eps=-.1), dict(eps=.6), dict(kind=2), dict(kind=-1), dict(d=None), dict(m=None),
                   dict(l=None)):
        assert call(**change) == 1, change
    for change in (dict(ws=None), dict(n=need - 1)):
        assert call(**change) == 3, change


def test_balance_entry_point_refuses():
    lib = _lib.load()
    need = lib.pfpn_balance_workspace_bytes(10, 4, 8)
    good = dict(x=P, dt=0, ld=32, R=10, A=4, N=8, K=1, loss=P, c=P, mp=P, d=P, ldd=32, ws=P, n=need)

    def call(**change):
        a = dict(good, **change)
        return lib.pfpn_balance_loss(a["x"], a["dt"], a["ld"], None, a["R"], a["A"], a["N"], a["K"], .01, 0, a["loss"], a["c"],
                                     a["mp"], a["d"], a["ldd"], a["ws"], a["n"], None)
    for change in (dict(x=None), dict(dt=5), dict(ld=31), dict(R=0), dict(R=(1 << 30) + 1), dict(A=0), dict(N=0),
                   dict(N=1025, ld=1 << 20, ldd=1 << 20), dict(A=4097, ld=1 << 20, ldd=1 << 20), dict(K=0), dict(K=9),
                   dict(N=128, K=65, ld=512, ldd=512), dict(loss=None), dict(c=None), dict(mp=None), dict(d=None), dict(ldd=31)):
        assert call(**change) == 1, change
    for change in (dict(ws=None), dict(n=need - 1)):
        assert call(**change) == 3, change
    assert lib.pfpn_balance_workspace_bytes(10, 1, 2000) == 0


def test_network_options():
    from pfpn_amd import networks
    base = dict(trainable=True, state_shape=[5], action_shape=[2], action_lower_bound=[-1, -1], action_upper_bound=[1, 1],
                common_net_shape=[], critic_net_shape=[8], actor_net_shape=[8])
    for bad in (dict(kl_coef=-0.1), dict(preference_beta=0.0), dict(preference_beta=math.inf), dict(preference_smoothing=0.6), dict(balance_beta=0.1, particles=1025)):
        with pytest.raises(ValueError):
            networks.ParticleFilteringClipPPONetwork(**base, **bad)
    with pytest.raises(NotImplementedError):
        networks.ParticleFilteringClipPPONetwork(**base, kl_coef=0.1, normalize_policy_output=True)
    for cls in ("ParticleFilteringSACNetwork", "ParticleFilteringDDPGNetwork"):
        with pytest.raises(NotImplementedError, match="balance_beta"):
            getattr(networks, cls)(**base, balance_beta=0.1)


@pytest.mark.parametrize("cls", ["ParticleFilteringSACNetwork", "ParticleFilteringDDPGNetwork"])
def test_networks_without_a_value_trunk_refuse_preference_steps(cls):
    """before anything of the step has happened (these networks' critics are Q functions: the step has no place for them)"""
    from pfpn_amd import networks
    net = getattr(networks, cls)(trainable=True, state_shape=[5], action_shape=[2], action_lower_bound=[-1, -1],
                                 action_upper_bound=[1, 1], common_net_shape=[], critic_net_shape=[8], actor_net_shape=[8])
    for call in (net.compute_preference_gradients, lambda *a: net.train_preference(None, None, [], *a)):
        with pytest.raises(NotImplementedError, match="train_preference"):
            call(torch.zeros(4, 5), torch.zeros(4, 2), torch.tensor([0, 2, 4]))


@pytest.mark.parametrize("cls", ["ParticleFilteringA2CNetwork", "ParticleFilteringVTraceNetwork", "ParticleFilteringSACNetwork",
                                 "ParticleFilteringDDPGNetwork"])
def test_kl_coef_is_not_taken_silently(cls):
    from pfpn_amd import networks
    base = dict(trainable=True, state_shape=[5], action_shape=[2], action_lower_bound=[-1, -1], action_upper_bound=[1, 1],
                common_net_shape=[], critic_net_shape=[8], actor_net_shape=[8])
    with pytest.raises(NotImplementedError, match="kl_coef"):
        getattr(networks, cls)(**base, kl_coef=0.1)
    getattr(networks, cls)(**base, kl_coef=0.0)
