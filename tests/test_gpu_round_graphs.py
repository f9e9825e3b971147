"""GPU: training rounds on captured steps (several steps a replay) against eager ones, and what the captured steps consist of."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
S, A = 197, 36
COLUMNS = ["state", "action", "value", "log_prob", "advantage"]


def make(dev, cls="ParticleFilteringClipPPONetwork", particles=64, **over):
    from pfpn_amd import networks
    opts = dict(common_net_shape=[], actor_net_shape=[1024, 512], critic_net_shape=[1024, 512], value_loss_coef=0.5, gamma=0.95,
                normalize_state=True, clip_state=5.0, normalize_advantage=True, particles=particles, resample=-1,
                resample_interval=150)
    opts.update(over)
    net = getattr(networks, cls)(trainable=True, state_shape=[S], action_shape=[A], action_lower_bound=-np.ones(A),
                                 action_upper_bound=np.ones(A), device=dev, seed=3, **opts)
    net.init()
    for op in net.init_ops:
        op()
    return net


def columns(rows, seed):
    r = np.random.default_rng(seed)
    return {k: v.astype(np.float32) for k, v in zip(COLUMNS, (
        r.normal(0, 1, (rows, S)), r.uniform(-1, 1, (rows, A)), r.normal(0, .1, rows), -30.0 + r.normal(0, .2, rows),
        r.normal(0, 1, rows)))}


@pytest.mark.parametrize("particles", [35, 64, 128])
def test_rounds_across_a_resample_tick_equal_eager_ones(dev, monkeypatch, particles):
    """12 rounds of 16 minibatch steps: eight steps a replay, single ones around the tick at step 150, then replays again -- with the
    program's own work between them.  From 64 particles on a step clears its kernels' exchange area on the way."""
    from pfpn_amd.models import SyncReplicasApplier
    got = []
    for graphs in ("0", "1", "1"):
        monkeypatch.setenv("PFPN_GRAPH_TRAIN", graphs)
        net = make(dev, particles=particles)
        opt = SyncReplicasApplier(net, [{"names": None, "lr": 5e-4}], norm_clip=1.0, world_size=1)
        trail = []
        for i in range(12):
            r = np.random.default_rng(i)
            losses = net.train_round(opt, [], COLUMNS, columns(512, i), [r.permutation(512)[:32] for _ in range(16)])
            trail.append((net.store.flat.clone(), [l for l, _ in losses]))
        assert (graphs == "1") == bool(getattr(net, "_round_graphs", {}))
        got.append(trail)
    for replayed in got[1:]:
        for i, ((p0, l0), (p1, l1)) in enumerate(zip(got[0], replayed)):
            assert l0 == l1 and torch.equal(p0, p1), "round %d" % i


def node_types(graph):
    """types of a captured graph's nodes, asked of the runtime: 0 a kernel, 1 a copy, 2 a memset"""
    import ctypes
    hip = ctypes.CDLL("libamdhip64.so")
    raw, n = ctypes.c_void_p(graph.raw_cuda_graph()), ctypes.c_size_t(0)
    assert hip.hipGraphGetNodes(raw, None, ctypes.byref(n)) == 0
    nodes = (ctypes.c_void_p * n.value)()
    assert hip.hipGraphGetNodes(raw, nodes, ctypes.byref(n)) == 0
    types = []
    for node in nodes:
        t = ctypes.c_int(-1)
        assert hip.hipGraphNodeGetType(ctypes.c_void_p(node), ctypes.byref(t)) == 0
        types.append(t.value)
    return types


@pytest.mark.parametrize("particles,kl,balance,B", [(35, 0.0, None, 32), (35, 0.0, None, 4096), (64, 0.0, None, 32), (128, 0.0, None, 30),
                                                    (256, 0.0, None, 512), (35, 0.1, 0.1, 32), (64, 0.1, 0.1, 512), (256, 0.1, 0.1, 64)])
def test_captured_steps_hold_no_memset_nodes(dev, monkeypatch, particles, kl, balance, B):
    """such nodes have given wrong results in later replays"""
    from pfpn_amd.graphs import GraphedLearnerStep, GraphedRollout
    from pfpn_amd.models import SyncReplicasApplier
    plain = torch.cuda.CUDAGraph
    monkeypatch.setattr(torch.cuda, "CUDAGraph", lambda: plain(keep_graph=True))
    net = make(dev, particles=particles, kl_coef=kl, balance_beta=balance)
    net.set_reference()
    opt = SyncReplicasApplier(net, [{"names": None, "lr": 5e-4}], norm_clip=1.0, world_size=1)
    b = columns(B, 0)
    g = GraphedLearnerStep(net, opt, *[torch.from_numpy(b[k]).to(dev) for k in COLUMNS])
    types = node_types(g.graph)
    assert types.count(0) >= 10 and 2 not in types, types
    types = node_types(GraphedRollout(net, 1).graph)
    assert types.count(0) >= 3 and 2 not in types, types


@pytest.mark.parametrize("cls", ["ParticleFilteringSACNetwork", "ParticleFilteringDDPGNetwork"])
def test_captured_off_policy_steps_hold_no_memset_nodes(dev, monkeypatch, cls):
    from pfpn_amd.graphs import GraphedLearnerStep
    from pfpn_amd.models import SyncReplicasApplier
    plain = torch.cuda.CUDAGraph
    monkeypatch.setattr(torch.cuda, "CUDAGraph", lambda: plain(keep_graph=True))
    net, B, r = make(dev, cls, particles=35, normalize_advantage=False), 64, np.random.default_rng(0)
    opt = SyncReplicasApplier(net, [{"names": net.critic_param_names(), "lr": 1e-4}, {"names": net.actor_param_names(), "lr": 1e-4}],
                              norm_clip=1.0, world_size=1)
    args = [torch.from_numpy(t.astype(np.float32)).to(dev) for t in (
        r.normal(0, 1, (B, S)), np.tanh(r.normal(0, 1, (B, A))), r.random(B), r.random(B) < .9, r.normal(0, 1, (B, S)))]
    types = node_types(GraphedLearnerStep(net, opt, *args, noise=net.make_train_noise(B)).graph)
    assert types.count(0) >= 10 and 2 not in types, types


class _Garbage(object):
    """a cycle that notes whether it was collected inside a capture (an older network's graph would end the process there)"""
    seen = []

    def __init__(self):
        self.me = self

    def __del__(self):
        _Garbage.seen.append(torch.cuda.is_current_stream_capturing())


@pytest.mark.parametrize("what", ["step", "rollout"])
def test_nothing_is_collected_inside_a_capture(dev, monkeypatch, what):
    import gc
    from pfpn_amd.graphs import GraphedLearnerStep, GraphedRollout
    from pfpn_amd.models import SyncReplicasApplier
    net = make(dev, particles=35)
    opt = SyncReplicasApplier(net, [{"names": None, "lr": 5e-4}], norm_clip=1.0, world_size=1)
    b = columns(32, 0)
    args = [torch.from_numpy(b[k]).to(dev) for k in COLUMNS]
    plain = net.compute_gradients if what == "step" else net.run_batch

    def step(*a, **kw):                     # leaves cycles behind before and while it runs
        _Garbage()
        out = plain(*a, **kw)
        for _ in range(50):
            _Garbage()
        return out
    monkeypatch.setattr(net, "compute_gradients" if what == "step" else "run_batch", step)
    del _Garbage.seen[:]
    before = gc.get_threshold()
    gc.set_threshold(1, 1, 1)
    try:
        g = GraphedLearnerStep(net, opt, *args) if what == "step" else GraphedRollout(net, 1)
    finally:
        gc.set_threshold(*before)
    assert gc.isenabled()
    gc.collect()
    assert len(_Garbage.seen) > 100 and not any(_Garbage.seen)
    assert g is not None


def test_an_outgrown_workspace_is_not_handed_out_again(dev):
    """a captured step holds the address of the scratch buffer it was captured with: when a larger size replaces the buffer of that
    stream, its memory must not become another tensor's"""
    from pfpn_amd import kernels
    with torch.cuda.stream(torch.cuda.Stream()):
        first = kernels.workspace(3 << 20, dev)
        lo, hi = first.data_ptr(), first.data_ptr() + first.numel()
        del first
        second = kernels.workspace(hi - lo + 1, dev)
        assert second.data_ptr() != lo and second.numel() >= 2 * (hi - lo)
        assert kernels.workspace(1000, dev).data_ptr() == second.data_ptr()
        others = [torch.empty(3 << 20, dtype=torch.uint8, device=dev) for _ in range(20)]
        assert all(t.data_ptr() >= hi or t.data_ptr() + t.numel() <= lo for t in others)
