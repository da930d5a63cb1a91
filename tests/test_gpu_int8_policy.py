"""precision="int8" and max_grad_norm through the engine, on the HIP path."""
import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs MI355X", allow_module_level=True)

from distributedes_amd import evaluate, preset
from distributedes_amd.core.engine import TrainState, train_step
from distributedes_amd.models import Int8Layers, MLPPolicy
from distributedes_amd.ops.hip import HipOps
from distributedes_amd.ops.reference import TorchOps


def _cfg(name, **kw):
    base = dict(pop=64, generations=3, episode_steps=12, device="cuda",
                noise_table_size=1 << 20, log_every=10 ** 9, precision="int8")
    return preset(name, **{**base, **kw})


@pytest.mark.parametrize("name", ["cartpole_es", "humanoid_es_10k",
                                  "cartpole_cem"])
def test_generations_replayed_and_eager_alike(name):
    """Captured generations give what eager ones give, bit for bit."""
    thetas, stats = [], []
    for graphs in (True, False):
        st = TrainState(_cfg(name, use_hip_graphs=graphs))
        got = [train_step(st) for _ in range(3)]
        assert all(s["hip_graphs"] == graphs for s in got)
        thetas.append(st.theta.clone())
        stats.append([s["episodic_return_mean"] for s in got])
        evaluate(st, episodes=16)           # another population size between
        train_step(st)
        thetas.append(st.theta.clone())
    assert torch.equal(thetas[0], thetas[2]) and torch.equal(thetas[1], thetas[3])
    assert stats[0] == stats[1] and torch.isfinite(thetas[3]).all()


@pytest.mark.parametrize("continuous", [False, True])
@pytest.mark.parametrize("P,shared", [(1, False), (37, False), (16, True),
                                      (700, True)])
def test_forward_against_the_torch_twin(continuous, P, shared):
    model = MLPPolicy(376, 17, hidden_sizes=(256, 256), continuous=continuous)
    g = torch.Generator().manual_seed(1)
    n = 1 if shared else P
    flat = torch.randn(n, model.dim + 3, generator=g) * 0.06
    obs = torch.randn(P, 376, generator=g).clamp(-5, 5)
    out = []
    for ops, dev in ((HipOps(), "cuda"), (TorchOps(), "cpu")):
        layers = Int8Layers(model, P, dev, shared=shared)
        layers.load(ops, flat.to(dev))
        out.append((layers, model.pop_forward_int8(ops, layers, obs.to(dev))))
    (a, got), (b, want) = out
    for x, y in zip(a.codes + a.scales + a.biases,
                    b.codes + b.scales + b.biases):
        assert torch.equal(x.cpu(), y)
    if continuous:
        # the first layer agrees to 1e-6; an activation on the border of two
        # codes may then take the other: one step of 1/127 times a weight of
        # 0.3 at most, in a few of 256 places
        torch.testing.assert_close(got.cpu(), want, rtol=0, atol=4 * 0.3 / 127)
        assert float((got.cpu() - want).abs().mean()) < 1e-4
    else:
        # the same action, or one whose value is as near
        assert got.dtype == want.dtype
        model.continuous = True
        v = model.pop_forward_int8(TorchOps(), b, obs).atanh()
        model.continuous = False
        lost = v.amax(-1) - v.gather(1, got.cpu().unsqueeze(1)).squeeze(1)
        assert float(lost.max()) <= 8 * 0.3 / 127


def test_bounded_update_on_the_gpu():
    fitness = torch.randn(64, generator=torch.Generator().manual_seed(0))
    thetas = {}
    for dev, backend in (("cpu", "torch_ref"), ("cuda", None)):
        st = TrainState(_cfg("cartpole_es", device=dev, max_grad_norm=0.1),
                        ops_backend=backend)
        offs, signs = st.member_offsets_signs(0)
        st.es_update(fitness.to(st.device), offs, signs)
        thetas[dev] = st.theta.cpu()
        assert float(st.grad_norm) > 0.1
    torch.testing.assert_close(thetas["cpu"], thetas["cuda"], rtol=1e-4,
                               atol=1e-5)
    st = TrainState(_cfg("humanoid_es_10k", max_grad_norm=0.1))
    s = train_step(st)
    assert s["grad_norm"] > 0 and torch.isfinite(st.theta).all()


@pytest.mark.parametrize("episodes", [1, 16, 200])
def test_evaluation_in_8_bits(episodes):
    st = TrainState(_cfg("humanoid_es_10k", episode_steps=20))
    a, b = (evaluate(st, episodes=episodes) for _ in range(2))
    assert a == b and a["env_steps"] == episodes * 20
    assert a["return_min"] <= a["return_mean"] <= a["return_max"]


@pytest.mark.parametrize("shared", [False, True])
def test_graphs_are_told_apart_by_all_buffers(shared):
    """Weights that share one buffer with weights of an earlier graph, and are
    others, get a graph of their own."""
    st = TrainState(_cfg("humanoid_es_10k", episode_steps=4))
    g = torch.Generator("cuda").manual_seed(1)
    P = 64

    def layers(shared):
        out = Int8Layers(st.model, P, "cuda", shared=shared)
        flat = torch.randn(1 if shared else P, st.dim, generator=g,
                           device="cuda") * 0.1
        out.load(st.ops, flat)
        return out

    a, b = layers(False), layers(shared)
    a.codes[0][:1].copy_(b.codes[0][:1])
    b.codes[0] = a.codes[0][:b.codes[0].shape[0]]
    ids = torch.arange(P)
    got = {}
    for graph in (True, False):
        for name, w in (("a", a), ("b", b)):
            got[name, graph] = st._hip_rollout.run(
                w, 7, ids, 4, st.normalizer, allow_graph=graph,
                observe=False)[0]
    assert not torch.equal(got["a", False], got["b", False])
    for name in "ab":
        assert torch.equal(got[name, True], got[name, False])
