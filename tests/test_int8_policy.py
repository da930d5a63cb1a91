"""precision="int8" and max_grad_norm through the engine, on the CPU."""
import math

import pytest
import torch

from distributedes_amd import evaluate, preset
from distributedes_amd.config import Config
from distributedes_amd.core.engine import TrainState, train_step
from distributedes_amd.models import Int8Layers, MLPPolicy
from distributedes_amd.ops.reference import TorchOps


def _cfg(name="cartpole_es", **kw):
    base = dict(pop=8, generations=3, episode_steps=20, device="cpu",
                noise_table_size=1 << 18, log_every=10 ** 9)
    return preset(name, **{**base, **kw})


@pytest.mark.parametrize("kw", [
    dict(model="nature_cnn", env="pong", precision="int8"),
    dict(max_grad_norm=-1.0), dict(max_grad_norm=math.nan),
    dict(algo="cem", max_grad_norm=1.0)])
def test_refused_by_the_config(kw):
    with pytest.raises(ValueError):
        Config(**kw).validate()


@pytest.mark.parametrize("continuous", [False, True])
@pytest.mark.parametrize("hidden", [(16,), (12, 9), (8, 7, 5)])
def test_forward_against_64_bits(continuous, hidden):
    """Each layer's inputs and weights are off by half a step of their scales at
    most: the output is off by what that passes on."""
    model = MLPPolicy(11, 6, hidden_sizes=hidden, continuous=continuous)
    g = torch.Generator().manual_seed(1)
    P = 5
    flat = torch.randn(P, model.dim, generator=g) * 0.3
    obs = torch.randn(P, 11, generator=g)
    layers = Int8Layers(model, P, "cpu")
    layers.load(TorchOps(), flat)
    got = model.pop_forward_int8(TorchOps(), layers, obs)
    x, err = obs.double(), torch.zeros(P, 11).double()
    names = [f"fc{i + 1}" for i in range(len(hidden))] + ["head"]
    for i, n in enumerate(names):
        w = model.spec.slice(flat, n + ".weight").double()
        b = model.spec.slice(flat, n + ".bias").double()
        half_x = (x.abs() + err).amax(-1, keepdim=True) / 127 * 0.501 + err
        half_w = w.abs().amax(-1, keepdim=True) / 127 * 0.501
        y = (w @ x.unsqueeze(-1)).squeeze(-1) + b
        err = ((w.abs() @ half_x.unsqueeze(-1))
               + (half_w * (x.abs() + half_x).sum(-1)[:, None, None])).squeeze(-1)
        last = i + 1 == len(names)
        x = y if last and not continuous else y.tanh()
    if continuous:
        assert got.shape == (P, 6)
        assert bool(((got.double() - x).abs() <= err + 1e-6).all())
    else:
        # the action taken is the best one up to the error
        taken = x.gather(1, got.unsqueeze(1)).squeeze(1)
        assert bool((taken + 2 * err.amax(-1) >= x.amax(-1)).all())


def test_one_policy_is_the_members_form():
    model = MLPPolicy(4, 2, hidden_sizes=(8, 8))
    theta = model.init_theta(3)
    obs = torch.randn(6, 4, generator=torch.Generator().manual_seed(2))
    one = Int8Layers(model, 6, "cpu", shared=True)
    one.load(TorchOps(), theta.unsqueeze(0))
    many = Int8Layers(model, 6, "cpu")
    many.load(TorchOps(), theta.expand(6, -1))
    a = model.pop_forward_int8(TorchOps(), one, obs)
    assert torch.equal(a, model.pop_forward_int8(TorchOps(), many, obs))


@pytest.mark.parametrize("algo", ["cartpole_es", "cartpole_cem"])
def test_training_in_8_bits(algo):
    st = TrainState(_cfg(algo, precision="int8"), ops_backend="torch_ref")
    before = st.theta.clone()
    for _ in range(2):
        s = train_step(st)
    assert s["env_steps"] == 8 * 20 and "grad_norm" not in s
    assert torch.isfinite(st.theta).all() and not torch.equal(before, st.theta)
    r = evaluate(st, episodes=6)
    assert r["env_steps"] == 6 * 20


def test_bounded_update():
    """The step is that of the direction scaled to the bound; a bound above the
    norm changes nothing."""
    fitness = torch.randn(8, generator=torch.Generator().manual_seed(0))
    thetas, norms = {}, {}
    for bound in (0.0, 1e6, 0.25):
        st = TrainState(_cfg(max_grad_norm=bound, optimizer="sgd"),
                        ops_backend="torch_ref")
        start = st.theta.clone()
        offs, signs = st.member_offsets_signs(0)
        st.es_update(fitness, offs, signs)
        thetas[bound], norms[bound] = st.theta - start, st.grad_norm
    assert norms[0.0] is None
    assert torch.equal(thetas[0.0], thetas[1e6])
    norm = float(norms[0.25])
    assert norm == float(norms[1e6]) and norm > 0.25
    # two roundings of theta (of size 1) around a step of lr * 0.25
    torch.testing.assert_close(thetas[0.25], thetas[0.0] * (0.25 / norm),
                               rtol=1e-5, atol=4 * 2.0 ** -24)
    st = TrainState(_cfg(max_grad_norm=0.25), ops_backend="torch_ref")
    assert train_step(st)["grad_norm"] > 0


def test_checkpoint_round_trip(tmp_path):
    from distributedes_amd.utils import load_checkpoint, save_checkpoint
    cfg = _cfg(precision="int8", max_grad_norm=0.5)
    a = TrainState(cfg, ops_backend="torch_ref")
    train_step(a)
    save_checkpoint(str(tmp_path / "c.pt"), a.checkpoint_payload())
    b = TrainState(cfg, ops_backend="torch_ref")
    b.load_payload(load_checkpoint(str(tmp_path / "c.pt")))
    train_step(a), train_step(b)
    assert torch.equal(a.theta, b.theta)


def test_command_line():
    from distributedes_amd.__main__ import main
    st = main(["--preset", "cartpole_es", "--ops", "torch_ref", "--set",
               "pop=8", "generations=2", "episode_steps=10", "device=cpu",
               "noise_table_size=65536", "precision=int8",
               "max_grad_norm=0.5", "log_every=1000"])
    assert st.generation == 2 and float(st.grad_norm) > 0
