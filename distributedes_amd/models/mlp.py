"""MLP policy (fc1/fc2/.../head), tanh activations.

Covers BASELINE configs #1 (CartPole 4->64->64->2, discrete argmax) and
#2 (Humanoid-dim 376->256->256->17, continuous tanh).
"""
from __future__ import annotations

import torch
import torch.nn as nn

from .base import PolicyModel


class MLPPolicy(PolicyModel):
    def __init__(self, obs_dim: int, num_actions: int, hidden_sizes=(64, 64),
                 continuous: bool = False):
        self.obs_dim = obs_dim
        self.obs_shape = (obs_dim,)
        self.num_actions = num_actions
        self.hidden_sizes = tuple(hidden_sizes)
        self.continuous = continuous
        super().__init__()

    def template(self) -> nn.Module:
        mod = nn.Sequential()
        sizes = (self.obs_dim,) + self.hidden_sizes
        layers = {}
        for i in range(len(self.hidden_sizes)):
            layers[f"fc{i+1}"] = nn.Linear(sizes[i], sizes[i + 1])
        layers["head"] = nn.Linear(sizes[-1], self.num_actions)
        mod = nn.Module()
        for name, layer in layers.items():
            mod.add_module(name, layer)
        return mod

    def pop_forward_ref(self, flat_w: torch.Tensor, obs: torch.Tensor) -> torch.Tensor:
        """flat_w [P, D] (fp32/bf16), obs [P, obs_dim] -> logits/actions:
        discrete -> int64 actions [P]; continuous -> fp32 actions [P, A]."""
        w = flat_w.to(torch.float32)
        x = obs.to(torch.float32).unsqueeze(-1)          # [P, in, 1]
        nh = len(self.hidden_sizes)
        for i in range(nh):
            W = self.spec.slice(w, f"fc{i+1}.weight")    # [P, out, in]
            b = self.spec.slice(w, f"fc{i+1}.bias")      # [P, out]
            x = torch.tanh(torch.baddbmm(b.unsqueeze(-1), W, x))
        W = self.spec.slice(w, "head.weight")
        b = self.spec.slice(w, "head.bias")
        out = torch.baddbmm(b.unsqueeze(-1), W, x).squeeze(-1)  # [P, A]
        if self.continuous:
            return torch.tanh(out)
        return out.argmax(dim=-1)

    def pop_forward_int8(self, ops, layers: "Int8Layers",
                         obs: torch.Tensor) -> torch.Tensor:
        """The forward with layers in 8 bits: obs [P, obs_dim] fp32 -> actions
        like pop_forward_ref's.  Every layer quantises its inputs, one scale a
        member; activations in between are fp32."""
        x = obs if layers.shared else obs.unsqueeze(1)
        last = len(layers.codes) - 1
        for i, (q, s, b) in enumerate(zip(layers.codes, layers.scales,
                                          layers.biases)):
            act = "tanh" if i < last or self.continuous else "none"
            if layers.shared:
                q, s, b = q[0], s[0], b[0]
            x = ops.int8_linear(x, q, s, b, activation=act)
        x = x if layers.shared else x.squeeze(1)
        return x if self.continuous else x.argmax(dim=-1)


class Int8Layers:
    """An MLP's layers in 8 bits, for P members or for one policy that all P
    environments share: codes, one scale a channel, biases (fp32).  Stands where
    a population's flat weights [P, D] stand; the buffers keep their addresses
    from load to load, as captured hipGraphs need."""

    def __init__(self, model: MLPPolicy, P: int, device, shared: bool = False):
        self.model = model
        self.shared = shared
        self.shape = (P, model.dim)
        n = 1 if shared else P
        self.names = [f"fc{i+1}" for i in range(len(model.hidden_sizes))] + ["head"]
        self.codes, self.scales, self.biases = [], [], []
        for name in self.names:
            out, cols = model.spec._by_name[name + ".weight"].shape
            # rows begin at multiples of 16 bytes: wide loads
            pad = (cols + 15) // 16 * 16
            self.codes.append(torch.empty(n, out, pad, dtype=torch.int8,
                                          device=device)[:, :, :cols])
            self.scales.append(torch.empty(n, out, device=device))
            self.biases.append(torch.empty(n, out, device=device))

    def load(self, ops, flat: torch.Tensor) -> None:
        """flat [P, >= D] fp32 (shared: [1, >= D])."""
        spec = self.model.spec
        for name, q, s, b in zip(self.names, self.codes, self.scales,
                                 self.biases):
            e = spec._by_name[name + ".weight"]
            w = flat[:, e.offset:e.offset + e.numel].unflatten(1, e.shape)
            ops.quantize_rows(w, out=(q, s))
            e = spec._by_name[name + ".bias"]
            b.copy_(flat[:, e.offset:e.offset + e.numel])

    def graph_key(self) -> tuple:
        """What a captured graph has of these weights: all buffers' addresses,
        and the form that it reads them in."""
        return (self.shared, *(t.data_ptr() for t in self.codes + self.scales
                               + self.biases))
