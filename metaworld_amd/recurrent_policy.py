"""A policy with memory on the device, for the environments that leave their batch there (torch_env.MetaWorldTorchVectorEnv).

The reference's meta-learning surface is made for such policies (its RNN-based observations, metaworld/wrappers.py:50-88, and
`metalearning_evaluation`, metaworld/evaluation.py:106-169) and leaves the policy to the user; here is one whose memory is a
selective state space scan: its state has the same size after any number of steps, thousands of environments act one token at a
time, and a training pass reads whole segments of a rollout at once.  A layer is

    x + out(scan(conv(v), gate z)),    v, z = in(norm(x))

with B, C and the step width d of the scan read off conv(v) (sequence.py has the operators).  The layer and its initialisation (decay
rates 1 .. states, step widths spread log-uniformly over 0.001 .. 0.1 through the inverse of softplus, step widths of a rank of a
sixteenth of the width) are those published by A. Gu and T. Dao, "Linear-Time Sequence Modeling with Selective State Spaces", 2023."""
from __future__ import annotations

import math

import torch

from . import sequence


class _Layer(torch.nn.Module):
    def __init__(self, width, inner, states, taps, dtype):
        super().__init__()
        self.rank, self.states, self.inner = max(1, math.ceil(width / 16)), states, inner
        self.norm_weight, self.norm_bias = torch.nn.Parameter(torch.ones(width)), torch.nn.Parameter(torch.zeros(width))
        self.into = torch.nn.Linear(width, 2 * inner, bias=False, dtype=dtype)
        self.conv_weight, self.conv_bias = torch.nn.Parameter(torch.empty(inner, taps).uniform_(-1, 1) * taps ** -0.5), torch.nn.Parameter(torch.zeros(inner))
        self.select = torch.nn.Linear(inner, self.rank + 2 * states, bias=False, dtype=dtype)
        self.step = torch.nn.Linear(self.rank, inner, bias=False, dtype=dtype)
        # decay rates 1 .. states, steps spread over 0.001 .. 0.1 (log-uniformly): memories of a few to a thousand tokens
        rate = torch.exp(torch.empty(inner).uniform_(math.log(1e-3), math.log(1e-1)))
        self.dt_bias = torch.nn.Parameter(rate + torch.log(-torch.expm1(-rate)))
        self.log_A = torch.nn.Parameter(torch.log(torch.arange(1, states + 1, dtype=torch.float32)).repeat(inner, 1))
        self.D = torch.nn.Parameter(torch.ones(inner))
        self.out = torch.nn.Linear(inner, width, bias=False, dtype=dtype)

    def _selected(self, v):
        d, B, C = self.select(v).split([self.rank, self.states, self.states], -1)
        return self.step(d), B, C

    def forward(self, x, reset, lengths, state):
        v, z = self.into(sequence.layer_norm(x, self.norm_weight, self.norm_bias)).chunk(2, -1)
        v, conv = sequence.causal_conv(v, self.conv_weight, self.conv_bias, state=state[0] if state is not None else None, reset=reset, lengths=lengths)
        dt, B, C = self._selected(v)
        y, scan = sequence.selective_scan(v, dt, -torch.exp(self.log_A), B, C, self.D, z, self.dt_bias, state=state[1] if state is not None else None, reset=reset, lengths=lengths)
        return x + self.out(y), (conv, scan)

    def act(self, x, reset, state):
        v, z = self.into(sequence.layer_norm(x, self.norm_weight, self.norm_bias)).chunk(2, -1)
        v = sequence.causal_conv_step(v, self.conv_weight, self.conv_bias, state=state[0], reset=reset)
        dt, B, C = self._selected(v)
        return x + self.out(sequence.selective_scan_step(v, dt, -torch.exp(self.log_A), B, C, self.D, z, self.dt_bias, state=state[1], reset=reset))


class RecurrentPolicy(torch.nn.Module):
    """Observations to actions in [-1, 1], with memory over an episode.

    `forward(obs [batch, time, obs_dim], reset, lengths, state)` -> (actions [batch, time, act_dim], state) for training on segments of
    a rollout; `act(obs [batch, obs_dim], state, reset)` -> actions [batch, act_dim] for acting, `state` updated in place, without
    gradient.  Both give the same actions token by token."""

    def __init__(self, obs_dim, act_dim=4, width=128, layers=2, expand=2, states=16, taps=4, dtype=torch.float32):
        super().__init__()
        self.config = dict(obs_dim=int(obs_dim), act_dim=int(act_dim), width=int(width), layers=int(layers), expand=int(expand), states=int(states), taps=int(taps), dtype=str(dtype).split(".")[-1])
        self.dtype = dtype
        self.embed = torch.nn.Linear(obs_dim, width, dtype=dtype)
        self.layers = torch.nn.ModuleList(_Layer(width, expand * width, states, taps, dtype) for _ in range(layers))
        self.norm_weight, self.norm_bias = torch.nn.Parameter(torch.ones(width)), torch.nn.Parameter(torch.zeros(width))
        self.head = torch.nn.Linear(width, act_dim, dtype=dtype)

    def initial_state(self, batch):
        """the memory of `batch` environments before their first token: per layer the convolution's inputs and the scan's state"""
        inner, device = self.layers[0].inner if len(self.layers) else 0, self.embed.weight.device
        c = self.config
        return [(torch.zeros(batch, c["taps"] - 1, inner, dtype=self.dtype, device=device), torch.zeros(batch, inner, c["states"], device=device)) for _ in self.layers]

    def forward(self, obs, reset=None, lengths=None, state=None):
        x, after = self.embed(obs.to(self.dtype)), []
        for k, layer in enumerate(self.layers):
            x, s = layer(x, reset, lengths, state[k] if state is not None else None)
            after.append(s)
        return torch.tanh(self.head(sequence.layer_norm(x, self.norm_weight, self.norm_bias))), after

    @torch.no_grad()
    def act(self, obs, state, reset=None):
        x = self.embed(obs.to(self.dtype))
        for layer, s in zip(self.layers, state):
            x = layer.act(x, reset, s)
        return torch.tanh(self.head(sequence.layer_norm(x, self.norm_weight, self.norm_bias)))

    def save(self, path):
        torch.save({"config": self.config, "weights": self.state_dict()}, path)

    @classmethod
    def load(cls, path, device="cuda"):
        found = torch.load(path, map_location=device, weights_only=True)
        config = dict(found["config"], dtype=getattr(torch, found["config"]["dtype"]))
        policy = cls(**config).to(device)
        policy.load_state_dict(found["weights"])
        return policy
