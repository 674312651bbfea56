"""Sequence policies: blocks of a linear-attention memory and a gated
feed-forward layer, trained over whole sequences at once and acted one token
at a time.  They take the place that the GRU has in the reference's recurrent
actor-critic (ttrl/nets/recurrent.py:49-196): the same time-major rows, the
same episode-start mask on the state entering a step, packed [logits | value]
rows out.

The state that a policy carries from step to step is one (lanes, heads, key,
value) array for each block, whatever the length of the episode."""

from __future__ import annotations

import math

import numpy as np

from ttrl_amd.engine.autograd import Tensor
from ttrl_amd.engine.layers import LayerNorm, Linear
from ttrl_amd.engine.nn import Module, ModuleList
from ttrl_amd.engine.ops import add, exp, gated_linear, linear_attention, linear_attention_step, neg, reshape
from ttrl_amd.engine.tensor import DeviceArray
from ttrl_amd.nets.heads import CategoricalHead, ValueHead, policy_value_packed

__all__ = ["GatedFeedForward", "LinearAttentionMemory", "SequenceBlock", "SequencePolicy"]


def _dims(t) -> tuple:
    return tuple(int(d) for d in t.shape)


class GatedFeedForward(Module):
    """down(act(x W_gate) * (x W_up)), rows (M, features)."""

    def __init__(self, features: int, hidden: int, device, *, activation: str = "silu"):
        if features <= 0 or hidden <= 0:
            raise ValueError(f"GatedFeedForward: features and hidden must be > 0, got {features} and {hidden}")
        self.activation = activation
        bound = 1.0 / math.sqrt(features)

        def weight():
            w = np.random.uniform(-bound, bound, (features, hidden)).astype(np.float32)
            return Tensor.from_numpy(w, device, requires_grad=True)

        self.w_gate, self.w_up = weight(), weight()
        self.down = Linear(hidden, features, device)

    def forward(self, x: Tensor) -> Tensor:
        return self.down(gated_linear(x, self.w_gate, self.w_up, activation=self.activation))


class LinearAttentionMemory(Module):
    """Linear attention over (T, B, features) with a learned decay for each
    head, exp(-exp(rate)); half-lives start spread over 2 to `horizon` steps.
    `kv_heads` key/value heads serve `heads` query heads."""

    def __init__(self, features: int, heads: int, key: int, value: int, device, *, kv_heads: int | None = None,
                 horizon: float = 256.0):
        kv_heads = heads if kv_heads is None else kv_heads
        if features <= 0 or heads <= 0 or kv_heads <= 0 or heads % kv_heads:
            raise ValueError(f"LinearAttentionMemory: features={features}, heads={heads} must be > 0 and heads a multiple "
                             f"of kv_heads={kv_heads}")
        if horizon < 2.0:
            raise ValueError(f"LinearAttentionMemory: horizon must be >= 2 steps, got {horizon}")
        self.heads, self.kv_heads, self.key, self.value = int(heads), int(kv_heads), int(key), int(value)
        self.q = Linear(features, heads * key, device, bias=False)
        self.k = Linear(features, kv_heads * key, device, bias=False)
        self.v = Linear(features, kv_heads * value, device, bias=False)
        self.out = Linear(heads * value, features, device)
        half_lives = np.geomspace(2.0, horizon, heads)
        self.rate = Tensor.from_numpy(np.log(math.log(2.0) / half_lives).astype(np.float32)[None], device, requires_grad=True)

    def initial_state(self, lanes: int) -> Tensor:
        state = DeviceArray(self.rate.device, (lanes, self.heads, self.key, self.value))
        state.fill(0.0)
        return Tensor(state)

    def _projected(self, rows: Tensor, lead: tuple):
        return (reshape(self.q(rows), lead + (self.heads, self.key)), reshape(self.k(rows), lead + (self.kv_heads, self.key)),
                reshape(self.v(rows), lead + (self.kv_heads, self.value)), neg(exp(self.rate)))

    def forward(self, x: Tensor, state: Tensor | None = None, starts: Tensor | None = None):
        """-> (outputs (T, B, features), final state)."""
        T, B, features = _dims(x)
        o, final = linear_attention(*self._projected(reshape(x, (T * B, features)), (T, B)), state, starts)
        y = self.out(reshape(o, (T * B, self.heads * self.value)))
        return reshape(y, (T, B, features)), final

    def step(self, x: Tensor, state: Tensor, starts: Tensor | None = None) -> Tensor:
        """One token (B, features); `state` is stepped in place.  No tape."""
        B = _dims(x)[0]
        o = linear_attention_step(*self._projected(x, (B,)), state, starts)
        return self.out(reshape(o, (B, self.heads * self.value)))


class SequenceBlock(Module):
    """x + memory(norm(x)), then x + feed-forward(norm(x))."""

    def __init__(self, features: int, heads: int, key: int, value: int, hidden: int, device, **memory):
        self.norm_memory = LayerNorm(features, device)
        self.memory = LinearAttentionMemory(features, heads, key, value, device, **memory)
        self.norm_gated = LayerNorm(features, device)
        self.gated = GatedFeedForward(features, hidden, device)

    def _feed(self, rows: Tensor) -> Tensor:
        return add(rows, self.gated(self.norm_gated(rows)))

    def forward(self, x: Tensor, state: Tensor | None = None, starts: Tensor | None = None):
        y, final = self.memory(self.norm_memory(x), state, starts)
        shape = _dims(x)
        rows = self._feed(reshape(add(x, y), (shape[0] * shape[1], shape[2])))
        return reshape(rows, shape), final

    def step(self, x: Tensor, state: Tensor, starts: Tensor | None = None) -> Tensor:
        return self._feed(add(x, self.memory.step(self.norm_memory(x), state, starts)))


class SequencePolicy(Module):
    """Observations (T, B, obs_features) -> packed rows (T * B, n_actions + 1)
    of [logits | value], row t * B + sequence."""

    def __init__(self, obs_features: int, n_actions: int, device, *, features: int, blocks: int, heads: int, key: int,
                 value: int, hidden: int, **memory):
        if blocks < 1:
            raise ValueError(f"SequencePolicy: blocks must be >= 1, got {blocks}")
        self.n_actions = int(n_actions)
        self.encoder = Linear(obs_features, features, device)
        self.blocks = ModuleList([SequenceBlock(features, heads, key, value, hidden, device, **memory)
                                  for _ in range(blocks)])
        self.norm = LayerNorm(features, device)
        self.policy = CategoricalHead(features, n_actions, device)
        self.critic = ValueHead(features, device)

    def initial_states(self, lanes: int) -> list:
        return [b.memory.initial_state(lanes) for b in self.blocks]

    def _checked(self, states) -> list:
        states = list(states)
        if len(states) != len(self.blocks):
            raise ValueError(f"SequencePolicy: {len(states)} states for {len(self.blocks)} blocks")
        return states

    def _head(self, rows: Tensor) -> Tensor:
        return policy_value_packed(self.policy, self.critic, self.norm(rows))

    def forward(self, obs: Tensor, states=None, starts: Tensor | None = None):
        """`starts` (T, B, 1) is positive where a step begins an episode.
        -> (packed rows, the blocks' final states)."""
        T, B, width = _dims(obs)
        rows = self.encoder(reshape(obs, (T * B, width)))
        x = reshape(rows, (T, B, _dims(rows)[1]))
        finals = []
        for block, state in zip(self.blocks, [None] * len(self.blocks) if states is None else self._checked(states)):
            x, final = block(x, state, starts)
            finals.append(final)
        return self._head(reshape(x, (T * B, _dims(rows)[1]))), finals

    def step(self, obs: Tensor, states, starts: Tensor | None = None) -> Tensor:
        """One token for each lane, obs (B, obs_features): packed rows
        (B, n_actions + 1); `states` are stepped in place.  Inside no_grad()."""
        states, x = self._checked(states), self.encoder(obs)
        for block, state in zip(self.blocks, states):
            x = block.step(x, state, starts)
        return self._head(x)
