"""The sequence policy on the GPU: whole sequences against a float64 forward
pass put together from the oracle's operators, gradients against that pass's
differences, token by token against whole sequences, and the recall example.

Tolerances, before the first run (u = 2^-24, about 6e-8): a row passes some ten
products over at most 64 values, each off by (K + 8) u = 4e-6 of its absolute
terms at most; norms bring every branch back to size 1, so rows agree to 1e-4
of 1 + their largest, and a directional derivative to 1e-4 of the product of
the norms of gradient and direction."""

from __future__ import annotations

import sys
from pathlib import Path

import numpy as np
import pytest

from oracle import sequence as O

pytestmark = pytest.mark.gpu

SIZES = [  # T, B, obs, actions, features, blocks, heads, kv_heads, key, value, hidden
    (1, 3, 5, 2, 8, 1, 2, 1, 4, 4, 12),
    (37, 4, 6, 3, 24, 2, 4, 2, 8, 5, 40),
    (70, 5, 3, 4, 33, 1, 3, 3, 16, 17, 65),
]


def _policy(device, size, seed=0):
    from ttrl_amd.nets import SequencePolicy

    T, B, obs, actions, features, blocks, heads, kv_heads, key, value, hidden = size
    np.random.seed(seed)
    policy = SequencePolicy(obs, actions, device, features=features, blocks=blocks, heads=heads, key=key, value=value,
                            hidden=hidden, kv_heads=kv_heads, horizon=32.0)
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((T, B, obs)).astype(np.float32)
    starts = (rng.random((T, B, 1)) < 0.15).astype(np.float32)
    states = [rng.standard_normal((B, heads, key, value)).astype(np.float32) for _ in range(blocks)]
    return policy, x, starts, states


def _forward64(size, p, x, starts, states):
    """The same network in float64 from its named parameters."""
    T, B, _, _, features, blocks, heads, kv_heads, key, value, _ = size

    def norm(r, at):
        c = r - r.mean(-1, keepdims=True)
        return c / np.sqrt((c * c).mean(-1, keepdims=True) + 1e-5) * p[at + ".weight"] + p[at + ".bias"]

    def lin(r, at):
        return r @ p[at + ".weight"] + p.get(at + ".bias", 0.0)

    rows, finals = lin(x.reshape(T * B, -1).astype(np.float64), "encoder"), []
    for i in range(blocks):
        at = f"blocks.{i}."
        n, mem = norm(rows, at + "norm_memory"), at + "memory."
        o, final, _ = O.attention_forward(
            lin(n, mem + "q").reshape(T, B, heads, key), lin(n, mem + "k").reshape(T, B, kv_heads, key),
            lin(n, mem + "v").reshape(T, B, kv_heads, value), -np.exp(p[mem + "rate"]), states[i], starts)
        rows = rows + lin(o.reshape(T * B, heads * value), mem + "out")
        g = at + "gated."
        rows = rows + lin(O.gated_forward(norm(rows, at + "norm_gated"), p[g + "w_gate"], p[g + "w_up"]), g + "down")
        finals.append(final)
    rows = norm(rows, "norm")
    return np.concatenate([lin(rows, "policy.logits"), lin(rows, "critic.value")], -1), finals


def _close(a, b):
    assert np.abs(a - b).max() <= 1e-4 * (1 + np.abs(b).max()), float(np.abs(a - b).max())


@pytest.mark.parametrize("size", SIZES)
def test_sequences_tokens_and_gradients(device, size):
    from ttrl_amd.engine import Tensor, backward_from, no_grad

    policy, x, starts, states = _policy(device, size)
    named = {n: t for n, t in policy.named_parameters()}
    p64 = {n: t.numpy().astype(np.float64) for n, t in named.items()}
    want, want_finals = _forward64(size, p64, x, starts, states)

    def put(a):
        return Tensor.from_numpy(a, device)

    rows, finals = policy(put(x), [put(s) for s in states], put(starts))
    _close(rows.numpy(), want)
    for a, b in zip(finals, want_finals):
        _close(a.numpy(), b)

    rng = np.random.default_rng(1)
    seed = rng.standard_normal(want.shape).astype(np.float32)
    backward_from([(rows, put(seed))])
    got, size2_g, size2_d, step = 0.0, 0.0, 0.0, 1e-6
    away = {n: rng.standard_normal(a.shape) for n, a in p64.items()}
    for n, t in named.items():
        g = t.grad.numpy().astype(np.float64)
        got += float((g * away[n]).sum())
        size2_g += float((g * g).sum())
        size2_d += float((away[n] ** 2).sum())
    ends = [float((_forward64(size, {n: a + s * away[n] for n, a in p64.items()}, x, starts, states)[0] * seed).sum())
            for s in (step, -step)]
    assert abs(got - (ends[0] - ends[1]) / (2 * step)) <= 1e-4 * np.sqrt(size2_g * size2_d)

    with no_grad():
        held = [put(s) for s in states]
        acted = [policy.step(put(x[t]), held, put(starts[t])).numpy() for t in range(size[0])]
    _close(np.concatenate(acted), want)
    for a, b in zip(held, want_finals):
        _close(a.numpy(), b)


def test_initial_states_are_zeros(device):
    policy, x, starts, _ = _policy(device, SIZES[1])
    from ttrl_amd.engine import Tensor, no_grad

    with no_grad():
        a, _ = policy(Tensor.from_numpy(x, device), policy.initial_states(x.shape[1]), Tensor.from_numpy(starts, device))
        b, _ = policy(Tensor.from_numpy(x, device), None, Tensor.from_numpy(starts, device))
    assert np.array_equal(a.numpy(), b.numpy())


def test_refusals(device):
    from ttrl_amd.engine import DeviceArray, Tensor, backward_from
    from ttrl_amd.engine.ops import mul
    from ttrl_amd.nets import GatedFeedForward, LinearAttentionMemory, SequencePolicy

    for make in (lambda: GatedFeedForward(0, 4, device), lambda: GatedFeedForward(4, 0, device),
                 lambda: LinearAttentionMemory(8, 4, 4, 4, device, kv_heads=3),
                 lambda: LinearAttentionMemory(8, 0, 4, 4, device),
                 lambda: LinearAttentionMemory(8, 2, 4, 4, device, horizon=1.0),
                 lambda: SequencePolicy(3, 2, device, features=8, blocks=0, heads=1, key=4, value=4, hidden=8)):
        with pytest.raises(ValueError):
            make()
    policy, x, starts, states = _policy(device, SIZES[0])
    with pytest.raises(RuntimeError):  # acting records no tape
        policy.step(Tensor.from_numpy(x[0], device), policy.initial_states(x.shape[1]))

    leaf = Tensor.from_numpy(np.ones((2, 3), np.float32), device, requires_grad=True)
    seed = Tensor.from_numpy(np.ones((2, 3), np.float32), device)
    with pytest.raises(ValueError):
        backward_from([])
    with pytest.raises(RuntimeError):
        backward_from([(leaf, seed)])
    with pytest.raises(ValueError):
        backward_from([(mul(leaf, 2.0), Tensor.from_numpy(np.ones((3, 2), np.float32), device))])
    with pytest.raises(ValueError):
        backward_from([(mul(leaf, 2.0), DeviceArray(device, (2, 3), np.int32))])
    out = mul(leaf, 2.0)
    backward_from([(out, seed)])
    assert np.array_equal(leaf.grad.numpy(), np.full((2, 3), 2.0, np.float32))
    with pytest.raises(RuntimeError):
        backward_from([(out, seed)])


def test_the_recall_example_learns(device):
    sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "tt-rl_amd" / "examples"))
    import sequence_recall

    result = sequence_recall.run(device, updates=300, log=None)
    assert result["losses"][-1] < 0.5 * result["losses"][0]
    assert result["recalled"] > 0.8  # a guess is right once in four
    assert result["difference"] <= 1e-4 * (1 + result["size"])


def test_states_of_another_count_are_refused(device):
    """A list with a state too few must not run fewer blocks in silence."""
    from ttrl_amd.engine import Tensor, no_grad

    policy, x, starts, states = _policy(device, SIZES[1])  # two blocks

    def put(a):
        return Tensor.from_numpy(a, device)

    for wrong in ([put(states[0])], [put(s) for s in states + states[:1]], []):
        with no_grad(), pytest.raises(ValueError, match="states"):
            policy(put(x), wrong, put(starts))
        with no_grad(), pytest.raises(ValueError, match="states"):
            policy.step(put(x[0]), wrong, put(starts[0]))
