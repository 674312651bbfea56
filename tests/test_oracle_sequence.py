"""The float64 oracle of the sequence operators: its gradients against central
differences, its episodes against separate runs, its 8-bit moments against
their own steps."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import sequence as S


def _differences(f, x, h=1e-5):
    d = np.zeros_like(x)
    for i in np.ndindex(*x.shape):
        keep = x[i]
        x[i] = keep + h
        up = f()
        x[i] = keep - h
        d[i] = (up - f()) / (2 * h)
        x[i] = keep
    return d


@pytest.mark.parametrize("steps", [False, True])
@pytest.mark.parametrize("G", [1, 2])
def test_attention_gradients_match_differences(steps, G):
    rng = np.random.default_rng(3 + G)
    T, B, H, K, V = 5, 2, 2, 3, 2
    x = {"q": rng.standard_normal((T, B, H, K)), "k": rng.standard_normal((T, B, G, K)),
         "v": rng.standard_normal((T, B, G, V)), "state": rng.standard_normal((B, H, K, V)),
         "log_decay": -rng.random((T, B, H) if steps else (1, H))}
    done = np.zeros((T, B, 1))
    done[2, 0] = done[0, 1] = 1
    do, df = rng.standard_normal((T, B, H, V)), rng.standard_normal((B, H, K, V))

    def loss():
        out, final, _ = S.attention_forward(x["q"], x["k"], x["v"], x["log_decay"], x["state"], done)
        return (out * do).sum() + (final * df).sum()

    got = S.attention_backward(x["q"], x["k"], x["v"], x["log_decay"], x["state"], done, do, df)
    for name in x:
        assert np.allclose(got[name], _differences(loss, x[name]), rtol=1e-6, atol=1e-7), name


def test_attention_episodes_are_separate():
    rng = np.random.default_rng(0)
    T, B, H, K, V = 7, 1, 2, 4, 3
    q, k, v = (rng.standard_normal((T, B, H, n)) for n in (K, K, V))
    g, s = -rng.random((T, B, H)), rng.standard_normal((B, H, K, V))
    done = np.zeros((T, B, 1))
    done[3] = 1
    out, final, _ = S.attention_forward(q, k, v, g, s, done)
    first, _, _ = S.attention_forward(q[:3], k[:3], v[:3], g[:3], s)
    second, last, _ = S.attention_forward(q[3:], k[3:], v[3:], g[3:])
    assert np.array_equal(out, np.concatenate([first, second])) and np.array_equal(final, last)


@pytest.mark.parametrize("act", ["silu", "gelu", "relu", "sigmoid"])
def test_gated_gradients_match_differences(act):
    rng = np.random.default_rng(1)
    x, wg, wu = rng.standard_normal((3, 4)), rng.standard_normal((4, 5)), rng.standard_normal((4, 5))
    bg, bu, dh = rng.standard_normal((1, 5)), rng.standard_normal((1, 5)), rng.standard_normal((3, 5))
    got = S.gated_backward(x, wg, wu, bg, bu, act, dh)
    for name, a in (("x", x), ("w_gate", wg), ("w_up", wu), ("b_gate", bg), ("b_up", bu)):
        want = _differences(lambda: (S.gated_forward(x, wg, wu, bg, bu, act) * dh).sum(), a)
        assert np.allclose(got[name], want, rtol=1e-6, atol=1e-7), name


def test_held_moments_are_within_half_a_step():
    rng = np.random.default_rng(2)
    m = (rng.standard_normal(1000) * np.exp(rng.standard_normal(1000) * 2)).astype(np.float32)
    v = np.square(m) * np.float32(0.1)
    v[::7] = 0
    for x, hold, held, root, n in ((m, S.hold_m, S.held_m, 2, 127), (v, S.hold_v, S.held_v, 4, 255)):
        codes, scale = hold(x)
        back = held(codes, scale).astype(np.float64)
        top = np.repeat(scale, 64)[:x.size].astype(np.float64)
        a, b = (np.abs(back) / top) ** (1.0 / root), (np.abs(x) / top) ** (1.0 / root)
        step = np.where((root == 4) & (x != 0) & (b < 0.5 / n), 1.0, 0.5) / n  # what is not zero is never held as zero
        assert (np.abs(a - b) <= step * (1 + 1e-4)).all()
        assert (np.sign(back) == np.sign(np.where(codes == 0, 0, x))).all()
        if root == 4:
            assert ((codes > 0) == (x > 0)).all()
