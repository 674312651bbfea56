"""Float64 restatement of the sequence operators, step by step: linear
attention with a decay for each head, the gated projections and AdamW with its
8-bit moments.  No counterpart in the reference; the tests pin the gradients to
central differences of these forwards."""

from __future__ import annotations

import math

import numpy as np

__all__ = ["adamw", "attention_backward", "attention_forward", "gated_backward", "gated_forward", "held_m", "held_v",
           "hold_m", "hold_v"]


def _decays(log_decay, done, T, B, H):
    with np.errstate(over="ignore"):
        a = np.exp(np.broadcast_to(np.asarray(log_decay, np.float64), (T, B, H))).copy()
    if done is not None:
        a[np.asarray(done).reshape(T, B) > 0] = 0.0
    return a


def _repeat(x, share):
    return np.repeat(np.asarray(x, np.float64), share, axis=2)


def attention_forward(q, k, v, log_decay, state=None, done=None, scale=None):
    """-> (out, final, states): states[t] is the one entering step t, in the episode of step t - 1."""
    q = np.asarray(q, np.float64)
    T, B, H, K = q.shape
    share, V = H // k.shape[2], v.shape[3]
    scale = 1.0 / math.sqrt(K) if scale is None else scale
    a, k, v = _decays(log_decay, done, T, B, H), _repeat(k, share), _repeat(v, share)
    S = np.zeros((B, H, K, V)) if state is None else np.asarray(state, np.float64).copy()
    out, states = np.zeros((T, B, H, V)), []
    for t in range(T):
        states.append(S)
        kept = np.where(a[t][..., None, None] > 0, S, 0.0) * a[t][..., None, None]
        S = kept + k[t][..., :, None] * v[t][..., None, :]
        out[t] = scale * np.einsum("bhk,bhkv->bhv", q[t], S)
    return out, S, states


def attention_backward(q, k, v, log_decay, state, done, dout, dfinal=None, scale=None):
    """-> gradients of q, k, v, log_decay (its own shape) and state."""
    out, _, states = attention_forward(q, k, v, log_decay, state, done, scale)
    q = np.asarray(q, np.float64)
    T, B, H, K = q.shape
    G, V = k.shape[2], v.shape[3]
    share = H // G
    scale = 1.0 / math.sqrt(K) if scale is None else scale
    a, kr, vr = _decays(log_decay, done, T, B, H), _repeat(k, share), _repeat(v, share)
    dS = np.zeros((B, H, K, V)) if dfinal is None else np.asarray(dfinal, np.float64).copy()
    dout = np.asarray(dout, np.float64)
    dq, dk, dv, dg = np.zeros_like(q), np.zeros_like(kr), np.zeros_like(vr), np.zeros((T, B, H))
    for t in reversed(range(T)):
        at = a[t][..., None, None]
        kept = np.where(at > 0, states[t], 0.0) * at
        now = kept + kr[t][..., :, None] * vr[t][..., None, :]
        dq[t] = scale * np.einsum("bhkv,bhv->bhk", now, dout[t])
        dS = dS + scale * q[t][..., :, None] * dout[t][..., None, :]
        dk[t] = np.einsum("bhkv,bhv->bhk", dS, vr[t])
        dv[t] = np.einsum("bhkv,bhk->bhv", dS, kr[t])
        dg[t] = (kept * dS).sum((-1, -2))
        dS = np.where(at > 0, dS, 0.0) * at
    dk, dv = (x.reshape(T, B, G, share, -1).sum(3) for x in (dk, dv))
    if np.ndim(log_decay) == 2:
        dg = dg.sum((0, 1)).reshape(1, H)
    return {"q": dq, "k": dk, "v": dv, "log_decay": dg, "state": dS}


_erf = np.vectorize(math.erf)


def _act(name, g):
    """Activation and derivative."""
    if name == "relu":
        return np.maximum(g, 0.0), (g > 0).astype(np.float64)
    if name == "gelu":
        half = 0.5 * (1.0 + _erf(g / math.sqrt(2.0)))
        return g * half, half + g * np.exp(-0.5 * g * g) / math.sqrt(2.0 * math.pi)
    s = 1.0 / (1.0 + np.exp(-g))
    return (s, s * (1.0 - s)) if name == "sigmoid" else (g * s, s * (1.0 + g * (1.0 - s)))


def _projections(x, wg, wu, bg, bu):
    x = np.asarray(x, np.float64)
    g, u = x @ np.asarray(wg, np.float64), x @ np.asarray(wu, np.float64)
    return (g if bg is None else g + bg), (u if bu is None else u + bu)


def gated_forward(x, wg, wu, bg=None, bu=None, act="silu"):
    g, u = _projections(x, wg, wu, bg, bu)
    return _act(act, g)[0] * u


def gated_backward(x, wg, wu, bg, bu, act, dh):
    g, u = _projections(x, wg, wu, bg, bu)
    a, slope = _act(act, g)
    x, dh = np.asarray(x, np.float64), np.asarray(dh, np.float64)
    dg, du = dh * u * slope, dh * a
    return {"x": dg @ np.asarray(wg, np.float64).T + du @ np.asarray(wu, np.float64).T, "w_gate": x.T @ dg,
            "w_up": x.T @ du, "b_gate": dg.sum(0, keepdims=True), "b_up": du.sum(0, keepdims=True)}


def adamw(p, g, m, v, t, lr, betas, eps, weight_decay):
    """Update number t in float64; -> (p, m, v)."""
    p, g, m, v = (np.asarray(x, np.float64) for x in (p, g, m, v))
    b1, b2 = betas
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    return p * (1 - lr * weight_decay) - lr * (m / (1 - b1 ** t)) / (np.sqrt(v / (1 - b2 ** t)) + eps), m, v


def _blocks(x):
    x = np.asarray(x, np.float32).reshape(-1)
    return np.pad(x, (0, -x.size % 64)).reshape(-1, 64), x.size


def _ratio(b):
    top = np.abs(b).max(1, keepdims=True)
    with np.errstate(invalid="ignore", divide="ignore"):
        return np.where(top > 0, np.abs(b) / top, np.float32(0)), top


def hold_m(x):
    """float32 moments -> (codes, block scales) of the 8-bit form, in float32 arithmetic."""
    b, n = _blocks(x)
    r, top = _ratio(b)
    c = np.rint(np.sqrt(r) * np.float32(127)) * np.sign(b)
    return c.astype(np.int8).reshape(-1)[:n], top.reshape(-1)


def hold_v(x):
    b, n = _blocks(x)
    r, top = _ratio(b)
    c = np.rint(np.sqrt(np.sqrt(r)) * np.float32(255))
    c = np.where(r > 0, np.maximum(c, 1), c)
    return c.astype(np.uint8).reshape(-1)[:n], top.reshape(-1)


def _scales(codes, scale):
    return np.repeat(np.asarray(scale, np.float32), 64)[:codes.size]


def held_m(codes, scale):
    c = codes.astype(np.float32) * np.float32(1.0 / 127.0)
    return c * np.abs(c) * _scales(codes, scale)


def held_v(codes, scale):
    c = codes.astype(np.float32) * np.float32(1.0 / 255.0)
    c = c * c
    return c * c * _scales(codes, scale)
