"""Operators of sequence policies: linear attention with a decay for each head
(a recurrent memory that trains over a whole sequence at once and acts one
token at a time) and the gated projections of a feed-forward block.

The reference's only memory is a GRU (ttrl/engine/recurrent.py:39-168), whose
unroll is a chain of dependent steps; rows are time-major and `done` resets
the state entering a step, as there.
"""

from __future__ import annotations

import ctypes as C
import math

import numpy as np

from ttrl_amd import _lib
from ttrl_amd.engine.autograd import Tensor, _detached, _needs
from ttrl_amd.engine.ops import _kernels as K
from ttrl_amd.engine.tensor import DeviceArray

__all__ = ["GATED_ACTIVATIONS", "gated_linear", "linear_attention", "linear_attention_step"]

MAX_HEAD = 128
GATED_ACTIVATIONS = tuple(_lib.GATES)


def _dims(t) -> tuple:
    return tuple(int(d) for d in t.shape)


def _p(t):
    return None if t is None else getattr(t, "data", t).ptr


class _Grads:
    """Where a kernel writes the gradients of `tensors`: a tensor's own buffer
    where it holds nothing yet, else an array added to it by `settle`."""

    def __init__(self):
        self._left = []

    def array(self, t: Tensor | None, shape=None, dev=None) -> DeviceArray:
        if t is None or not t.requires_grad:
            return DeviceArray(dev, shape)
        buf, beta = t._grad_target()
        t._note_write(beta, False)
        if beta == 0.0:
            return buf
        own = DeviceArray(t.device, t.shape)
        self._left.append((own, buf))
        return own

    def settle(self) -> None:
        for own, buf in self._left:
            K.binary_into("add", buf, own, buf)
        self._left.clear()


def _attention_shapes(who: str, q, k, v, log_decay, state, done, lead: int):
    """Checks the operands of `lead` leading axes; -> (leading extents, H, kv heads, K, V, a decay per row)."""
    qs, ks, vs = _dims(q), _dims(k), _dims(v)
    axes = "(T, B" if lead == 2 else "(B"
    for name, s in (("q", qs), ("k", ks), ("v", vs)):
        if len(s) != lead + 2:
            raise ValueError(f"{who}: {name} must be shaped {axes}, heads, width), got {s}")
    head, H, width, G, V = qs[:lead], qs[lead], qs[lead + 1], ks[lead], vs[lead + 1]
    if ks != head + (G, width) or vs != head + (G, V):
        raise ValueError(f"{who}: q {qs}, k {ks} and v {vs} must share {axes}), k and v their heads, q and k their width")
    if H < 1 or G < 1 or H % G:
        raise ValueError(f"{who}: {H} heads cannot share {G} key/value heads evenly")
    if not (1 <= width <= MAX_HEAD and 1 <= V <= MAX_HEAD):
        raise ValueError(f"{who}: head widths of 1 to {MAX_HEAD} are supported, got {width} for keys and {V} for values")
    ds = _dims(log_decay)
    if ds not in ((1, H), head + (H,)) :
        raise ValueError(f"{who}: log_decay must be shaped (1, {H}) or {head + (H,)}, got {ds}")
    B = head[-1]
    if state is not None and _dims(state) != (B, H, width, V):
        raise ValueError(f"{who}: state must be shaped {(B, H, width, V)}, got {_dims(state)}")
    if done is not None and _dims(done) != head + (1,):
        raise ValueError(f"{who}: done must be shaped {head + (1,)}, got {_dims(done)}")
    for name, t in (("q", q), ("k", k), ("v", v), ("log_decay", log_decay), ("state", state), ("done", done)):
        if t is not None and t.dtype != np.float32:
            raise ValueError(f"{who}: {name} must be float32, got {t.dtype}")
    # one row: a decay per head and a decay per row are the same numbers
    return head, H, G, width, V, ds != (1, H)


def linear_attention(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, state: Tensor | None = None,
                     done: Tensor | None = None, *, scale: float | None = None):
    """o_t = scale q_t^T S_t with S_t = exp(log_decay) S_{t-1} + k_t v_t^T.

    q (T, B, H, K), k (T, B, G, K), v (T, B, G, V), H a multiple of G; a head
    h uses key/value head h // (H // G).  `log_decay` is (1, H), or (T, B, H)
    for a decay of each step; `state` (B, H, K, V) enters the first step
    (zeros when None); `done` (T, B, 1) resets the state entering a step
    where it is positive.  `scale` defaults to 1 / sqrt(K).
    -> (outputs (T, B, H, V), final state (B, H, K, V)) as tape tensors.

    The backward reads `state` and the final state where they are, as it reads
    q, k and v: a state that goes on in `linear_attention_step` before the
    backward has to be a copy, and the backward refuses one that was stepped."""
    (T, B), H, G, width, V, steps = _attention_shapes("linear_attention", q, k, v, log_decay, state, done, 2)
    dev = q.device
    d = _lib.LinearAttentionDesc()
    d.T, d.B, d.H, d.kv_heads, d.K, d.V = T, B, H, G, width, V
    d.q, d.k, d.v, d.log_decay, d.decay_steps = q.data.ptr, k.data.ptr, v.data.ptr, log_decay.data.ptr, int(steps)
    d.done, d.state = _p(done), _p(state)
    d.scale = 1.0 / math.sqrt(width) if scale is None else float(scale)
    space = [C.c_long() for _ in range(3)]
    _lib.check(_lib.lib().ttrl_linear_attention_space(C.byref(d), *(C.byref(n) for n in space)), "linear_attention")
    forward_n, saved_n, work_n = (n.value for n in space)
    parents = (q, k, v, log_decay) + ((state,) if state is not None else ())
    train = _needs(*parents)
    out, final = DeviceArray(dev, (T, B, H, V)), DeviceArray(dev, (B, H, width, V))
    saved_n = saved_n if train else forward_n
    saved = DeviceArray(dev, (saved_n,)) if saved_n else None
    d.out, d.final_state, d.saved = out.ptr, final.ptr, _p(saved)
    dev.call("ttrl_linear_attention_forward", C.byref(d))
    if not train:
        return _detached(out), _detached(final)
    outputs = Tensor(out, True, parents, "linear_attention")
    kept = (q.data, k.data, v.data, log_decay.data, state and state.data, done and done.data, saved, final)
    dfinal: list = []
    before = (0 if state is None else state.data.steps_noted(), final.steps_noted())

    def _backward(grad: DeviceArray):
        _q, _k, _v, _g, _s, _d, _saved, _final = kept  # alive until here
        if _s is not None and _s.steps_noted() != before[0]:
            raise RuntimeError("linear_attention: the state that entered was stepped in place after the forward, and the "
                               "backward reads it; step a copy")
        if dfinal and log_decay.requires_grad and _final.steps_noted() != before[1]:
            raise RuntimeError("linear_attention: the final state was stepped in place after the forward, and its part of "
                               "the decay's gradient reads it; step a copy")
        grads = _Grads()
        work = DeviceArray(dev, (max(1, work_n),))
        arrays = [grads.array(t, t.shape, dev) for t in (q, k, v)]
        d.dout, d.dfinal, d.work = grad.ptr, _p(dfinal[0] if dfinal else None), work.ptr
        d.dq, d.dk, d.dv = (a.ptr for a in arrays)
        d.dlog_decay = grads.array(log_decay).ptr if log_decay.requires_grad else None
        d.dstate = grads.array(state).ptr if state is not None and state.requires_grad else None
        dev.call("ttrl_linear_attention_backward", C.byref(d))
        grads.settle()
        dfinal.clear()

    outputs._backward = _backward
    last = Tensor(final, True, (outputs,), "linear_attention_state")

    def _final_backward(grad: DeviceArray):
        dfinal.append(grad)
        if outputs.grad is None:
            zero = DeviceArray(dev, outputs.shape)
            zero.fill(0.0)
            outputs._accumulate(zero)

    last._backward = _final_backward
    return outputs, last


def linear_attention_step(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, state: Tensor,
                          done: Tensor | None = None, *, scale: float | None = None) -> Tensor:
    """One token of `linear_attention` for each of B lanes, as an acting step
    takes it: q (B, H, K), k (B, G, K), v (B, G, V), `log_decay` (1, H) or
    (B, H), `done` (B, 1).  `state` (B, H, K, V) is stepped in place;
    -> the outputs (B, H, V).  Records no tape.  A backward that still has to
    read `state` refuses to after this; replays of a captured step are not
    seen, so there the caller keeps the two apart."""
    who = "linear_attention_step"
    (B,), H, G, width, V, rows = _attention_shapes(who, q, k, v, log_decay, state, done, 1)
    if state is None:
        raise ValueError(f"{who}: a state is needed, it is stepped in place")
    if _needs(q, k, v, log_decay, state):
        raise RuntimeError(f"{who} records no tape; call it inside no_grad(), or use linear_attention")
    dev = q.device
    out = DeviceArray(dev, (B, H, V))
    dev.call("ttrl_linear_attention_token", B, H, G, width, V, q.data.vp, k.data.vp, v.data.vp, log_decay.data.vp,
             int(rows), _p(done), C.c_float(1.0 / math.sqrt(width) if scale is None else float(scale)), state.data.vp,
             out.vp)
    state.data.note_step()
    return _detached(out)


def gated_linear(x: Tensor, w_gate: Tensor, w_up: Tensor, b_gate: Tensor | None = None, b_up: Tensor | None = None, *,
                 activation: str = "silu") -> Tensor:
    """act(x @ w_gate + b_gate) * (x @ w_up + b_up), both products, the
    activation and their product in one kernel; weights stored (in, out).
    Forward products of more than 2^28 multiply-adds and the gradients are
    formed from operands of 22 bits (`ttrl_gated_desc` in ttrl_hip.h states
    the bound), smaller ones in FP32."""
    who = "gated_linear"
    if activation not in _lib.GATES:
        raise ValueError(f"{who}: activation must be one of {list(GATED_ACTIVATIONS)}, got {activation!r}")
    if len(x.shape) != 2 or len(w_gate.shape) != 2 or _dims(w_gate) != _dims(w_up):
        raise ValueError(f"{who}: expected (M, K) and two (K, N) weights, got {x.shape}, {w_gate.shape}, {w_up.shape}")
    (M, width), (K2, N) = _dims(x), _dims(w_gate)
    if width != K2:
        raise ValueError(f"{who}: input has {width} features, weights expect {K2}")
    if width < 1 or N < 1:
        raise ValueError(f"{who}: weights of {K2} x {N} are empty")
    for name, b in (("b_gate", b_gate), ("b_up", b_up)):
        if b is not None and b.data.numel != N:
            raise ValueError(f"{who}: {name} has {b.data.numel} elements, expected {N}")
    tensors = (x, w_gate, w_up, b_gate, b_up)
    for name, t in zip(("x", "w_gate", "w_up", "b_gate", "b_up"), tensors):
        if t is not None and t.dtype != np.float32:
            raise ValueError(f"{who}: {name} must be float32, got {t.dtype}")
    dev, train = x.device, _needs(*tensors)
    h = DeviceArray(dev, (M, N))
    g, u = (DeviceArray(dev, (M, N)) for _ in range(2)) if train else (None, None)
    d = _lib.GatedDesc(M, width, N, _lib.GATES[activation], *(_p(t) for t in tensors), _p(g), _p(u), h.ptr)
    forward_n, backward_n = C.c_long(), C.c_long()
    _lib.check(_lib.lib().ttrl_gated_space(C.byref(d), C.byref(forward_n), C.byref(backward_n)), who)
    work = DeviceArray(dev, (forward_n.value,), np.uint8) if forward_n.value else None
    d.work = _p(work)
    dev.call("ttrl_gated_forward", C.byref(d))
    if not train:
        return _detached(h)
    out = Tensor(h, True, tuple(t for t in tensors if t is not None), "gated_linear")
    kept = (x.data, w_gate.data, w_up.data, g, u)

    def _backward(grad: DeviceArray):
        _kept, grads = kept, _Grads()  # alive until here
        work = DeviceArray(dev, (max(1, backward_n.value),), np.uint8)
        d.work, d.dh = work.ptr, grad.ptr
        d.dx, d.dw_gate, d.dw_up, d.db_gate, d.db_up = (
            grads.array(t).ptr if t is not None and t.requires_grad else None for t in tensors)
        dev.call("ttrl_gated_backward", C.byref(d))
        grads.settle()

    out._backward = _backward
    return out
