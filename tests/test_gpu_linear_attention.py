"""Linear attention with per-head decays on the GPU against the float64 oracle
(oracle/sequence.py): outputs, final state and every gradient, over lengths,
widths, head layouts, resets and segments; the single-token form against the
sequence; values that are not finite; refusals.

Tolerance, from float32's rounding before the first run: an element is a sum
of products, so its error is at most n u times the same sum over absolute
values, u = 2^-24.  n counts the roundings on the longest path: a head's inner
products (K + V), a chunk's inner sums (32), one per chunk for the state (T /
32, twice where segments are joined), the weights (an exponent of up to 104 in
float32, 104 u, and a handful of factors).  n = K + V + T / 8 + 256 covers them
and the sums over shared heads.  The gradient of a log decay is a sum, from its
step to the end of its episode, of q . dq - k . dk: its bound is n u times the
sum of their absolute terms."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import sequence as O

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _inputs(seed, T, B, H, G, K, V, steps, resets, state, dfinal):
    rng = np.random.default_rng(seed)

    def normal(*s):
        return rng.standard_normal(s).astype(np.float32)

    x = {"q": normal(T, B, H, K), "k": normal(T, B, G, K), "v": normal(T, B, G, V)}
    x["log_decay"] = (-rng.exponential(0.2, (T, B, H) if steps else (1, H))).astype(np.float32)
    x["state"] = normal(B, H, K, V) if state else None
    x["done"] = None if resets is None else (rng.random((T, B, 1)) < resets).astype(np.float32)
    return x, normal(T, B, H, V), normal(B, H, K, V) if dfinal else None


def _tensor(device, a, grad, offset=0):
    """A tensor of `a`, `offset` floats into its allocation."""
    from ttrl_amd.engine.autograd import Tensor
    from ttrl_amd.engine.tensor import DeviceArray

    block = DeviceArray(device, (a.size + offset,))
    view = block.view(offset, a.shape)
    view.upload(a)
    return Tensor(view, grad)


def _run(device, x, dout, dfinal, offset=0, scale=None):
    from ttrl_amd.engine.autograd import backward_from
    from ttrl_amd.engine.ops import linear_attention

    t = {n: None if a is None else _tensor(device, a, n != "done", offset) for n, a in x.items()}
    out, final = linear_attention(t["q"], t["k"], t["v"], t["log_decay"], t["state"], t["done"], scale=scale)
    got = {"out": out.numpy(), "final": final.numpy()}
    seeds = [(out, _tensor(device, dout, False))]
    if dfinal is not None:
        seeds.append((final, _tensor(device, dfinal, False)))
    backward_from(seeds)
    got.update({n: t[n].grad.numpy() for n in ("q", "k", "v", "log_decay", "state") if t[n] is not None})
    return got


def _wanted(x, dout, dfinal, scale=None):
    """-> (values, the sums of absolute terms that bound their errors)."""
    args = (x["q"], x["k"], x["v"], x["log_decay"], x["state"], x["done"])
    out, final, _ = O.attention_forward(*args, scale)
    want = {"out": out, "final": final, **O.attention_backward(*args, dout, dfinal, scale)}
    size = [None if a is None else np.abs(a) for a in (x["q"], x["k"], x["v"])]
    size += [x["log_decay"], None if x["state"] is None else np.abs(x["state"]), x["done"]]
    sout, sfinal, _ = O.attention_forward(*size, scale and abs(scale))
    sb = O.attention_backward(*size, np.abs(dout), None if dfinal is None else np.abs(dfinal), scale and abs(scale))
    T, B, H, K = x["q"].shape
    share = H // x["k"].shape[2]
    term = (size[0] * sb["q"]).sum(-1) + np.repeat((size[1] * sb["k"]).sum(-1), share, 2)
    far = np.cumsum(term[::-1], 0)[::-1] + sb["log_decay"].max(initial=0.0) if T else term
    bound = {"out": sout, "final": sfinal, **sb, "log_decay": far if x["log_decay"].ndim == 3 else far.sum((0, 1))[None]}
    return want, bound


def _check(got, want, bound, n, names=None):
    for name in names or got:
        err = np.abs(got[name].astype(np.float64) - want[name])
        lim = n * U * bound[name] + 1e-30
        assert got[name].shape == want[name].shape, name
        assert (err <= lim).all(), (name, float((err / lim).max()))


CASES = [
    # T, B, H, G, K, V, steps, resets, state, dfinal
    (1, 1, 1, 1, 1, 1, False, None, False, False),
    (1, 3, 4, 2, 16, 16, True, 0.5, True, True),
    (31, 2, 2, 1, 17, 5, True, 0.1, True, True),
    (32, 16, 8, 8, 64, 64, False, 0.02, True, False),
    (33, 1, 3, 3, 64, 32, False, None, True, True),
    (65, 2, 6, 3, 40, 72, True, 0.05, True, True),
    (100, 1, 1, 1, 128, 128, True, 0.03, False, False),
    (96, 5, 4, 1, 3, 100, False, 0.2, True, True),
    (257, 1, 2, 2, 33, 65, True, 1.0, True, True),
    (700, 2, 2, 1, 16, 48, False, 0.01, True, True),
    (1500, 1, 1, 1, 24, 8, True, 0.002, True, False),
    (64, 600, 2, 2, 16, 16, False, 0.02, True, False),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x) for x in c))
def test_matches_the_oracle(device, case):
    T, B, H, G, K, V = case[:6]
    x, dout, dfinal = _inputs(hash(case[:6]) % 1000, *case)
    got = _run(device, x, dout, dfinal)
    _check(got, *_wanted(x, dout, dfinal), K + V + T / 8 + 256)


@pytest.mark.parametrize("offset", [1, 2, 4])
def test_any_alignment(device, offset):
    x, dout, dfinal = _inputs(7, 70, 2, 4, 2, 32, 64, True, 0.05, True, True)
    got = _run(device, x, dout, dfinal, offset=offset, scale=-0.3)
    _check(got, *_wanted(x, dout, dfinal, -0.3), 32 + 64 + 9 + 256)


def test_strong_and_infinite_decays(device):
    """A strong decay takes nothing from the weights after it, and one that
    underflows forgets as a reset does."""
    x, dout, dfinal = _inputs(8, 90, 2, 2, 2, 16, 16, True, 0.02, True, True)
    x["log_decay"][::9] = -100.0
    x["log_decay"][4::13, 0] = -np.inf
    x["log_decay"][7::17, 1] = -1e30
    x["log_decay"][:, :, 1] *= np.float32(0.001)
    got = _run(device, x, dout, dfinal)
    _check(got, *_wanted(x, dout, dfinal), 16 + 16 + 12 + 256)
    forgets = (x["done"] > 0) | (x["log_decay"] < -104)
    assert (got["log_decay"][forgets] == 0).all()


def test_no_step_and_no_sequence(device):
    for T, B in ((0, 3), (4, 0)):
        x, dout, dfinal = _inputs(9, T, B, 2, 1, 8, 4, False, None, True, True)
        got = _run(device, x, dout, dfinal)
        assert got["out"].shape == (T, B, 2, 4) and np.array_equal(got["final"], x["state"])
        assert np.array_equal(got["state"], dfinal) and not got["log_decay"].any()
        assert got["q"].shape == x["q"].shape


@pytest.mark.parametrize("T,B", [(90, 2), (300, 1)])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_what_is_not_finite_stays_in_its_episode(device, T, B, bad):
    """Episodes other than the spoilt one, and its steps before the spoilt one
    (after it, for gradients), are what they are without it."""
    x, dout, _ = _inputs(10, T, B, 2, 2, 16, 24, True, None, True, False)
    x["done"] = np.zeros((T, B, 1), np.float32)
    x["done"][[20, 50, 75]] = 1
    t = 60
    clean, bound = _wanted(x, dout, None)
    n = 16 + 24 + T / 8 + 256
    other = np.ones((T, B), bool)
    other[50:75, 0] = False
    for name in ("q", "k", "v", "log_decay"):
        y = {m: None if a is None else a.copy() for m, a in x.items()}
        y[name][t, 0] = bad if name != "log_decay" else np.nan
        got = _run(device, y, dout, None)
        for out in ("out", "q", "k", "v", "log_decay"):
            keep = other.copy()
            if out == "out":
                keep[50:t, 0] = True
            _check({out: got[out][keep]}, {out: clean[out][keep]}, {out: bound[out][keep]}, n)
        _check(got, clean, bound, n, ("state",))
        if T == 90:
            _check(got, clean, bound, n, ("final",))
    spoilt = dout.copy()
    spoilt[t, 0] = bad
    got = _run(device, x, spoilt, None)
    for out in ("q", "k", "v", "log_decay"):
        keep = other.copy()
        keep[t + 1:75, 0] = True
        _check({out: got[out][keep]}, {out: clean[out][keep]}, {out: bound[out][keep]}, n)


def test_tokens_are_the_sequence(device):
    from ttrl_amd.engine.ops import linear_attention_step

    for seed, (B, H, G, K, V, steps) in enumerate([(1, 8, 8, 64, 64, False), (5, 4, 2, 40, 72, True), (3, 2, 1, 7, 9, True),
                                                   (2, 1, 1, 128, 128, False), (70, 3, 3, 16, 1, True)]):
        T = 6
        x, _, _ = _inputs(20 + seed, T, B, H, G, K, V, steps, 0.2, True, False)
        (want, final, _), size = O.attention_forward(*x.values()), {n: np.abs(a) for n, a in x.items()}
        size["log_decay"] = x["log_decay"]
        bout, bfinal, _ = O.attention_forward(*size.values())
        state = _tensor(device, x["state"], False)
        for t in range(T):
            at = {n: _tensor(device, a if n == "log_decay" and not steps else a[t], False, offset=t % 2)
                  for n, a in x.items() if n != "state"}
            out = linear_attention_step(at["q"], at["k"], at["v"], at["log_decay"], state, at["done"])
            _check({"out": out.numpy()}, {"out": want[t]}, {"out": bout[t]}, K + 8 * T + 64)
        _check({"final": state.numpy()}, {"final": final}, {"final": bfinal}, 8 * T + 64)


def test_a_token_forgets_what_is_not_finite(device):
    from ttrl_amd.engine.ops import linear_attention_step

    x, _, _ = _inputs(30, 1, 2, 2, 2, 8, 8, False, 0.0, True, False)
    x["state"][0] = np.nan
    x["done"][0, 0] = 1
    state = _tensor(device, x["state"], False)
    t = {n: _tensor(device, a if n == "log_decay" else a[0], False) for n, a in x.items() if n != "state"}
    out = linear_attention_step(t["q"], t["k"], t["v"], t["log_decay"], state, t["done"])
    x["state"][0] = 0
    want, final, _ = O.attention_forward(*x.values())
    assert np.allclose(out.numpy(), want[0], rtol=1e-5, atol=1e-5) and np.allclose(state.numpy(), final, rtol=1e-6)


def test_gradients_add_to_what_is_there(device):
    """One tensor as q and k, and a second pass onto a kept gradient."""
    from ttrl_amd.engine.autograd import backward_from
    from ttrl_amd.engine.ops import linear_attention

    x, dout, _ = _inputs(40, 40, 2, 2, 2, 16, 16, False, 0.1, False, False)
    x["k"] = x["q"]
    qk, v, g = (_tensor(device, x[n], True) for n in ("q", "v", "log_decay"))
    done = _tensor(device, x["done"], False)
    for _ in range(2):
        out, _ = linear_attention(qk, qk, v, g, None, done)
        backward_from([(out, _tensor(device, dout, False))])
    want, bound = _wanted(x, dout, None)
    both = {"x": 2 * (want["q"] + want["k"])}, {"x": 2 * (bound["q"] + bound["k"])}
    _check({"x": qk.grad.numpy()}, *both, 300)
    _check({"v": v.grad.numpy()}, {"v": 2 * want["v"]}, {"v": 2 * bound["v"]}, 300)


def test_a_captured_pass_replays(device):
    from ttrl_amd.engine.autograd import backward_from
    from ttrl_amd.engine.ops import linear_attention
    from ttrl_amd.engine.step import TrainStep

    x, dout, dfinal = _inputs(41, 200, 1, 2, 1, 32, 32, True, 0.02, True, True)
    eager = _run(device, x, dout, dfinal)
    t = {n: _tensor(device, a, n != "done") for n, a in x.items()}
    t.update(dout=_tensor(device, dout, False), dfinal=_tensor(device, dfinal, False))
    made = {}

    def body(t):
        for a in t.values():
            a.zero_grad()
        made["out"], made["final"] = linear_attention(t["q"], t["k"], t["v"], t["log_decay"], t["state"], t["done"])
        backward_from([(made["out"], t["dout"]), (made["final"], t["dfinal"])])
        return {}

    with TrainStep(body, t, device, mode="graph") as step:
        step.run()
        for _ in range(3):
            step.replay()
            device.synchronize()
            got = {"out": made["out"].numpy(), "final": made["final"].numpy()}
            got.update({n: t[n].grad.numpy() for n in ("q", "k", "v", "log_decay", "state")})
            for n in got:
                assert np.array_equal(got[n], eager[n]), n


def test_refusals(device):
    from ttrl_amd.engine.ops import linear_attention, linear_attention_step

    def t(*shape, grad=False):
        return _tensor(device, np.zeros(shape, np.float32), grad)

    q, k, v, g, s = t(4, 2, 4, 8), t(4, 2, 2, 8), t(4, 2, 2, 6), t(1, 4), t(2, 4, 8, 6)
    linear_attention(q, k, v, g, s, t(4, 2, 1))
    for bad in ((t(4, 2, 32), k, v, g, s, None), (q, t(4, 2, 3, 8), t(4, 2, 3, 6), g, s, None), (q, t(4, 2, 2, 7), v, g, s, None),
                (q, k, t(3, 2, 2, 6), g, s, None), (q, k, v, t(1, 2), s, None), (q, k, v, g, t(2, 4, 6, 8), None),
                (q, k, v, g, s, t(4, 2)), (t(4, 2, 4, 129), t(4, 2, 2, 129), v, g, None, None)):
        with pytest.raises(ValueError):
            linear_attention(*bad)
    with pytest.raises(ValueError):
        linear_attention_step(t(2, 4, 8), t(2, 2, 8), t(2, 2, 6), g, None)
    with pytest.raises(RuntimeError):
        linear_attention_step(t(2, 4, 8, grad=True), t(2, 2, 8), t(2, 2, 6), g, s)


# T, B, H, G, K, V, steps, resets, state, dfinal.  Sweeps that run through several
# chunks and leave the states at every 256th step (256 heads and more), and ones
# cut into segments of three to eight chunks, with widths of unlike tiles.
LONG = [
    (300, 32, 8, 4, 8, 12, True, 0.01, True, True),
    (600, 64, 4, 4, 16, 8, False, 0.005, True, True),
    (513, 86, 3, 1, 5, 33, True, None, True, False),
    (767, 128, 2, 2, 4, 4, True, 0.003, False, True),
    (700, 25, 4, 2, 16, 24, True, 0.01, True, True),
    (1500, 2, 6, 3, 40, 72, True, 0.003, True, True),
    (1500, 2, 6, 3, 40, 72, False, None, True, False),
    (1111, 7, 3, 1, 33, 9, False, 0.002, False, True),
]


@pytest.mark.parametrize("case", LONG, ids=lambda c: "-".join(str(x) for x in c))
def test_many_chunks_match_the_oracle(device, case):
    T, B, H, G, K, V = case[:6]
    x, dout, dfinal = _inputs(T + B, *case)
    if x["done"] is not None:  # resets at the ends of segments and beside them
        for i, t in enumerate((95, 96, 97, 255, 256, 257, 511, 512, 513)):
            if t < T:
                x["done"][t, i % B] = 1
    got = _run(device, x, dout, dfinal)
    _check(got, *_wanted(x, dout, dfinal), K + V + T / 8 + 256)


def test_many_chunks_at_any_alignment(device):
    for case in ((300, 32, 8, 4, 8, 12, True, 0.01, True, True), (700, 25, 4, 2, 16, 24, True, 0.01, True, True)):
        x, dout, dfinal = _inputs(3, *case)
        got = _run(device, x, dout, dfinal, offset=1)
        _check(got, *_wanted(x, dout, dfinal), case[4] + case[5] + case[0] / 8 + 256)


def test_a_state_stepped_before_the_backward_is_refused(device):
    """The backward reads the state that entered and, for the final state's
    part of the decay's gradient, the one that left: a token step in place
    between forward and backward must not spoil gradients in silence."""
    from ttrl_amd.engine.autograd import Tensor, backward_from, no_grad
    from ttrl_amd.engine.ops import linear_attention, linear_attention_step
    from ttrl_amd.engine.tensor import DeviceArray

    x, dout, dfinal = _inputs(50, 40, 2, 2, 2, 8, 8, True, None, True, True)
    eager = _run(device, x, dout, dfinal)

    def forward():
        t = {n: _tensor(device, x[n], True) for n in ("q", "k", "v", "log_decay")}
        both = DeviceArray(device, (2,) + x["state"].shape)  # two states of one allocation
        both.upload(np.stack([x["state"]] * 2))
        n = x["state"].size
        t["state"], other = (Tensor(both.view(i * n, x["state"].shape)) for i in range(2))
        out, final = linear_attention(*t.values())
        return t, other, out, final, [(out, _tensor(device, dout, False)), (final, _tensor(device, dfinal, False))]

    def act(state):
        with no_grad():
            linear_attention_step(*(_tensor(device, x[n][0], False) for n in ("q", "k", "v", "log_decay")), state)

    t, other, out, final, seeds = forward()
    act(t["state"])
    with pytest.raises(RuntimeError, match="in place"):
        backward_from(seeds)
    t, other, out, final, seeds = forward()
    act(Tensor(final.data))
    with pytest.raises(RuntimeError, match="in place"):
        backward_from(seeds)
    # what the backward does not read may be stepped
    t, other, out, final, seeds = forward()
    act(other)
    backward_from(seeds)
    for n in ("q", "k", "v", "log_decay"):
        assert np.array_equal(t[n].grad.numpy(), eager[n]), n
    act(t["state"])  # and the state itself once it is done
    t, other, out, final, seeds = forward()
    act(Tensor(final.data))
    backward_from(seeds[:1])
    want, bound = _wanted(x, dout, None)
    for n in ("q", "k", "v", "log_decay"):
        _check({n: t[n].grad.numpy()}, {n: want[n]}, {n: bound[n]}, 8 + 8 + 5 + 256)


@pytest.mark.parametrize("T,B,resets,state", [(90, 57, None, False), (255, 8, 0.01, True), (1000, 256, 0.002, True), (1000, 2, None, True)])
def test_a_shared_decay_of_short_memory(device, T, B, resets, state):
    """The gradient of a decay that all steps share sums pairs of steps (i, j)
    with a weight of i - j, a few steps where memory is short: rounding must not
    be carried over the sequence instead.  Tolerance: every pair's terms are off
    by K u and less in the mean (u = 2^-24), and what 32 steps sum of them may
    cancel, so 32 + K of u times the root of the sum of squares of the steps'
    terms |q . dq| + |k . dk|."""
    K, V = 16, 16
    x, dout, _ = _inputs(60, T, B, 1, 1, K, V, False, resets, state, False)
    x["log_decay"][:] = np.log(0.75)
    got = _run(device, x, dout, None)
    want, _ = _wanted(x, dout, None)
    term = np.abs(x["q"] * want["q"]).sum(-1) + np.abs(x["k"] * want["k"]).sum(-1)
    err = abs(float(got["log_decay"][0, 0]) - float(want["log_decay"][0, 0]))
    assert err <= (32 + K) * U * float(np.sqrt((term ** 2).sum())) + 2 * U * abs(float(want["log_decay"][0, 0]))


def test_more_lanes_than_a_launch_counts(device):
    """One step of more lanes and heads than a launch has workgroups of 256
    threads for, with decays and resets, token by token and as a sequence."""
    from ttrl_amd.engine.autograd import backward_from
    from ttrl_amd.engine.ops import linear_attention, linear_attention_step

    B = (1 << 24) + 70
    rng = np.random.default_rng(70)

    def normal(*s):
        return np.resize(rng.standard_normal(100003).astype(np.float32), s)

    q, k, v, s = normal(B, 1, 1), normal(B, 1, 1), normal(B, 1, 1), normal(B, 1, 1, 1)
    g, done = np.full((1, 1), -0.5, np.float32), np.resize(np.float32([0, 0, 1]), (B, 1))
    state = _tensor(device, s, False)
    out = linear_attention_step(*(_tensor(device, a, False) for a in (q, k, v, g)), state, _tensor(device, done, False), scale=1.0)
    keep = (np.float32(np.exp(np.float32(-0.5))) * (done <= 0))[..., None]
    want = keep * s[..., 0] + k * v
    size = np.abs(keep * s[..., 0]) + np.abs(k * v)
    assert (np.abs(state.numpy()[..., 0] - want) <= 4 * U * size).all()
    assert (np.abs(out.numpy() - q * want) <= 6 * U * np.abs(q) * size).all()

    B = 1 << 24
    x = {n: _tensor(device, a[:B].reshape((1,) * lead + a[:B].shape), True) for n, a, lead in
         (("q", q, 1), ("k", k, 1), ("v", v, 1), ("state", s, 0))}
    decay = _tensor(device, g, True)
    out, _ = linear_attention(x["q"], x["k"], x["v"], decay, x["state"], _tensor(device, done[None, :B], False), scale=1.0)
    backward_from([(out, _tensor(device, np.ones((1, B, 1, 1), np.float32), False))])
    terms = (q * keep * s[..., 0])[:B].astype(np.float64)
    assert abs(decay.grad.numpy()[0, 0] - terms.sum()) <= 64 * U * np.sqrt((terms ** 2).sum()) + 2 * U * abs(terms.sum())
