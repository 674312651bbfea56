"""AdamW over many tensors on the GPU against the float64 oracle and, for the
8-bit moments, against the same float32 steps on the host: the kernel rounds
every product and sum on its own, so codes and scales are the host's bit for
bit.

Tolerance of the float64 comparison, before the first run (u = 2^-24): m and v
take three roundings a step, the step eight, so a parameter after s steps is
off by at most 16 s u (|p| + lr s), a moment by 8 s u of its absolute terms."""

from __future__ import annotations

import math

import numpy as np
import pytest

from oracle import sequence as O

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
LR, BETAS, EPS, WD = 3e-3, (0.9, 0.99), 1e-8, 0.05


def _tensors(device, shapes, seed, offset=0):
    from ttrl_amd.engine.autograd import Tensor
    from ttrl_amd.engine.tensor import DeviceArray

    rng = np.random.default_rng(seed)
    out = []
    for i, s in enumerate(shapes):
        n = int(np.prod(s))
        at = (offset + i) % 4 if offset else 0
        view = DeviceArray(device, (n + at,)).view(at, s)
        view.upload(rng.standard_normal(s).astype(np.float32))
        out.append(Tensor(view, True))
    return out


def _set_grads(device, params, grads):
    from ttrl_amd.engine.tensor import to_device

    for p, g in zip(params, grads):
        p.zero_grad()
        p.grad = to_device(g, device)


def _grads(rng, shapes):
    return [(0.1 * rng.standard_normal(s) * np.exp(rng.standard_normal(s))).astype(np.float32) for s in shapes]


ODD = [(1, 1), (3,), (64,), (65, 1), (7, 9, 5), (1, 63), (200, 33), (4096,), (4097,), (1, 1, 1, 32)]
MANY = [(1 + i % 7, 1 + (5 * i) % 11) for i in range(150)]


@pytest.mark.parametrize("shapes,offset", [(ODD, 0), (ODD, 1), (MANY, 0), ([(5, 5)], 0)])
def test_32_bits_match_the_oracle(device, shapes, offset):
    from ttrl_amd.engine.optim import AdamW

    params = _tensors(device, shapes, 1, offset)
    ref = [(p.numpy().astype(np.float64), np.zeros(p.shape), np.zeros(p.shape)) for p in params]
    opt = AdamW(params, lr=LR, betas=BETAS, eps=EPS, weight_decay=WD)
    rng = np.random.default_rng(2)
    for t in range(1, 4):
        grads = _grads(rng, shapes)
        _set_grads(device, params, grads)
        opt.step()
        ref = [O.adamw(p, g, m, v, t, LR, BETAS, EPS, WD) for (p, m, v), g in zip(ref, grads)]
    assert opt.t == 3
    m, v = opt.moments()
    for p, mi, vi, (rp, rm, rv) in zip(params, m, v, ref):
        assert (np.abs(p.numpy() - rp) <= 16 * 3 * U * (np.abs(rp) + 3 * LR)).all()
        assert (np.abs(mi.numpy() - rm) <= 8 * 3 * U * 3).all()
        assert (np.abs(vi.numpy() - rv) <= 8 * 3 * U * rv + 1e-30).all()


def _host_step(p, g, m, v, t):
    """The kernel's float32 steps; -> (p, m, v)."""
    f = np.float32
    b1, b2 = BETAS
    bc1, bc2 = 1.0 - b1 ** t, 1.0 - b2 ** t
    m = m * f(b1) + g * f(1.0 - b1)
    v = v * f(b2) + (g * g) * f(1.0 - b2)
    step = m / (np.sqrt(v) * f(1.0 / math.sqrt(bc2)) + f(EPS)) * f(LR / bc1)
    return p * f(1.0 - LR * WD) - step, m, v


@pytest.mark.parametrize("shapes,offset", [(ODD, 0), (ODD, 1), (MANY, 0)])
def test_8_bits_match_the_host_bit_for_bit(device, shapes, offset):
    from ttrl_amd.engine.optim import AdamW

    params = _tensors(device, shapes, 3, offset)
    opt = AdamW(params, lr=LR, betas=BETAS, eps=EPS, weight_decay=WD, state_bits=8)
    host = [p.numpy().reshape(-1) for p in params]
    held = [(O.hold_m(np.zeros_like(p)), O.hold_v(np.zeros_like(p))) for p in host]
    rng = np.random.default_rng(4)
    for t in range(1, 5):
        grads = _grads(rng, shapes)
        if t == 2:
            grads = [np.where(np.arange(g.size).reshape(g.shape) % 3 == 0, np.float32(0), g) for g in grads]
        _set_grads(device, params, grads)
        opt.step()
        for i, g in enumerate(grads):
            (cm, sm), (cv, sv) = held[i]
            host[i], m, v = _host_step(host[i], g.reshape(-1), O.held_m(cm, sm), O.held_v(cv, sv), t)
            held[i] = O.hold_m(m), O.hold_v(v)
    state = opt.state_dict()
    m, v = opt.moments()
    for i, p in enumerate(params):
        (cm, sm), (cv, sv) = held[i]
        assert np.array_equal(p.numpy().reshape(-1), host[i])
        assert np.array_equal(state["m"][i].reshape(-1), cm) and np.array_equal(state["v"][i].reshape(-1), cv)
        assert np.array_equal(state["m_scale"][i], sm) and np.array_equal(state["v_scale"][i], sv)
        assert np.array_equal(m[i].numpy().reshape(-1), O.held_m(cm, sm))
        assert np.array_equal(v[i].numpy().reshape(-1), O.held_v(cv, sv))


@pytest.mark.parametrize("bits", [32, 8])
def test_zero_gradients_decay_alone(device, bits):
    from ttrl_amd.engine.optim import AdamW

    params = _tensors(device, [(70,)], 6)
    before = params[0].numpy()
    opt = AdamW(params, lr=LR, weight_decay=WD, state_bits=bits)
    _set_grads(device, params, [np.zeros(70, np.float32)])
    opt.step()
    assert np.array_equal(params[0].numpy(), before * np.float32(1.0 - LR * WD))
    assert not any(a.numpy().any() for side in opt.moments() for a in side)


@pytest.mark.parametrize("bits", [32, 8])
def test_what_is_not_finite_spoils_its_element_or_block(device, bits):
    from ttrl_amd.engine.optim import AdamW

    shapes = [(200,), (10,)]
    clean = None
    for bad in (0.0, np.nan, np.inf):
        params = _tensors(device, shapes, 7)
        opt = AdamW(params, lr=LR, state_bits=bits)
        for s in range(2):
            grads = _grads(np.random.default_rng(8 + s), shapes)
            grads[0][100] = bad
            _set_grads(device, params, grads)
            opt.step()
        got = [p.numpy() for p in params]
        if clean is None:
            clean = got
            continue
        keep = np.ones(200, bool)
        keep[slice(64, 128) if bits == 8 else slice(100, 101)] = False
        assert np.array_equal(got[0][keep], clean[0][keep]) and np.array_equal(got[1], clean[1])
        assert not np.isfinite(got[0][100])


@pytest.mark.parametrize("bits", [32, 8])
def test_a_checkpoint_resumes_bit_for_bit(device, bits):
    from ttrl_amd.engine.optim import AdamW

    shapes, ends = ODD[:6], []
    for resume in (False, True):
        params = _tensors(device, shapes, 9)
        opt = AdamW(params, lr=LR, betas=BETAS, state_bits=bits)
        for s in range(4):
            if resume and s == 2:
                saved, opt = opt.state_dict(), AdamW(params, lr=1.0, state_bits=bits)
                opt.load_state_dict(saved)
            _set_grads(device, params, _grads(np.random.default_rng(s), shapes))
            opt.step()
        ends.append([p.numpy() for p in params])
    assert all(np.array_equal(a, b) for a, b in zip(*ends))


@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_step_counts_by_itself(device, bits):
    from ttrl_amd.engine.optim import AdamW
    from ttrl_amd.engine.ops import mean_all, square, sub
    from ttrl_amd.engine.autograd import Tensor
    from ttrl_amd.engine.step import TrainStep

    ends = []
    for mode in ("eager", "graph"):
        params = _tensors(device, [(9, 8), (1, 8)], 10)
        opt = AdamW(params, lr=LR, betas=BETAS, state_bits=bits)
        x = {"y": Tensor.from_numpy(np.ones((9, 8), np.float32), device)}

        def body(x):
            loss = mean_all(square(sub(params[0] + params[1], x["y"])))
            loss.backward()
            return {}

        with TrainStep(body, x, device, optimizer=opt, mode=mode) as step:
            for _ in range(5):
                step.run()
            assert opt.t == 5
            ends.append([p.numpy() for p in params])
    assert all(np.array_equal(a, b) for a, b in zip(*ends))


def test_refusals(device):
    from ttrl_amd.engine.optim import AdamW

    params = _tensors(device, [(4, 4), (3,)], 11)
    for kw in ({"lr": 0.0}, {"betas": (1.0, 0.9)}, {"eps": 0.0}, {"weight_decay": -1.0}, {"state_bits": 16}):
        with pytest.raises(ValueError):
            AdamW(params, **kw)
    with pytest.raises(ValueError):
        AdamW([])
    with pytest.raises(ValueError):
        AdamW([params[0], params[0]])
    opt = AdamW(params, state_bits=8)
    with pytest.raises(RuntimeError):
        opt.step()
    with pytest.raises(ValueError):
        opt.load_state_dict(AdamW(params).state_dict())
    state = opt.state_dict()
    state["m"] = [a.astype(np.float32) for a in state["m"]]
    with pytest.raises(ValueError):
        opt.load_state_dict(state)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_what_is_not_finite_stays_in_the_moments(device, bad):
    """In 8 bits a gradient that is not finite spoils both moments of its block
    and no others', and they stay spoilt."""
    from ttrl_amd.engine.optim import AdamW

    shapes, at = [(200,), (10,)], 100
    ends = []
    for value in (0.0, bad):
        params = _tensors(device, shapes, 7)
        opt = AdamW(params, lr=LR, state_bits=8)
        held = []
        for s in range(3):
            grads = _grads(np.random.default_rng(8 + s), shapes)
            if s == 1:
                grads[0][at] = value
            _set_grads(device, params, grads)
            opt.step()
            held.append([[a.numpy() for a in side] for side in opt.moments()])
        ends.append((held, opt.state_dict()))
    (clean, _), (got, state) = ends
    block = np.zeros(200, bool)
    block[64:128] = True
    for s in range(3):
        for side in range(2):
            a, b = got[s][side], clean[s][side]
            assert np.array_equal(a[1], b[1]) and np.array_equal(a[0][~block], b[0][~block])
            assert s == 0 or not np.isfinite(a[0][block]).any(), (s, side)
    for name in ("m_scale", "v_scale"):
        assert not np.isfinite(state[name][0][1]) and np.isfinite(state[name][0][[0, 2, 3]]).all()


# A set large enough that a workgroup takes four rounds, beside odd tensors off
# 16 bytes; and one of 69 workgroups, which share the desks where they take tickets.
LARGE = [(2053, 2049), (3, 1001), (77,), (1, 4096)]
SHARED = [(200, 301), (9, 1000), (5,)]


@pytest.mark.parametrize("shapes,offset,steps", [(LARGE, 0, 2), (LARGE, 1, 2), (SHARED, 0, 6), (SHARED, 1, 6)])
@pytest.mark.parametrize("bits", [32, 8])
def test_large_sets_match_the_host_bit_for_bit(device, shapes, offset, steps, bits):
    from ttrl_amd.engine.optim import AdamW

    params = _tensors(device, shapes, 13, offset)
    opt = AdamW(params, lr=LR, betas=BETAS, eps=EPS, weight_decay=WD, state_bits=bits)
    host = [(p.numpy().reshape(-1), np.zeros(p.data.numel, np.float32), np.zeros(p.data.numel, np.float32)) for p in params]
    rng = np.random.default_rng(14)
    for t in range(1, steps + 1):
        grads = _grads(rng, shapes)
        _set_grads(device, params, grads)
        opt.step()
        host = [_host_step(p, g.reshape(-1), m, v, t) for (p, m, v), g in zip(host, grads)]
        if bits == 8:
            host = [(p, O.held_m(*O.hold_m(m)), O.held_v(*O.hold_v(v))) for p, m, v in host]
    m, v = opt.moments()
    for i, (p, hm, hv) in enumerate(host):
        for name, a, b in (("p", params[i], p), ("m", m[i], hm), ("v", v[i], hv)):
            assert np.array_equal(a.numpy().reshape(-1), b), (i, name)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_captured_step_of_many_workgroups_counts_by_itself(device, bits):
    from ttrl_amd.engine.autograd import Tensor
    from ttrl_amd.engine.ops import mean_all, square, sub
    from ttrl_amd.engine.optim import AdamW
    from ttrl_amd.engine.step import TrainStep

    ends = []
    for mode in ("eager", "graph"):
        params = _tensors(device, [(200, 301), (1, 301), (200, 1)], 15)
        opt = AdamW(params, lr=LR, betas=BETAS, state_bits=bits)
        x = {"y": Tensor.from_numpy(np.ones((200, 301), np.float32), device)}

        def body(x):
            loss = mean_all(square(sub(params[0] + params[1] + params[2], x["y"])))
            loss.backward()
            return {}

        with TrainStep(body, x, device, optimizer=opt, mode=mode) as step:
            for _ in range(7):
                step.run()
            assert opt.t == 7
            ends.append([p.numpy() for p in params])
    assert all(np.array_equal(a, b) for a, b in zip(*ends))
