"""The gated projections on the GPU against the float64 oracle: outputs and
every gradient over rows, widths, activations and alignments.

Tolerance, from float32's rounding before the first run (u = 2^-24): a
projection's error is at most (K + 8) u times the sum of its absolute terms,
P.  All four activations have slopes and second derivatives of at most 1.2, so
h = act(g) u is off by at most (K + 16) u (1.2 P_g |u| + |act| P_u + |h|), and dg and
du by the same with dh; their errors and (M or N + 8) u of the absolute terms
add up in the products that follow."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import sequence as O

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def _tensor(device, a, grad=True, offset=0):
    from ttrl_amd.engine.autograd import Tensor
    from ttrl_amd.engine.tensor import DeviceArray

    view = DeviceArray(device, (a.size + offset,)).view(offset, a.shape)
    view.upload(a)
    return Tensor(view, grad)


def _inputs(seed, M, K, N, bias):
    rng = np.random.default_rng(seed)

    def normal(*s, scale=1.0):
        return (scale * rng.standard_normal(s)).astype(np.float32)

    x = {"x": normal(M, K), "w_gate": normal(K, N, scale=K ** -0.5), "w_up": normal(K, N, scale=K ** -0.5),
         "b_gate": normal(1, N) if bias else None, "b_up": normal(1, N) if bias else None}
    return x, normal(M, N)


def _run(device, x, act, dh, offset=0):
    from ttrl_amd.engine.autograd import backward_from
    from ttrl_amd.engine.ops import gated_linear

    t = {n: None if a is None else _tensor(device, a, True, offset) for n, a in x.items()}
    h = gated_linear(*t.values(), activation=act)
    got = {"out": h.numpy()}
    backward_from([(h, _tensor(device, dh, False, offset))])
    got.update({n: a.grad.numpy() for n, a in t.items() if a is not None})
    return got


def _bounds(x, act, dh):
    f = {n: None if a is None else a.astype(np.float64) for n, a in x.items()}
    size = {n: 0.0 if a is None else np.abs(a) for n, a in f.items()}
    (M, K), N = f["x"].shape, f["w_gate"].shape[1]
    g, u = O._projections(f["x"], f["w_gate"], f["w_up"], f["b_gate"], f["b_up"])
    pg, pu = size["x"] @ size["w_gate"] + size["b_gate"], size["x"] @ size["w_up"] + size["b_up"]
    a, slope = O._act(act, g)
    d = np.abs(dh.astype(np.float64))
    n = (K + 16) * U
    out = n * (1.2 * pg * np.abs(u) + np.abs(a) * pu + np.abs(a * u) + 1e-30)
    eg = n * d * (1.2 * pg * np.abs(u) + 1.2 * pu + np.abs(slope * u))  # of dg
    eu = n * d * (1.2 * pg + np.abs(a))  # of du
    ag, au = d * np.abs(u * slope), d * np.abs(a)
    xt = size["x"].T
    return {"out": out, "w_gate": xt @ (eg + (M + 8) * U * ag), "w_up": xt @ (eu + (M + 8) * U * au),
            "b_gate": (eg + (M + 8) * U * ag).sum(0, keepdims=True), "b_up": (eu + (M + 8) * U * au).sum(0, keepdims=True),
            "x": (eg + (2 * N + 8) * U * ag) @ size["w_gate"].T + (eu + (2 * N + 8) * U * au) @ size["w_up"].T}


def _check(got, x, act, dh):
    want = O.gated_backward(*x.values(), act, dh)
    want["out"] = O.gated_forward(*x.values(), act)
    lim = _bounds(x, act, dh)
    for n, a in got.items():
        err = np.abs(a.astype(np.float64) - want[n])
        assert a.shape == want[n].shape, n
        assert (err <= lim[n] + 1e-30).all(), (n, float((err / (lim[n] + 1e-30)).max()))


SIZES = [(1, 1, 1), (1, 512, 2048), (2, 64, 100), (5, 33, 7), (16, 500, 64), (17, 16, 65), (64, 128, 64), (65, 31, 129),
         (200, 100, 333), (1000, 72, 60)]


@pytest.mark.parametrize("act", ["silu", "gelu", "relu", "sigmoid"])
@pytest.mark.parametrize("M,K,N", SIZES)
def test_matches_the_oracle(device, M, K, N, act):
    x, dh = _inputs(M + K + N, M, K, N, bias=(M + N) % 2 == 1)
    if act == "relu":  # a gate that rounding decides has no float64 value
        g = O._projections(*x.values())[0]
        dh[np.abs(g) < 1e-4] = 0
    _check(_run(device, x, act, dh), x, act, dh)


@pytest.mark.parametrize("offset", [1, 2, 3])
def test_any_alignment(device, offset):
    for M in (1, 70):
        x, dh = _inputs(offset, M, 48, 96, bias=True)
        _check(_run(device, x, "silu", dh, offset), x, "silu", dh)


def test_large_rows(device):
    """Rows and widths of a training batch (the matrix-core path)."""
    x, dh = _inputs(5, 2050, 260, 516, bias=True)
    _check(_run(device, x, "gelu", dh), x, "gelu", dh)


def test_extreme_projections(device):
    """Gates far from zero saturate, they do not turn into NaN."""
    x, dh = _inputs(6, 3, 4, 8, bias=True)
    x["b_gate"][0, :4] = [200, -200, 1e4, -1e4]
    for act in ("silu", "gelu", "sigmoid"):
        got = _run(device, x, act, dh)
        assert all(np.isfinite(a).all() for a in got.values()), act
        want = O.gated_forward(*x.values(), act)
        assert np.allclose(got["out"], want, rtol=1e-4, atol=1e-5), act


@pytest.mark.parametrize("M", [3, 300])
def test_what_is_not_finite_stays_in_its_row(device, M):
    x, dh = _inputs(7, M, 32, 64, bias=False)
    clean = _run(device, x, "silu", dh)
    for bad in (np.nan, np.inf):
        y = {n: None if a is None else a.copy() for n, a in x.items()}
        y["x"][2, 5] = bad
        got = _run(device, y, "silu", dh)
        for n in ("out", "x"):
            rest = np.delete(np.arange(M), 2)
            assert np.array_equal(got[n][rest], clean[n][rest]), n
        assert not np.isfinite(got["out"][2]).any()


def test_no_rows_and_no_tape(device):
    from ttrl_amd.engine.autograd import no_grad
    from ttrl_amd.engine.ops import gated_linear

    x, dh = _inputs(8, 0, 8, 12, bias=True)
    got = _run(device, x, "silu", dh)
    assert got["out"].shape == (0, 12) and not any(got[n].any() for n in ("w_gate", "w_up", "b_gate", "b_up"))
    x, dh = _inputs(9, 40, 8, 12, bias=True)
    with no_grad():
        h = gated_linear(*(_tensor(device, a) for a in x.values()))
    assert not h.requires_grad and np.array_equal(h.numpy(), _run(device, x, "silu", dh)["out"])


def test_gradients_add_and_bias_alone(device):
    from ttrl_amd.engine.autograd import backward_from
    from ttrl_amd.engine.ops import gated_linear

    x, dh = _inputs(10, 30, 20, 24, bias=True)
    t = {n: _tensor(device, a) for n, a in x.items()}
    for _ in range(2):
        backward_from([(gated_linear(*t.values(), activation="gelu"), _tensor(device, dh, False))])
    want = O.gated_backward(*x.values(), "gelu", dh)
    lim = _bounds(x, "gelu", dh)
    for n, a in t.items():
        assert (np.abs(a.grad.numpy() - 2 * want[n]) <= 2 * lim[n] + 8 * U * np.abs(want[n])).all(), n
    only = {n: _tensor(device, a, n.startswith("b_")) for n, a in x.items()}
    backward_from([(gated_linear(*only.values(), activation="gelu"), _tensor(device, dh, False))])
    for n in ("b_gate", "b_up"):
        assert (np.abs(only[n].grad.numpy() - want[n]) <= lim[n]).all(), n
    assert only["x"].grad is None and only["w_gate"].grad is None


def test_a_captured_pass_replays(device):
    from ttrl_amd.engine.autograd import backward_from
    from ttrl_amd.engine.ops import gated_linear
    from ttrl_amd.engine.step import TrainStep

    x, dh = _inputs(11, 130, 40, 72, bias=True)
    eager = _run(device, x, "silu", dh)
    t = {n: _tensor(device, a) for n, a in x.items()}
    seed = _tensor(device, dh, False)
    made = {}

    def body(t):
        for a in t.values():
            a.zero_grad()
        made["h"] = gated_linear(*t.values())
        backward_from([(made["h"], seed)])
        return {}

    with TrainStep(body, t, device, mode="graph") as step:
        step.run()
        for _ in range(3):
            step.replay()
            device.synchronize()
            assert np.array_equal(made["h"].numpy(), eager["out"])
            for n, a in t.items():
                assert np.array_equal(a.grad.numpy(), eager[n]), n


def test_refusals(device):
    from ttrl_amd.engine.ops import gated_linear

    def t(*shape):
        return _tensor(device, np.zeros(shape, np.float32))

    for bad in ((t(2, 3), t(4, 5), t(4, 5)), (t(2, 4), t(4, 5), t(4, 6)), (t(2, 4), t(4, 5), t(4, 5), t(1, 4)),
                (t(8), t(4, 5), t(4, 5))):
        with pytest.raises(ValueError):
            gated_linear(*bad)
    with pytest.raises(ValueError):
        gated_linear(t(2, 4), t(4, 5), t(4, 5), activation="tanh")


@pytest.mark.parametrize("M", [70, 300])
def test_small_values_beside_large_ones_that_meet_zeros(device, M):
    """The largest value of every row of x, and of every row of the slopes,
    meets a weight of zero, so all of the result comes from values 1e-7 of it
    and less: the same bounds hold, in which the large ones have no part."""
    x, dh = _inputs(11, M, 64, 48, False)
    x["x"][:, 5] = 1e7
    x["w_gate"][5] = x["w_up"][5] = 0
    dh[:, 7] = 1e7
    x["w_gate"][:, 7] = x["w_up"][:, 7] = 0
    _check(_run(device, x, "sigmoid", dh), x, "sigmoid", dh)


# Products large enough to be packed forward too, in small and large tiles;
# ragged in every extent.
@pytest.mark.parametrize("M,K,N,act,bias", [(2050, 523, 517, "gelu", True), (1031, 1029, 520, "relu", False),
                                            (4100, 100, 1501, "sigmoid", True), (4100, 1500, 2100, "silu", False), (26000, 300, 260, "gelu", True)])
def test_packed_products(device, M, K, N, act, bias):
    x, dh = _inputs(M, M, K, N, bias)
    if act == "relu":
        g = O._projections(*x.values())[0]
        dh[np.abs(g) < 1e-4] = 0
    _check(_run(device, x, act, dh), x, act, dh)


@pytest.mark.parametrize("N", [517, 520])
def test_packed_products_at_any_alignment(device, N):
    x, dh = _inputs(3, 2050, 515, N, True)
    _check(_run(device, x, "silu", dh, 1), x, "silu", dh)


def test_packed_products_keep_what_is_not_finite_in_its_row(device):
    x, dh = _inputs(7, 2050, 520, 516, bias=False)
    clean = _run(device, x, "silu", dh)
    for bad in (np.nan, np.inf):
        y = {n: None if a is None else a.copy() for n, a in x.items()}
        y["x"][2, 5] = bad
        got = _run(device, y, "silu", dh)
        rest = np.delete(np.arange(2050), 2)
        for n in ("out", "x"):
            assert np.array_equal(got[n][rest], clean[n][rest]), n
        assert not np.isfinite(got["out"][2]).any()


def test_packed_products_of_small_values_beside_large_ones(device):
    """As above where the forward is packed too; and rows of very small and of
    very large values, which the rows' scales take in."""
    x, dh = _inputs(11, 2050, 520, 516, False)
    x["x"][:, 5] = 1e7
    x["w_gate"][5] = x["w_up"][5] = 0
    dh[:, 7] = 1e7
    x["w_gate"][:, 7] = x["w_up"][:, 7] = 0
    _check(_run(device, x, "sigmoid", dh), x, "sigmoid", dh)
    x, dh = _inputs(12, 2050, 520, 516, False)
    x["x"] *= np.float32(2.0) ** np.linspace(-60, 12, 2050).astype(np.float32)[:, None]
    dh *= np.float32(2.0) ** np.linspace(20, -40, 2050).astype(np.float32)[:, None]
    _check(_run(device, x, "sigmoid", dh), x, "sigmoid", dh)


def test_very_many_rows(device):
    """More rows than a grid has workgroups in y (64 rows each)."""
    x, dh = _inputs(13, 64 * 65535 + 70, 2, 3, True)
    _check(_run(device, x, "silu", dh), x, "silu", dh)


# One value of a row (the values that one output sums over) far above the rest,
# that meets zeros in every second column of the other operand: half of the sums
# have no part of it, beside others that have.
@pytest.mark.parametrize("outlier", [1e6, 1e7, 1e9, 1e12])
@pytest.mark.parametrize("product", ["forward", "input", "weight"])
@pytest.mark.parametrize("M,K,N", [(300, 64, 48), (2050, 520, 516)])
def test_large_values_that_meet_zeros_in_some_columns(device, M, K, N, product, outlier):
    x, dh = _beside(21, M, K, N, product, outlier)
    _check(_run(device, x, "sigmoid", dh), x, "sigmoid", dh)


@pytest.mark.parametrize("product,M,K,N", [("forward", 16500, 130, 600), ("input", 4100, 1500, 2100), ("weight", 4100, 1500, 2100)])
def test_large_values_that_meet_zeros_in_large_tiles(device, M, K, N, product):
    x, dh = _beside(22, M, K, N, product, 1e9)
    _check(_run(device, x, "sigmoid", dh), x, "sigmoid", dh)


def _beside(seed, M, K, N, product, outlier):
    x, dh = _inputs(seed, M, K, N, False)
    if product == "forward":
        x["x"][:, 5] = outlier
        x["w_gate"][5, 1::2] = x["w_up"][5, 1::2] = 0
    elif product == "input":
        dh[:, 7] = outlier
        x["w_gate"][1::2, 7] = x["w_up"][1::2, 7] = 0
    else:
        x["x"][11] *= np.float32(outlier)
        dh[11, 1::2] = 0
    return x, dh


def test_sums_of_nothing_but_small_values(device):
    """Inputs that are zero but for one step in a hundred, beside a gate whose
    slopes reach down to 1e-9 of their largest: sums of few or no terms."""
    x, dh = _inputs(23, 700, 90, 130, False)
    rng = np.random.default_rng(24)
    x["x"] *= rng.random(x["x"].shape) < 0.01
    dh *= np.exp(-20 * rng.random(dh.shape)).astype(np.float32)
    _check(_run(device, x, "silu", dh), x, "silu", dh)


@pytest.mark.parametrize("M,K,N", [(3, 32, 64), (300, 32, 64), (2050, 520, 516)])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_what_is_not_finite_shows_beside_zeros(device, M, K, N, bad):
    """A product of zero and NaN or infinity is NaN, whether all of a row or
    column is zero or not, in each product and at every size."""
    def clean():
        return _inputs(31, M, K, N, bias=False)

    x, dh = clean()
    x["w_gate"][:] = x["w_up"][:] = 0
    x["x"][2, 5] = bad
    out = _run(device, x, "silu", dh)["out"]
    assert np.isnan(out[2]).all() and not np.delete(out, 2, 0).any()

    x, dh = clean()
    x["w_gate"][:, 9] = x["w_up"][:, 9] = 0
    x["x"][2, 5] = bad
    out = _run(device, x, "sigmoid", dh)["out"]
    assert np.isnan(out[2, 9]) and np.isfinite(np.delete(out, 2, 0)).all()

    x, dh = clean()  # dx: a weight row of zeros beside a slope that is not finite
    x["w_gate"][4] = x["w_up"][4] = 0
    dh[1, 3] = bad
    dx = _run(device, x, "sigmoid", dh)["x"]
    assert np.isnan(dx[1, 4]) and np.isfinite(np.delete(dx, 1, 0)).all()

    x, dh = clean()  # dW: a feature of zeros beside it
    x["x"][:, 4] = 0
    dh[1, 3] = bad
    got = _run(device, x, "sigmoid", dh)
    for n in ("w_gate", "w_up"):
        assert np.isnan(got[n][4, 3]) and np.isfinite(np.delete(got[n], 3, 1)).all(), n


# Forward products whose sums are formed in several parts: few tiles, a long sum.
@pytest.mark.parametrize("M,K,N,act,bias", [(300, 1024, 1024, "silu", True), (100, 2100, 1333, "gelu", True),
                                            (70, 4099, 1021, "sigmoid", False)])
def test_packed_products_in_parts(device, M, K, N, act, bias):
    x, dh = _inputs(41, M, K, N, bias)
    _check(_run(device, x, act, dh), x, act, dh)


def test_packed_products_in_parts_at_any_alignment(device):
    x, dh = _inputs(42, 300, 1024, 1024, True)
    _check(_run(device, x, "silu", dh, 1), x, "silu", dh)


def test_very_many_columns(device):
    """More columns than a launch's threads count, forward; bias gradients of
    more columns than are summed at once."""
    from ttrl_amd.engine.autograd import no_grad
    from ttrl_amd.engine.ops import gated_linear

    N = (1 << 27) + 80
    w = [np.resize(np.random.default_rng(s).standard_normal(100003).astype(np.float32), (1, N)) for s in (1, 2)]
    with no_grad():
        h = gated_linear(_tensor(device, np.float32([[0.5]])), *(_tensor(device, a) for a in w), activation="relu").numpy()
    assert np.array_equal(h, np.maximum(np.float32(0.5) * w[0], 0) * (np.float32(0.5) * w[1]))
    x, dh = _inputs(51, 40, 3, 40001, True)
    _check(_run(device, x, "silu", dh), x, "silu", dh)
