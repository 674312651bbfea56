"""Inputs of the measured cases of the gated projections have gradients that
rounding cannot decide: where relu's gate lies near zero nothing is asked of it."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def cases():
    path = Path(__file__).resolve().parents[1] / "perf" / "operators.py"
    spec = importlib.util.spec_from_file_location("operator_cases", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


# Sizes and seeds at which plain form and float64 parted by 2.9e-5 and 1.3e-4.
@pytest.mark.parametrize("rows,width,hidden,bias,seed", [(4974, 64, 4096, False, 1011), (7218, 128, 4096, True, 1026)])
def test_relu_gradients_have_one_value(cases, rows, width, hidden, bias, seed):
    """Tolerance: float32's rounding over sums of up to 8192 terms, 2e-6 of a
    gradient's norm (a product's mean error is under 2^-24, and errors of a sum's
    terms add up as their root); one gate that flips is 1e-5 and more."""
    case = {"kind": "gated", "rows": rows, "in": width, "hidden": hidden, "act": "relu", "bias": bias}
    inputs = cases._gated_inputs(case, seed)
    gate = inputs["x"].double() @ inputs["w_gate"].double()
    if bias:
        gate += inputs["b_gate"].double()
    near = gate.abs() < 1e-4
    asked = inputs["dout"] != 0
    assert near.any() and not (asked & near).any() and (asked | near).double().mean() > 0.9999  # few of the others
    plain, exact = cases._plain_gated_grads(inputs, "relu"), cases.exact(case, seed)
    for name, want in exact["grads"].items():
        assert float((plain["grads"][name].double() - want).norm() / want.norm()) < 2e-6, name
