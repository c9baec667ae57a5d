"""
Gated products over microscaled 4-bit weights where x or W holds what is not finite: NaN wherever the formula gives NaN, infinities with their
signs, and every other number as ever.  Against plain numpy in 64 bits; tolerances as in test_mxfp4.py, activations' slopes up to 1.13.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

import mxfp4_plain as plain
from test_mxfp4 import ALPHA, DEV, LIMIT, f64, held, numbers, sums_bound

ACTIVATIONS = ["silu", "relu", "clamped_swish", "gelu_tanh"]
# (rows, rows of W a half, columns): codes spread in registers; x in pieces, K split between CTAs and not; codes spread into tensor memory, split
# and not; and for rows in four bits their own kernel, split and not.
SIZES = [(3, 128, 512), (12, 77, 512), (9, 6000, 512), (8, 4200, 2048), (33, 2600, 4096), (40, 150, 512), (100, 4900, 512), (300, 2500, 136)]


@pytest.fixture(scope="module")
def ops():
    from tinyserve_llm_b200.ops import get_ops
    return get_ops()


def expected(xv, values, act):
    """What the formula gives, and how far off a kernel may be where that is finite."""
    with np.errstate(invalid="ignore", over="ignore"):
        y, off = xv @ values.T, sums_bound(np.nan_to_num(xv, nan=0.0, posinf=0.0, neginf=0.0), np.nan_to_num(values, nan=0.0), xv.shape[1])
        half = y.shape[1] // 2
        g, u, dg, du = y[:, :half], y[:, half:], off[:, :half], off[:, half:]
        want = plain.gated(act, g, u, LIMIT, ALPHA)
        factor = np.abs(plain.gated(act, g, np.zeros_like(g) if act == "clamped_swish" else np.ones_like(g), LIMIT, ALPHA))
        top = np.abs(np.clip(u, -LIMIT, LIMIT)) if act == "clamped_swish" else np.abs(u)
        slack = 1.13 * dg * (top + 1) + factor * du + 1.13 * dg * du + 2.0 ** -16 * np.abs(want)
        return want, slack + 2.0 ** -8 * (np.abs(want) + slack)


def compare(got, want, slack):
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
    np.testing.assert_array_equal(np.where(np.isinf(got), got, 0.0), np.where(np.isinf(want), want, 0.0))
    finite = np.isfinite(want) & np.isfinite(slack)
    assert (np.abs(got[finite] - want[finite]) <= slack[finite]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("both", [False, True], ids=["rows16", "rows4"])
@pytest.mark.parametrize("act", ACTIVATIONS)
@pytest.mark.parametrize("m, inter, k", SIZES)
def test_nans_of_rows_gates_and_ups(ops, m, inter, k, act, both):
    """A NaN in a row of x; blocks of W that are NaN in a gate's row, in an up's, in both of an output."""
    x, w = numbers((m, k), torch.bfloat16, m + k), f64(numbers((2 * inter, k), torch.float32, inter + k, 2.0 / k ** 0.5))
    x[1, 70] = float("nan")
    w[3, 100], w[inter + 7, 33], w[11, 5], w[inter + 11, 60] = [float("nan")] * 4
    values = plain.rounded(w)
    xv = plain.rounded(f64(x)) if both else f64(x)
    want, slack = expected(xv, values, act)
    nan = np.zeros((m, inter), dtype=bool)
    nan[1], nan[:, [3, 7, 11]] = True, True
    np.testing.assert_array_equal(np.isnan(want), nan)
    rows = ops.quantize_mxfp4(x.to(DEV)) if both else x.to(DEV)
    compare(f64(ops.linear_gated_mxfp4(rows, held(w, DEV), act, LIMIT, ALPHA)), want, slack)
    ops.check_device_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("act", ACTIVATIONS)
@pytest.mark.parametrize("m, inter, k", SIZES)
def test_infinite_numbers_through_activations(ops, m, inter, k, act):
    x, w = numbers((m, k), torch.bfloat16, m + k), f64(numbers((2 * inter, k), torch.float32, inter + k, 2.0 / k ** 0.5))
    x[0, 70], x[1, 5], x[1, 40], x[2, 3], x[2, 4] = float("inf"), float("inf"), float("-inf"), float("-inf"), float("nan")
    values = plain.rounded(w)
    want, slack = expected(f64(x), values, act)
    compare(f64(ops.linear_gated_mxfp4(x.to(DEV), held(w, DEV), act, LIMIT, ALPHA)), want, slack)
    ops.check_device_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("act", ACTIVATIONS)
def test_nans_through_the_activation_alone(ops, act, dtype):
    """The elementwise kernel, and the products over bfloat16 weights that share the activations."""
    z = numbers((4, 16), dtype, 5)
    z[0, 2], z[1, 10], z[2, 3], z[2, 11] = [float("nan")] * 4
    got = ops.gated_activation(z.to(DEV), act, LIMIT, ALPHA)
    want = np.zeros((4, 8), dtype=bool)
    want[[0, 1, 2], [2, 2, 3]] = True
    np.testing.assert_array_equal(np.isnan(f64(got)), want)
    for m in (4, 40, 600):
        x, w = numbers((m, 64), dtype, 6).to(DEV), numbers((2 * 256, 64), dtype, 7).to(DEV)
        x[1, 5] = float("nan")
        w[3, 5] = float("nan")
        y = f64(ops.linear_gated(x, w, act, LIMIT, ALPHA))
        want = np.zeros((m, 256), dtype=bool)
        want[1], want[:, 3] = True, True
        np.testing.assert_array_equal(np.isnan(y), want)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["relu2", "xielu", "tanh"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_nans_through_activations_of_one_argument(ops, dtype, kind):
    """The elementwise kernel, products with the activation in their epilogue and not, and a projection held in four bits."""
    from tinyserve_llm_b200.parts.base import Runtime
    from tinyserve_llm_b200.parts.linear import QuantizedLinear
    z = numbers((3, 40), dtype, 5)
    z[0, 2], z[1, 0] = float("nan"), float("nan")
    np.testing.assert_array_equal(np.isnan(f64(ops.unary_activation(z.to(DEV), kind, 0.8, 0.8))), np.isnan(f64(z)))
    for m in (4, 40, 300):
        x, w = numbers((m, 128), dtype, 6).to(DEV), numbers((256, 128), dtype, 7).to(DEV)
        x[1, 5] = float("nan")
        w[3, 5] = float("nan")
        want = np.zeros((m, 256), dtype=bool)
        want[1], want[:, 3] = True, True
        np.testing.assert_array_equal(np.isnan(f64(ops.linear_unary(x, w, kind, 0.8, 0.8))), want)
        if dtype == torch.bfloat16:
            held_in_four = QuantizedLinear(w, Runtime(torch.bfloat16, torch.device(DEV), ops, weight_format="mxfp4"))
            np.testing.assert_array_equal(np.isnan(f64(held_in_four.unary(x, kind, 0.8, 0.8))), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("pairs", [3, 40, 2000])
def test_nans_through_squares_of_experts(ops, pairs, dtype):
    x, w = numbers((pairs, 64), dtype, 8).to(DEV), numbers((2, 48, 64), dtype, 9).to(DEV)
    x[1, 5] = float("nan")
    offsets = torch.tensor([0, pairs // 2 + 1, pairs], dtype=torch.int32, device=DEV)
    got = f64(ops.moe_linear(x, w, offsets, None, 1, pairs, "relu2"))
    want = np.zeros((pairs, 48), dtype=bool)
    want[1] = True
    np.testing.assert_array_equal(np.isnan(got), want)
