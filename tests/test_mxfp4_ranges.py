"""
Products over microscaled 4-bit weights whose bfloat16 rows hold numbers far apart: every kernel multiplies a bfloat16 number as it is, whatever
stands in its block of 32.  Against plain numpy in 64 bits.

Tolerance.  A number is one to three terms: itself, or three pieces of eight bits that add up to it exactly, none larger than 1.25 times the
number.  So a sum has at most 3 K terms, whose magnitudes come to no more than twice S, the sum of the products' magnitudes.  Tensor cores
add 16 or more terms at a time, each addition off by at most 2^-22 of what stands there: (3 K / 16 + 8) 2^-22 times 2 S.  Numbers that are in
no piece are added one by one, K additions at most, each off by 2^-24 of S.  Both together stay under (2 K + 64) 2^-23 S.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

import mxfp4_plain as plain
from test_mxfp4 import ALPHA, DEV, LIMIT, check, f64, numbers
from tinyserve_llm_b200.ops import MXFP4


@pytest.fixture(scope="module")
def ops():
    from tinyserve_llm_b200.ops import get_ops
    return get_ops()


# (rows, rows of W, columns).  The kernel that spreads codes in registers; three pieces a row, tiles of 8, 16, 32 and 64 rows of x, K split
# between CTAs and not, more tiles than SMs; codes spread into tensor memory.
REGISTERS = [(3, 512, 512), (12, 300, 512), (7, 1300, 8192)]
PIECES = [(5, 9000, 2048), (8, 9600, 1792), (9, 12000, 512), (16, 1300, 4224), (20, 1300, 4224), (24, 9600, 1792), (33, 5200, 4096), (64, 2400, 8832),
          (50, 9600, 4096), (40, 19200, 4096)]
SPREAD = [(100, 300, 512), (300, 520, 520), (20, 2560, 2304), (64, 130, 65536), (40, 2603, 2048), (200, 2500, 2176), (200, 9400, 640)]
SIZES = REGISTERS + PIECES + SPREAD


def bound(x, w, k):
    return (2 * k + 64) * 2.0 ** -23 * (np.abs(x) @ np.abs(w).T)


def far_apart(m, k, every, seed):
    """Rows of numbers around one with a number 2^9 to 2^24 times as large in one block of `every`; and which column of a block it is in."""
    x = numbers((m, k), torch.float32, seed)
    column = 5
    for i in range(m):
        for n, block in enumerate(range(i % every, k // 32, every)):
            x[i, 32 * block + column] = (1.0 + 0.37 * (n % 3)) * 2.0 ** (9 + (i + n) % 16) * (-1) ** n
    return x.to(torch.bfloat16), column


def matrix(codes: np.ndarray, scales: np.ndarray, k: int) -> MXFP4:
    """A matrix of the given codes [rows, k] and scales [rows, k / 32], in rows of full blocks or with a last one that ends early."""
    n, blocks = scales.shape
    packed = np.zeros((n, blocks * 32), dtype=np.uint8)
    packed[:, :k] = codes
    wide = torch.zeros((n, -(-blocks // 16) * 16), dtype=torch.uint8, device=DEV)
    wide[:, :blocks] = torch.from_numpy(scales).to(DEV)
    return MXFP4(torch.from_numpy(packed[:, 0::2] | (packed[:, 1::2] << 4)).to(DEV), wide[:, :blocks], k)


def weights(n, k, column, seed):
    """W, and its values, with nothing in every other row at the columns where x is large: what is small in x is then all that counts."""
    gen, blocks = np.random.default_rng(seed), -(-k // 32)
    codes, scales = gen.integers(0, 16, (n, k), dtype=np.uint8), gen.integers(114, 121, (n, blocks), dtype=np.uint8)
    codes[::2, column::32] = 0
    padded = np.zeros((n, blocks * 32), dtype=np.uint8)
    padded[:, :k] = codes
    return matrix(codes, scales, k), plain.values(padded.reshape(n, blocks, 32), scales, k)


def one_a_row(n, k, at, code):
    """W with one number a row, at column `at` of it, under scale 1."""
    codes = np.zeros((n, k), dtype=np.uint8)
    codes[np.arange(n), at] = code
    return matrix(codes, np.full((n, -(-k // 32)), 127, dtype=np.uint8), k)


@pytest.mark.gpu
@pytest.mark.parametrize("every", [1, 7], ids=["each block", "some blocks"])
@pytest.mark.parametrize("m, n, k", SIZES)
def test_small_numbers_beside_large_ones(ops, m, n, k, every):
    x, column = far_apart(m, k, every, m + k)
    weight, values = weights(n, k, column, n + k)
    xv = f64(x)
    want, off = xv @ values.T, bound(xv, values, k)
    check(ops.linear_mxfp4(x.to(DEV), weight, out_dtype=torch.float32), want, off)
    check(ops.linear_mxfp4(x.to(DEV), weight), want, off)
    torch.cuda.synchronize()
    ops.check_device_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("m, inter, k", [(3, 256, 512), (8, 4200, 2048), (9, 6000, 512), (24, 4800, 1792), (64, 1301, 2048), (40, 2600, 4096),
                                         (33, 9601, 4096), (200, 4700, 640), (100, 150, 512)])
def test_gated_small_numbers_beside_large_ones(ops, m, inter, k):
    x, column = far_apart(m, k, 3, m + k)
    weight, values = weights(2 * inter, k, column, inter + k)
    xv = f64(x)
    y, off = xv @ values.T, bound(xv, values, k)
    g, u, dg, du = y[:, :inter], y[:, inter:], off[:, :inter], off[:, inter:]
    want = plain.gated("clamped_swish", g, u, LIMIT, ALPHA)
    factor = np.abs(plain.gated("clamped_swish", g, np.zeros_like(g), LIMIT, ALPHA))
    slack = 1.13 * dg * (np.abs(np.clip(u, -LIMIT, LIMIT)) + 1) + factor * du + 1.13 * dg * du + 2.0 ** -16 * np.abs(want)
    check(ops.linear_gated_mxfp4(x.to(DEV), weight, "clamped_swish", LIMIT, ALPHA), want, slack)
    torch.cuda.synchronize()
    ops.check_device_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("m, n, k", SIZES)
def test_numbers_of_every_size(ops, m, n, k):
    """Exponents from bfloat16's smallest subnormal numbers up, drawn at random: products with rows of W that hold one number are exact."""
    gen = torch.Generator().manual_seed(m + n)
    bits = torch.randint(0, 0x6f80, (m, k), generator=gen, dtype=torch.int32) | (torch.randint(0, 2, (m, k), generator=gen, dtype=torch.int32) << 15)
    x = bits.to(torch.int16).view(torch.bfloat16)                                # up to 2^96
    rows = np.arange(n)
    at = (rows * 37) % k
    want = f64(x)[:, at] * np.where(rows % 3 == 0, 1.0, -1.5)
    got = f64(ops.linear_mxfp4(x.to(DEV), one_a_row(n, k, at, np.where(rows % 3 == 0, 2, 11)), out_dtype=torch.float32))
    normal = np.abs(want) >= 2.0 ** -126                                          # below, a product may be flushed or not
    np.testing.assert_array_equal(got[normal], want[normal])
    assert (np.abs(got[~normal]) <= 2.0 ** -126).all()
    ops.check_device_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("m, n, k", SIZES)
def test_the_largest_numbers(ops, m, n, k):
    """bfloat16's largest number times one is itself, though its first piece alone, rounded up, is past float32's range."""
    x = numbers((m, k), torch.bfloat16, 3)
    top = torch.finfo(torch.bfloat16).max
    x[0, 37], x[1, 38] = top, -top
    at = 37 + np.arange(n) % 3
    got = f64(ops.linear_mxfp4(x.to(DEV), one_a_row(n, k, at, 2), out_dtype=torch.float32))
    np.testing.assert_array_equal(got, f64(x)[:, at])


@pytest.mark.gpu
@pytest.mark.parametrize("m, n, k", [(1, 9000, 2048), (2, 1300, 16384), (12, 1300, 4224), (30, 1300, 4224), (33, 5200, 4096), (9, 130, 65536)])
def test_stretches_of_wider_rows(ops, m, n, k):
    """Rows of x apart from one another, one of them with infinities and one with a NaN: each row gives what it gives by itself, in a row of its own."""
    x, column = far_apart(m, k, 5, 3)
    if m > 2:
        x[0, 70], x[0, k - 1], x[2, 40] = float("inf"), float("-inf"), float("nan")
    weight, values = weights(n, k, column, n + k)
    wide = torch.full((m, k + 72), float("nan"), dtype=torch.bfloat16)
    wide[:, 64:64 + k] = x
    part = wide.to(DEV)[:, 64:64 + k]
    assert part.stride(0) == k + 72 and part.data_ptr() % 16 == 0
    got = ops.linear_mxfp4(part, weight, out_dtype=torch.float32)
    assert torch.equal(got.nan_to_num(nan=7.0), ops.linear_mxfp4(x.to(DEV), weight, out_dtype=torch.float32).nan_to_num(nan=7.0))
    xv = f64(x)
    with np.errstate(invalid="ignore"):
        want = xv @ values.T
    np.testing.assert_array_equal(np.isnan(f64(got)), np.isnan(want))
    infinite = np.isinf(want)
    np.testing.assert_array_equal(f64(got)[infinite], want[infinite])
    finite = np.isfinite(xv).all(axis=1)
    check(got[torch.from_numpy(finite).to(DEV)], want[finite], bound(xv[finite], values, k))
    torch.cuda.synchronize()
    ops.check_device_errors()
