"""
Microscaled 4-bit floating point: quantisation and back, the products whose weights (or both sides) are held in it, against plain numpy in
64 bits.

Tolerances.  Codes times scales are bfloat16 numbers exactly, products of two of them float32 numbers exactly, so a product differs from
the 64-bit one by its float32 sums alone: tensor cores add 16 (or 64) products at a time, each addition off by at most one step of the
largest addend, 2^-23 of it, so K / 16 + 8 additions are off by at most (K / 16 + 8) 2^-22 of the sum of magnitudes.  Then comes one
rounding to the output type, at most 2^-8 of the value in bfloat16.  Activations have slopes up to 1.13 and are off by less than
2^-16 of their value themselves.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

import mxfp4_plain as plain
from tinyserve_llm_b200.ops import MXFP4, KernelError

DEV = "cuda"
LIMIT, ALPHA = 7.0, 1.702


@pytest.fixture(scope="module")
def ops():
    from tinyserve_llm_b200.ops import get_ops
    return get_ops()


def numbers(shape, dtype, seed, scale=1.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=gen) * torch.exp(0.8 * torch.randn(shape[-1:], generator=gen)) * scale
    return x.to(dtype)


def held(x: np.ndarray, device="cpu", garbage=0) -> MXFP4:
    """A matrix in four bits as a loader would make it from the oracle's codes; `garbage`: what rows of scales have behind their last block."""
    codes, scales = plain.quantize(x)
    rows, blocks = scales.shape
    flat = codes.reshape(rows, -1)
    packed = torch.from_numpy(flat[:, 0::2] | (flat[:, 1::2] << 4)).to(device)
    wide = torch.full((rows, -(-blocks // 16) * 16), garbage, dtype=torch.uint8, device=device)
    wide[:, :blocks] = torch.from_numpy(scales).to(device)
    return MXFP4(packed, wide[:, :blocks], x.shape[1])


def f64(t: torch.Tensor) -> np.ndarray:
    return t.double().cpu().numpy()


def sums_bound(x, w, k):
    return (k / 16 + 8) * 2.0 ** -22 * (np.abs(x) @ np.abs(w).T)


def check(got: torch.Tensor, want: np.ndarray, bound: np.ndarray) -> None:
    assert tuple(got.shape) == want.shape
    slack = bound + (2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -24) * (np.abs(want) + bound)
    off = np.abs(f64(got) - want)
    worst = np.unravel_index(np.argmax(off - slack), off.shape) if off.size else ()
    assert not off.size or (off <= slack).all(), f"{worst}: got {f64(got)[worst]}, want {want[worst]}, off {off[worst]}, allowed {slack[worst]}"


# ------------------------------------------------------------------------------------------------------------ the container, refusals
def test_container_refuses_what_the_kernels_do_not_take():
    q = held(np.ones((3, 70)))
    assert q.rows == 3 and q.cols == 70 and tuple(q.scales.shape) == (3, 3) and q.ld_scales == 16 and q.ld_codes == 48
    for codes, scales, cols in ((q.codes, q.scales, 97), (q.codes, q.scales, 64), (q.codes, q.scales, 0), (q.codes[:2], q.scales, 70),
                                (q.codes.int(), q.scales, 70), (q.codes, q.scales.float(), 70), (q.codes[0], q.scales[0], 70),
                                (q.codes, q.scales.contiguous(), 70),                      # rows of three bytes
                                (q.codes.t().contiguous().t(), q.scales, 70)):
        with pytest.raises(ValueError):
            MXFP4(codes, scales, cols)
    wide = torch.zeros((3, 64), dtype=torch.uint8)
    with pytest.raises(ValueError):
        MXFP4(wide[:, 1:49], q.scales, 70)                                                 # rows that do not start aligned
    assert MXFP4(wide[:, 16:64], q.scales, 70).ld_codes == 64


def test_sizes_past_the_kernels_whole_numbers_are_refused():
    """The kernels count rows and columns in 32 bits: what they would count wrongly (4,294,967,328 columns as 32) never reaches them."""
    from tinyserve_llm_b200.ops import Ops
    ops, bare = Ops.__new__(Ops), lambda shape, dtype: torch.empty(shape, dtype=dtype, device="meta")
    for cols in (2 ** 30, 2 ** 31 + 32, 2 ** 32 + 32):
        with pytest.raises(KernelError, match="columns"):
            ops.quantize_mxfp4(bare((1, cols), torch.bfloat16))
        with pytest.raises(ValueError, match="numbers"):
            MXFP4(bare((1, cols // 2), torch.uint8), bare((1, cols // 32), torch.uint8), cols)
    tall = lambda rows: MXFP4(bare((rows, 16), torch.uint8), bare((rows, 16), torch.uint8)[:, :1], 32)  # noqa: E731
    for rows in (2 ** 30, 2 ** 32 + 6):
        with pytest.raises(KernelError, match="rows"):
            ops.linear_mxfp4(bare((rows, 32), torch.bfloat16), tall(6))
        with pytest.raises(KernelError, match="rows"):
            ops.linear_mxfp4(bare((4, 32), torch.bfloat16), tall(rows))
        with pytest.raises(KernelError, match="rows"):
            ops.linear_gated_mxfp4(tall(rows), tall(6), "silu")


def test_oracle_rounds_to_the_nearest_of_two():
    x = np.array([[0.0, -0.0, 0.25, 0.2500001, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 5.0001, 6.0, 7.0, 7.9, -0.75, -3.5] + [0.0] * 16])
    want = [0, 0, 0, 0.5, 1, 1, 2, 2, 4, 4, 6, 6, 6, 6, -1, -4]
    np.testing.assert_array_equal(plain.rounded(x)[0, :16], want)
    np.testing.assert_array_equal(plain.quantize(np.array([[np.inf] * 32, [np.nan] + [0] * 31, [2.0 ** -149] * 32, [0] * 32, [3e38] * 32]))[1][:, 0],
                                  [255, 255, 0, 0, 252])


@pytest.mark.gpu
def test_refusals(ops):
    x, w = torch.zeros((4, 64), dtype=torch.bfloat16, device=DEV), held(np.zeros((6, 64)), DEV)
    for bad in (x.float(), x[:, :56], x[0], x.cpu(), x.t().contiguous().t(), torch.zeros((4, 72), dtype=torch.bfloat16, device=DEV)[:, 4:68]):
        with pytest.raises(KernelError):
            ops.linear_mxfp4(bad, w)
    odd = held(np.zeros((6, 60)), DEV)
    with pytest.raises(KernelError):
        ops.linear_mxfp4(torch.zeros((4, 60), dtype=torch.bfloat16, device=DEV), odd)       # no multiple of eight columns
    with pytest.raises(KernelError):
        ops.linear_mxfp4(x, held(np.zeros((6, 64))))                                         # a weight on the host
    with pytest.raises(KernelError):
        ops.linear_mxfp4(held(np.zeros((4, 60)), DEV), w)
    with pytest.raises(KernelError):
        ops.linear_mxfp4(x, w, out_dtype=torch.float16)
    with pytest.raises(KernelError):
        ops.linear_mxfp4(x, w, out=torch.empty((4, 5), dtype=torch.bfloat16, device=DEV))
    with pytest.raises(KernelError):
        ops.linear_gated_mxfp4(x, w, "tanh")
    with pytest.raises(KernelError):
        ops.linear_gated_mxfp4(x, held(np.zeros((5, 64)), DEV), "silu")
    for bad in (x.half(), x[0], x.cpu(), x.t().contiguous().t(), x[:, :0]):
        with pytest.raises(KernelError):
            ops.quantize_mxfp4(bad)
    with pytest.raises(KernelError):
        ops.dequantize_mxfp4(w, torch.float16)
    with pytest.raises(KernelError):
        ops.dequantize_mxfp4(held(np.zeros((6, 64))))
    assert tuple(ops.linear_mxfp4(x[:0], w).shape) == (0, 6) and ops.quantize_mxfp4(x[:0]).rows == 0
    assert tuple(ops.dequantize_mxfp4(ops.quantize_mxfp4(x[:0])).shape) == (0, 64)


# ------------------------------------------------------------------------------------------------------------ quantisation
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows, cols", [(1, 1), (1, 32), (3, 33), (5, 31), (2, 176), (70, 2000), (1, 8192), (1001, 520), (9, 4099)])
def test_quantize_and_back(ops, rows, cols, dtype):
    x = numbers((rows, cols), dtype, rows + cols, 0.02)
    q = ops.quantize_mxfp4(x.to(DEV))
    codes, scales = plain.quantize(f64(x))
    np.testing.assert_array_equal(q.scales.cpu().numpy(), scales)
    np.testing.assert_array_equal(plain.unpack(q.codes.cpu().numpy(), scales.shape[1]), codes)
    for out in (torch.bfloat16, torch.float32):
        np.testing.assert_array_equal(f64(ops.dequantize_mxfp4(q, out)), plain.values(codes, scales, cols))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_borders(ops, dtype):
    """Midpoints, numbers next to them, every exponent, subnormals, zeros of both signs, what is not finite."""
    points = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.96875, 0.5, 1, 1.5, 2, 3, 4])
    x = torch.zeros((280, 64), dtype=dtype)
    step = 2.0 ** -7 if dtype == torch.bfloat16 else 2.0 ** -23
    for i in range(280):                                           # row i: around 2^(i - 150), down into the subnormals
        near = points * (1 + step * ((i % 3) - 1)) * 2.0 ** (i - 152)
        row = np.concatenate([[4.0 * 2.0 ** (i - 152)], near, -near, [0.0, -0.0]])[:32]
        x[i, :32] = torch.from_numpy(row).to(dtype)
        x[i, 32 + i % 32] = 2.0 ** (i - 152)
    x[270, 3], x[271, 40], x[272, 0] = float("nan"), float("inf"), -float("inf")
    q = ops.quantize_mxfp4(x.to(DEV))
    codes, scales = plain.quantize(f64(x))
    np.testing.assert_array_equal(q.scales.cpu().numpy(), scales)
    np.testing.assert_array_equal(plain.unpack(q.codes.cpu().numpy(), 2), codes)
    want = plain.values(codes, scales, 64)
    np.testing.assert_array_equal(f64(ops.dequantize_mxfp4(q, torch.float32)), want)
    np.testing.assert_array_equal(f64(ops.dequantize_mxfp4(q, torch.bfloat16)), want)


@pytest.mark.gpu
def test_every_code_under_every_scale(ops):
    """16 codes x 256 scales, back to numbers: exact where the type has room, infinite beyond it, NaN under scale 255."""
    codes = torch.arange(16, dtype=torch.uint8).repeat(2)
    packed = (codes[0::2] | (codes[1::2] << 4)).expand(256, 16).contiguous()
    scales = torch.zeros((256, 16), dtype=torch.uint8)
    scales[:, 0] = torch.arange(256)
    q = MXFP4(packed.to(DEV), scales.to(DEV)[:, :1], 32)
    want = plain.values(codes.numpy().reshape(1, 1, 32).repeat(256, 0), scales[:, :1].numpy(), 32)
    for dtype in (torch.float32, torch.bfloat16):
        got = f64(ops.dequantize_mxfp4(q, dtype))
        room = np.where(np.abs(want) >= 2.0 ** 128, np.copysign(np.inf, want), want)
        np.testing.assert_array_equal(got, room)


@pytest.mark.gpu
def test_quantize_takes_stretches_of_wider_rows(ops):
    wide = numbers((37, 300), torch.bfloat16, 3).to(DEV)
    for x in (wide[:, 8:208], wide[:, 3:100], wide[::2, 64:192], wide[:1, 1:]):
        q = ops.quantize_mxfp4(x)
        codes, scales = plain.quantize(f64(x))
        np.testing.assert_array_equal(q.scales.cpu().numpy(), scales)
        np.testing.assert_array_equal(plain.unpack(q.codes.cpu().numpy(), scales.shape[1]), codes)


# ------------------------------------------------------------------------------------------------------------ products
SIZES = [(1, 16, 32), (1, 2048, 2048), (3, 40, 176), (7, 333, 104), (8, 512, 4096), (9, 1000, 520), (17, 130, 8), (32, 96, 8192), (33, 257, 264),
         (64, 2048, 1024), (65, 500, 2000), (128, 129, 640), (130, 1000, 1032), (200, 70, 64), (300, 5000, 512), (700, 4100, 776), (2048, 2048, 2048),
         # a few rows over larger weights, and some hundred in one round of wide tiles: rows of x in two pieces
         (5, 9000, 2048), (9, 3001, 1792), (16, 2600, 2176), (20, 2560, 2304), (40, 2603, 2048), (64, 130, 65536), (200, 2500, 2176), (513, 700, 8192)]


@pytest.mark.gpu
@pytest.mark.parametrize("both", [False, True], ids=["rows16", "rows4"])
@pytest.mark.parametrize("m, n, k", SIZES + [(5, 24, 33), (50, 300, 1001), (190, 300, 2017)])
def test_product(ops, m, n, k, both):
    if not both and k % 8:
        pytest.skip("bfloat16 rows come in multiples of eight columns")
    x, w = numbers((m, k), torch.bfloat16, m + k), f64(numbers((n, k), torch.float32, n + k, 0.02))
    weight, values = held(w, DEV, garbage=255), plain.rounded(w)
    rows, xv = (ops.quantize_mxfp4(x.to(DEV)), plain.rounded(f64(x))) if both else (x.to(DEV), f64(x))
    want, bound = xv @ values.T, sums_bound(xv, values, k)
    check(ops.linear_mxfp4(rows, weight), want, bound)
    check(ops.linear_mxfp4(rows, weight, out_dtype=torch.float32), want, bound)
    out = torch.empty((m, n), dtype=torch.float32, device=DEV)
    assert ops.linear_mxfp4(rows, weight, out_dtype=torch.float32, out=out) is out
    check(out, want, bound)
    torch.cuda.synchronize()
    ops.check_device_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("both", [False, True], ids=["rows16", "rows4"])
@pytest.mark.parametrize("act", ["silu", "relu", "clamped_swish", "gelu_tanh"])
@pytest.mark.parametrize("m, inter, k", [(1, 176, 64), (4, 1001, 256), (8, 8192, 2048), (20, 5, 32), (33, 100, 264), (64, 520, 1024),
                                         (150, 77, 520), (300, 2500, 136), (1100, 2052, 512)])
def test_gated_product(ops, m, inter, k, act, both):
    x, w = numbers((m, k), torch.bfloat16, m + k), f64(numbers((2 * inter, k), torch.float32, inter + k, 2.0 / k ** 0.5))
    weight, values = held(w, DEV), plain.rounded(w)
    rows, xv = (ops.quantize_mxfp4(x.to(DEV)), plain.rounded(f64(x))) if both else (x.to(DEV), f64(x))
    y, off = xv @ values.T, sums_bound(xv, values, k)
    g, u, dg, du = y[:, :inter], y[:, inter:], off[:, :inter], off[:, inter:]
    want = plain.gated(act, g, u, LIMIT, ALPHA)
    factor = np.abs(plain.gated(act, g, np.ones_like(g), LIMIT, ALPHA))            # |act(g)|, twice it for the activation with u + 1
    bound = 1.13 * dg * (np.abs(u) + 1) + factor * du + 1.13 * dg * du + 2.0 ** -16 * np.abs(want)
    check(ops.linear_gated_mxfp4(rows, weight, act, LIMIT, ALPHA), want, bound)
    torch.cuda.synchronize()
    ops.check_device_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("both", [False, True], ids=["rows16", "rows4"])
@pytest.mark.parametrize("m, n, k", [(2, 20, 320), (40, 20, 320), (150, 20, 320), (2, 5000, 1152), (40, 5000, 1152), (150, 5000, 1152)])
def test_scales_from_end_to_end(ops, m, n, k, both):
    """Blocks under the smallest scale, scales past what one factor holds, and the largest: exact products of one column that is not zero."""
    scales, blocks = [0, 1, 126, 127, 128, 129, 130, 180, 251, 252], k // 32
    w, codes, bytes_ = np.zeros((n, k)), np.zeros((n, blocks, 32), dtype=np.uint8), np.full((n, blocks), 120, dtype=np.uint8)
    bytes_[:, :10] = scales
    for i in range(n):
        block, high = (i % 20) // 2, i % 2
        w[i, 32 * block + 5] = (6.0 if high else -0.5) * 2.0 ** (scales[block] - 127)
        codes[i, block, 5] = 7 if high else 9
    flat = codes.reshape(n, -1)
    wide = torch.zeros((n, -(-blocks // 16) * 16), dtype=torch.uint8, device=DEV)
    wide[:, :blocks] = torch.from_numpy(bytes_).to(DEV)
    weight = MXFP4(torch.from_numpy(flat[:, 0::2] | (flat[:, 1::2] << 4)).to(DEV), wide[:, :blocks], k)
    x = torch.zeros((m, k), dtype=torch.bfloat16)
    x[:, 5::32] = torch.tensor([2.0 ** (-(i % 2) - 3) for i in range(m)]).to(torch.bfloat16)[:, None]
    rows, xv = (ops.quantize_mxfp4(x.to(DEV)), plain.rounded(f64(x))) if both else (x.to(DEV), f64(x))
    want = xv @ w.T
    got = f64(ops.linear_mxfp4(rows, weight, out_dtype=torch.float32))
    normal = np.abs(want) >= 2.0 ** -126                           # below, a sum may be flushed or not
    np.testing.assert_array_equal(got[normal], want[normal])
    assert (np.abs(got[~normal]) <= 2.0 ** -126).all()


@pytest.mark.gpu
@pytest.mark.parametrize("both", [False, True], ids=["rows16", "rows4"])
@pytest.mark.parametrize("m", [3, 40, 500])
def test_what_is_not_finite_stays_in_its_row_and_column(ops, m, both):
    n, k = 300, 512
    x, w = numbers((m, k), torch.bfloat16, 1), f64(numbers((n, k), torch.float32, 2, 0.02))
    x[1, 70] = float("nan")
    w[7, 100] = float("nan")                                       # its block becomes NaN
    weight = held(w, DEV)
    got = f64(ops.linear_mxfp4(ops.quantize_mxfp4(x.to(DEV)) if both else x.to(DEV), weight))
    bad = np.zeros((m, n), dtype=bool)
    bad[1], bad[:, 7] = True, True
    np.testing.assert_array_equal(np.isnan(got), bad)


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True], ids=["linear", "gated"])
@pytest.mark.parametrize("m, n, k", [(3, 300, 512), (3, 5000, 2048), (20, 5000, 1152), (20, 130, 65536), (40, 300, 512), (200, 2500, 2176),
                                     (500, 300, 512)])
def test_infinite_numbers_in_bfloat16_rows(ops, m, n, k, gated):
    """Infinities times numbers that are not zero are infinite, times zero or against each other NaN, beside a NaN NaN; other rows are as ever."""
    n -= n % 2
    x, w = numbers((m, k), torch.bfloat16, 1), f64(numbers((n, k), torch.float32, 2, 0.02))
    x[0, 70], x[1, 5], x[1, 40], x[2, 3], x[2, 4] = float("inf"), float("inf"), float("-inf"), float("-inf"), float("nan")
    values, xv = plain.rounded(w), f64(x)
    with np.errstate(invalid="ignore"):
        want, bound = xv @ values.T, sums_bound(np.where(np.isfinite(xv), xv, 0.0), values, k)
    if gated:
        half = n // 2
        with np.errstate(invalid="ignore", over="ignore"):
            g, u = want[:, :half], want[:, half:]
            want = plain.gated("relu", g, u, 0.0, 1.0)
            bound = bound[:, :half] * (np.abs(u) + 1) + np.abs(g) * bound[:, half:] + bound[:, :half] * bound[:, half:]
        got = f64(ops.linear_gated_mxfp4(x.to(DEV), held(w, DEV), "relu"))
        finite = np.isfinite(want) & np.isfinite(bound)
        rows = slice(3, None)                                      # where gate or up is infinite, relu's NaN is the hardware's maximum
    else:
        got, finite, rows = f64(ops.linear_mxfp4(x.to(DEV), held(w, DEV))), np.isfinite(want), slice(None)
        np.testing.assert_array_equal(np.isnan(got), np.isnan(want))
        np.testing.assert_array_equal(np.where(np.isinf(got), got, 0.0), np.where(np.isinf(want), want, 0.0))
    slack = (bound + 2.0 ** -8 * (np.abs(want) + bound))[rows][finite[rows]]
    with np.errstate(invalid="ignore"):
        assert (np.abs(got - want)[rows][finite[rows]] <= slack).all()


@pytest.mark.gpu
def test_offsets_past_32_bits(ops):
    """Two thousand million outputs and more: the last rows are what a product of theirs alone gives, and so are the last rows' codes."""
    m, n, k = 20032, 110080, 64
    w, x = held(f64(numbers((n, k), torch.float32, 21, 0.05)), DEV), numbers((m, k), torch.bfloat16, 22).to(DEV)
    values = f64(ops.dequantize_mxfp4(w, torch.float32))
    for rows, xv in ((x, f64(x[-40:])), (ops.quantize_mxfp4(x), plain.rounded(f64(x[-40:])))):
        y = ops.linear_mxfp4(rows, w)
        assert y.numel() > 2 ** 31
        check(y[-40:], xv @ values.T, sums_bound(xv, values, k))
    q = ops.quantize_mxfp4(y.t().contiguous())
    tail = ops.quantize_mxfp4(y[:, -3:].t().contiguous())
    assert torch.equal(q.codes[-3:], tail.codes) and torch.equal(q.scales[-3:], tail.scales)
    assert torch.equal(ops.dequantize_mxfp4(q)[-3:], ops.dequantize_mxfp4(tail))
    ops.check_device_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("both", [False, True], ids=["rows16", "rows4"])
@pytest.mark.parametrize("m, n, k", [(4, 256, 512), (40, 5120, 1152), (200, 512, 256), (400, 2048, 4096)])
def test_out_that_starts_between_words(ops, m, n, k, both):
    w, x = held(f64(numbers((n, k), torch.float32, 23, 0.02)), DEV), numbers((m, k), torch.bfloat16, 24).to(DEV)
    x = ops.quantize_mxfp4(x) if both else x
    room = torch.full((m * n + 2,), 7.0, dtype=torch.bfloat16, device=DEV)
    out = room[1:-1].view(m, n)
    assert out.data_ptr() % 4 == 2
    assert torch.equal(ops.linear_mxfp4(x, w, out=out), ops.linear_mxfp4(x, w))
    assert float(room[0]) == 7 and float(room[-1]) == 7


@pytest.mark.gpu
@pytest.mark.parametrize("m", [5, 40, 200])
def test_strided_rows(ops, m):
    wide, w = numbers((m, 704), torch.bfloat16, 4).to(DEV), f64(numbers((90, 512), torch.float32, 5, 0.02))
    x, values = wide[:, 64:576], plain.rounded(w)
    held_wide = held(np.concatenate([w, w], axis=0), DEV)
    every_other = MXFP4(held_wide.codes[::2], held_wide.scales[::2], 512)
    check(ops.linear_mxfp4(x, held(w, DEV)), f64(x) @ values.T, sums_bound(f64(x), values, 512))
    order = [2 * i % 90 for i in range(90)]
    check(ops.linear_mxfp4(x, every_other), f64(x) @ values[order].T, sums_bound(f64(x), values[order], 512))


@pytest.mark.gpu
def test_run_of_them_in_a_graph(ops):
    """A feed-forward as the engine runs it, both ways of holding the rows, captured once and replayed on new inputs; rows behind stay."""
    k, inter, m = 512, 704, 48
    wu, wd = f64(numbers((2 * inter, k), torch.float32, 6, 0.05)), f64(numbers((k, inter), torch.float32, 7, 0.05))
    up, down = held(wu, DEV), held(wd, DEV)
    x = numbers((m, k), torch.bfloat16, 8).to(DEV)
    room = torch.full((m + 4, k), 7.0, dtype=torch.bfloat16, device=DEV)

    def layer(x, out):
        a = ops.linear_gated_mxfp4(x, up, "silu")
        b = ops.linear_gated_mxfp4(ops.quantize_mxfp4(x), up, "silu")
        return ops.linear_mxfp4(a, down, out=out), ops.linear_mxfp4(ops.quantize_mxfp4(b), down)

    layer(x, room[:m])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y16, y4 = layer(x, room[:m])
    for seed in (9, 10):
        x.copy_(numbers((m, k), torch.bfloat16, seed).to(DEV))
        graph.replay()
        torch.cuda.synchronize()
        eager16, eager4 = layer(x, torch.empty_like(y16))
        assert torch.equal(y16, eager16) and torch.equal(y4, eager4)
        assert bool((room[m:] == 7).all())
    ops.check_device_errors()


@pytest.mark.gpu
def test_two_streams_at_once(ops):
    """Nothing is shared between two calls under way: many products on two streams give what they give alone."""
    w = held(f64(numbers((2048, 1024), torch.float32, 11, 0.02)), DEV)
    xs = [numbers((m, 1024), torch.bfloat16, m).to(DEV) for m in (4, 64)]
    alone = [(ops.linear_mxfp4(x, w), ops.linear_mxfp4(ops.quantize_mxfp4(x), w)) for x in xs]
    torch.cuda.synchronize()
    streams, found = [torch.cuda.Stream() for _ in xs], [[], []]
    for _ in range(20):
        for i, (stream, x) in enumerate(zip(streams, xs)):
            with torch.cuda.stream(stream):
                found[i].append((ops.linear_mxfp4(x, w), ops.linear_mxfp4(ops.quantize_mxfp4(x), w)))
    torch.cuda.synchronize()
    for (a, b), results in zip(alone, found):
        assert all(torch.equal(a, c) and torch.equal(b, d) for c, d in results)
    ops.check_device_errors()
