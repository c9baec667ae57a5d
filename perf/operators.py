"""
Matrices held in microscaled 4-bit floating point, and the products that read them, as cases that can be timed.

A row of K numbers is cut into blocks of 32.  A block has one scale, a power of two 2^(s - 127) held in the byte s, and 32 codes of four
bits: a sign, two bits of exponent, one of mantissa, which stand for 0, 0.5, 1, 1.5, 2, 3, 4 and 6.  With a the largest magnitude of the
block, s - 127 = floor(log2 a) - 2, at least -127 (0 for a block of zeros); a number x becomes the code nearest to x / 2^(s - 127), ties to
the code whose last bit is 0, magnitudes over 6 to 6.  A block that holds an infinity or a NaN has s = 255 and stands for NaN.

Kinds of cases: `quantize` (numbers to codes and scales and back), `linear` (y = x . W^T, W in four bits), `gated` (act(x . Wgate^T) times
x . Wup^T, the two halves of one W), each product with rows of x in bfloat16, or first rounded to four bits themselves (`both`).
Weights of the sizes of Llama 3.2 1B and Llama 3.1 8B layers, N(0, 0.02); x as a norm's output, some channels larger than others.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
BLOCK = 32
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
SWISH_LIMIT, SWISH_ALPHA = 7.0, 1.702


# ------------------------------------------------------------------------------------------------------------ the cases
def _quantize(name, rows, cols, dtype):
    return {"kind": "quantize", "rows": rows, "cols": cols, "dtype": dtype} | ({"name": name} if name else {})


def _linear(name, rows, cols, out, both=False, out_dtype="bf16"):
    return {"kind": "linear", "rows": rows, "cols": cols, "out": out, "both": both, "out_dtype": out_dtype} | ({"name": name} if name else {})


def _gated(name, rows, cols, inter, both=False, act="silu"):
    return {"kind": "gated", "rows": rows, "cols": cols, "inter": inter, "both": both, "act": act} | ({"name": name} if name else {})


def listed() -> list[dict]:
    return [
        # an 8B model's gate and up projections, as a model is loaded
        _quantize("quantize_28672x4096", 28672, 4096, "bf16"),
        # rows of a prompt portion of odd length, 32-bit numbers, columns that end inside a block
        _quantize("quantize_f32_1001x2000", 1001, 2000, "f32"),
        # one request decoding: the smallest product of a layer
        _linear("linear_1", 1, 2048, 2048),
        # eight requests decoding: a 1B model's down projection
        _linear("linear_8", 8, 8192, 2048),
        # decode steps of some dozens of requests beside short portions, an 8B model's output projection
        _linear("linear_77", 77, 4096, 4096),
        # a prompt through a 1B model's down projection
        _linear("linear_2048", 2048, 8192, 2048),
        # a decode step of eight requests through an 8B model's gate and up projections
        _gated("gated_8", 8, 4096, 14336),
        # a prompt through a 1B model's gate and up projections
        _gated("gated_2048", 2048, 2048, 8192),
        # both sides in four bits: a decode step of four requests, a portion of odd length with odd sizes, whole prompts
        _linear("both_4", 4, 2048, 2048, both=True),
        _linear("both_333", 333, 4112, 1000, both=True, out_dtype="f32"),
        _linear("both_2048", 2048, 8192, 2048, both=True),
        _gated("both_gated_2048", 2048, 4096, 14336, both=True),
    ]


def draw(rng) -> dict:
    """One more case: kinds evenly, sizes over the logarithm of their range, odd ones among them."""
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(("quantize", "linear", "linear", "gated", "both", "both_gated"))
    if kind == "quantize":
        return _quantize(None, log(1, 8192), log(16, 8192), rng.choice(("bf16", "f32")))
    rows = log(1, 2048)
    cols = 16 * log(4, 512) if rng.random() < 0.5 else rng.choice((2048, 4096, 8192))
    if kind in ("linear", "both"):
        out = log(16, 8192) if rng.random() < 0.5 else rng.choice((512, 2048, 4096, 8192))
        return _linear(None, rows, cols, out, kind == "both", rng.choice(("bf16", "f32")))
    inter = log(16, 8192) if rng.random() < 0.5 else rng.choice((2048, 8192))
    return _gated(None, rows, cols, inter, kind == "both_gated", rng.choice(("silu", "relu", "clamped_swish", "gelu_tanh")))


def work(case: dict) -> dict:
    rows, cols = case["rows"], case["cols"]
    if case["kind"] == "quantize":              # the numbers once, codes and scales written and read again, the values they stand for
        size, blocks = DTYPES[case["dtype"]].itemsize, rows * -(-cols // BLOCK)
        return {"bytes": 2 * rows * cols * size + 2 * blocks * 17, "flops": 2 * rows * cols}
    outs = case["out"] if case["kind"] == "linear" else 2 * case["inter"]
    stored = rows * case["out"] * DTYPES[case["out_dtype"]].itemsize if case["kind"] == "linear" else rows * case["inter"] * 2
    return {"bytes": rows * cols * 2 + outs * -(-cols // BLOCK) * 17 + stored, "flops": 2 * rows * cols * outs}


# ------------------------------------------------------------------------------------------------------------ the plain form
def _plain_quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes uint8 [rows, blocks * 16], two a byte, the lower four bits the earlier one; scales uint8 [rows, blocks], rows 16-byte apart)."""
    rows, cols = x.shape
    blocks = -(-cols // BLOCK)
    v = torch.zeros((rows, blocks * BLOCK), dtype=torch.float32, device=x.device)
    v[:, :cols] = x
    v = v.view(rows, blocks, BLOCK)
    top = v.abs().amax(dim=2)
    finite = torch.isfinite(v).all(dim=2)
    exponent = torch.frexp(torch.where(finite, top, 1.0)).exponent - 1          # floor(log2)
    s = torch.where(top > 0, (exponent - 2 + 127).clamp(min=0), 0)
    s = torch.where(finite, s, 255)
    scaled = torch.ldexp(v, (127 - s.clamp(max=254))[:, :, None]).abs()
    code = torch.zeros_like(v, dtype=torch.uint8)
    for k, (low, high) in enumerate(zip(VALUES[:-1], VALUES[1:])):              # past the midpoint, or on it where the upper code is even
        middle = (low + high) / 2
        code += (scaled >= middle) if (k + 1) % 2 == 0 else (scaled > middle)
    code = torch.where(finite[:, :, None], code | (torch.signbit(v).to(torch.uint8) << 3), 0).view(rows, blocks * 16, 2)
    scales = torch.full((rows, -(-blocks // 16) * 16), 127, dtype=torch.uint8, device=x.device)
    scales[:, :blocks] = s.to(torch.uint8)
    return code[:, :, 0] | (code[:, :, 1] << 4), scales[:, :blocks]


def _plain_values(codes: torch.Tensor, scales: torch.Tensor, cols: int) -> torch.Tensor:
    rows, blocks = scales.shape
    nibbles = torch.stack((codes & 15, codes >> 4), dim=2).view(rows, blocks, BLOCK)
    table = torch.tensor(VALUES + tuple(-v for v in VALUES), dtype=torch.float32, device=codes.device)
    s = scales.to(torch.int32)
    factor = torch.where(s == 255, float("nan"), torch.ldexp(torch.ones_like(s, dtype=torch.float32), s - 127))
    return (table[nibbles.to(torch.int32)] * factor[:, :, None]).view(rows, blocks * BLOCK)[:, :cols]


def _activate(g: torch.Tensor, u: torch.Tensor, act: str) -> torch.Tensor:
    if act == "relu":
        return torch.clamp(g, min=0) * u
    if act == "clamped_swish":
        g, u = torch.clamp(g, max=SWISH_LIMIT), torch.clamp(u, -SWISH_LIMIT, SWISH_LIMIT)
        return g / (1 + torch.exp(-SWISH_ALPHA * g)) * (u + 1)
    if act == "gelu_tanh":
        return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g * g * g))) * u
    return g / (1 + torch.exp(-g)) * u


def _plain(state: dict) -> torch.Tensor:
    case, x = state["case"], state["x"]
    if case["kind"] == "quantize":
        codes, scales = _plain_quantize(x)
        return _plain_values(codes, scales, case["cols"]).to(x.dtype)
    if case["both"]:
        codes, scales = _plain_quantize(x)
        x = _plain_values(codes, scales, case["cols"])
    y = x.float() @ _plain_values(state["codes"], state["scales"], case["cols"]).t()
    if case["kind"] == "linear":
        return y.to(DTYPES[case["out_dtype"]])
    inter = case["inter"]
    return _activate(y[:, :inter], y[:, inter:], case["act"]).to(x.dtype if not case["both"] else torch.bfloat16)


# ------------------------------------------------------------------------------------------------------------ inputs, calls
def _draw_tensors(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    rows, cols = case["rows"], case["cols"]
    x = torch.randn((rows, cols), generator=gen, device=DEV)
    channel = torch.exp(0.8 * torch.randn((cols,), generator=gen, device=DEV))
    if case["kind"] == "quantize":
        return {"case": case, "x": (0.02 * x * channel).to(DTYPES[case["dtype"]])}
    outs = case["out"] if case["kind"] == "linear" else 2 * case["inter"]
    weight = 0.02 * torch.randn((outs, cols), generator=gen, device=DEV)
    return {"case": case, "x": (x * channel).to(torch.bfloat16), "weight": weight}


def prepare(case: dict, seed: int) -> dict:
    state = _draw_tensors(case, seed)
    if "weight" in state:                                   # a program holds its weights in four bits
        state["codes"], state["scales"] = _plain_quantize(state.pop("weight"))
    return state


def run(state: dict):
    if not own:
        return _plain(state)
    from tinyserve_llm_b200.ops import MXFP4, get_ops
    ops, case, x = get_ops(), state["case"], state["x"]
    if case["kind"] == "quantize":
        return ops.dequantize_mxfp4(ops.quantize_mxfp4(x), x.dtype)
    weight = MXFP4(state["codes"], state["scales"], case["cols"])
    rows = ops.quantize_mxfp4(x) if case["both"] else x
    if case["kind"] == "linear":
        return ops.linear_mxfp4(rows, weight, out_dtype=DTYPES[case["out_dtype"]])
    return ops.linear_gated_mxfp4(rows, weight, case["act"], SWISH_LIMIT, SWISH_ALPHA)


# ------------------------------------------------------------------------------------------------------------ 64 bits
def _nearest(x: torch.Tensor) -> torch.Tensor:
    """The values a float64 matrix has in four bits, by distances: of the nearest values the one whose code is even (finite x only)."""
    rows, cols = x.shape
    out = torch.zeros_like(x)
    table = torch.tensor(VALUES, dtype=torch.float64, device=x.device)
    for c in range(0, cols, BLOCK):
        part = x[:, c:c + BLOCK]
        top = part.abs().max(dim=1, keepdim=True).values
        power = torch.floor(torch.log2(torch.where(top > 0, top, 1.0)))
        power = power - (torch.exp2(power) > top).double() + (torch.exp2(power + 1) <= top).double()   # a logarithm that was rounded
        scale = torch.exp2(torch.where(top > 0, torch.clamp(power - 2, min=-127.0), torch.full_like(power, -127.0)))
        target = part.abs() / scale
        best, gap = torch.zeros_like(part), target.clone()
        for k in range(1, 8):
            distance = (target - table[k]).abs()
            better = (distance <= gap) if k % 2 == 0 else (distance < gap)
            best, gap = torch.where(better, table[k], best), torch.where(better, distance, gap)
        out[:, c:c + BLOCK] = torch.copysign(best * scale, part)
    return out


def exact(case: dict, seed: int):
    state = _draw_tensors(case, seed)
    x = state["x"].double()
    if case["kind"] == "quantize":
        return _nearest(x)
    x = _nearest(x) if case["both"] else x
    y = torch.matmul(x, _nearest(state["weight"].double()).t())
    if case["kind"] == "linear":
        return y
    g, u = y.chunk(2, dim=1)
    act = case["act"]
    if act == "clamped_swish":
        g, u = g.clamp(max=SWISH_LIMIT), u.clamp(-SWISH_LIMIT, SWISH_LIMIT)
        return g * torch.sigmoid(SWISH_ALPHA * g) * (u + 1)
    if act == "relu":
        return torch.where(g > 0, g, 0.0) * u
    if act == "gelu_tanh":
        return g * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3)) * u
    return g * torch.sigmoid(g) * u
