"""
Bias-free projection y = x . W^T with W stored [out_features, in_features] (the checkpoint layout).

bfloat16: the library matrix product (cuBLAS through torch.mm), as the reference does through
nn.Linear (model/llama.py:200-201, :220-221).  float32: the engine's own kernels (every operand as two TF32 numbers on the tensor
cores, or FFMA), so that no reduced-precision matrix mode can slip in and the reduction order of a
row does not depend on what else is in the batch.

`QuantizedLinear` holds its weight in microscaled 4-bit floating point, made from the checkpoint's when the part is built, and
multiplies on the engine's own kernels; `projection` gives a part one or the other as the runtime says.
"""

from __future__ import annotations

import torch

from tinyserve_llm_b200.parts.base import Runtime


def fuse_rows(tensors: list[torch.Tensor]) -> torch.Tensor:
    """Stack projections that share an input into one weight, rows in the order given."""
    return torch.cat(tensors, dim=0).contiguous()


class Linear:
    def __init__(self, weight: torch.Tensor, rt: Runtime) -> None:
        assert weight.dim() == 2
        self.rt = rt
        self.weight = weight.to(device=rt.device, dtype=rt.dtype).contiguous()
        self.out_features, self.in_features = self.weight.shape

    def __call__(self, x: torch.Tensor, out_dtype: torch.dtype | None = None,
                 out: torch.Tensor | None = None) -> torch.Tensor:
        return self.rt.ops.linear(x, self.weight, out_dtype=out_dtype, out=out)

    def columns(self, x: torch.Tensor, out_dtype: torch.dtype | None = None) -> torch.Tensor:
        """The product of a stretch of columns of wider rows."""
        return self.rt.ops.linear_columns(x, self.weight, out_dtype=out_dtype)

    def gated(self, x: torch.Tensor, activation: str, limit: float = 0.0, alpha: float = 1.0) -> torch.Tensor:
        """act(x . Wgate^T, x . Wup^T) of the two halves of the weight's rows, in the products' epilogue where a kernel has one."""
        return self.rt.ops.linear_gated(x, self.weight, activation, limit, alpha)

    def unary(self, x: torch.Tensor, activation: str, a: float = 0.0, b: float = 0.0) -> torch.Tensor:
        """act(x . W^T) for an activation of one argument."""
        return self.rt.ops.linear_unary(x, self.weight, activation, a, b)


class QuantizedLinear(Linear):
    """
    `weight` is an `MXFP4`, a quarter of bfloat16's bytes and a little more.  With the runtime's `activation_format` the rows of x are
    rounded to four bits too, ahead of every product.
    """

    def __init__(self, weight: torch.Tensor, rt: Runtime) -> None:
        assert weight.dim() == 2
        self.rt = rt
        self.out_features, self.in_features = weight.shape
        if self.in_features % 8:
            raise NotImplementedError(f"a projection of {self.in_features} inputs cannot be held in four bits: the products take multiples of 8")
        self.weight = rt.ops.quantize_mxfp4(weight.to(rt.device))
        torch.cuda.current_stream(rt.device).synchronize()       # from here on nothing writes it: products may read it ahead of their turn
        self.weight.settled = True
        rt.shared["quantized_bytes"] = rt.shared.get("quantized_bytes", 0) + self.weight.nbytes

    def _rows(self, x: torch.Tensor):
        return self.rt.ops.quantize_mxfp4(x) if self.rt.activation_format == "mxfp4" else x

    def __call__(self, x: torch.Tensor, out_dtype: torch.dtype | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
        return self.rt.ops.linear_mxfp4(self._rows(x), self.weight, out_dtype=out_dtype, out=out)

    def columns(self, x: torch.Tensor, out_dtype: torch.dtype | None = None) -> torch.Tensor:
        return self(x, out_dtype)

    def gated(self, x: torch.Tensor, activation: str, limit: float = 0.0, alpha: float = 1.0) -> torch.Tensor:
        return self.rt.ops.linear_gated_mxfp4(self._rows(x), self.weight, activation, limit, alpha)

    def unary(self, x: torch.Tensor, activation: str, a: float = 0.0, b: float = 0.0) -> torch.Tensor:
        return self.rt.ops.unary_activation(self(x), activation, a, b)


def projection(weight: torch.Tensor, rt: Runtime) -> Linear:
    """A projection of attention or of a feed-forward, its weight held as the runtime's `weight_format` says."""
    return QuantizedLinear(weight, rt) if rt.weight_format == "mxfp4" else Linear(weight, rt)
