"""
A matrix held in microscaled 4-bit floating point (the OCP microscaling format MXFP4: E2M1 codes, one E8M0 scale for 32 of them).

A row of `cols` numbers is cut into blocks of 32.  A block has one scale, the power of two 2^(s - 127) held in the byte s (255: the
block is NaN), and 32 codes of four bits, which stand for 0, 0.5, 1, 1.5, 2, 3, 4 and 6 and, eight further on, their negatives.
"""

from __future__ import annotations

import torch

BLOCK = 32
MOST = 2 ** 30 - 1                 # columns of a matrix, rows of a product: the kernels count them in 32 bits


class MXFP4:
    """
    `codes`: uint8 [rows, blocks * 16], two codes a byte, the lower four bits the earlier one, codes behind the last column 0;
    `scales`: uint8 [rows, blocks].  The rows of either start 16-byte aligned (a row of scales is usually a stretch of a wider one).
    `settled`: the codes and scales were written long ago and stay as they are (a loaded model's weights): products may read them before
    the kernels ahead of them on the stream have finished.
    `ld_codes`, `ld_scales`: bytes from a row to the next (of a single row: what the next one's would be).
    """

    __slots__ = ("codes", "scales", "rows", "cols", "settled", "ld_codes", "ld_scales")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, cols: int, settled: bool = False) -> None:
        if codes.dtype is not torch.uint8 or scales.dtype is not torch.uint8 or codes.dim() != 2 or scales.dim() != 2:
            raise ValueError("MXFP4: codes and scales must be uint8 matrices")
        (rows, code_bytes), (scale_rows, blocks) = codes.shape, scales.shape
        if cols <= 0 or blocks != -(-cols // BLOCK) or code_bytes != blocks * 16 or rows != scale_rows:
            raise ValueError(f"MXFP4: codes {tuple(codes.shape)} and scales {tuple(scales.shape)} do not hold rows of {cols} numbers: "
                             f"{-(-cols // BLOCK)} blocks of 16 bytes and one scale each")
        if cols > MOST:
            raise ValueError(f"MXFP4: rows of {cols} numbers; the kernels take up to {MOST}")
        if codes.device != scales.device:
            raise ValueError(f"MXFP4: codes on {codes.device}, scales on {scales.device}")
        (ld_codes, one), (ld_scales, one_too) = codes.stride(), scales.stride()
        if rows <= 1:
            ld_codes, ld_scales = code_bytes, -(-blocks // 16) * 16
        if (one != 1 or (one_too != 1 and blocks > 1) or ld_codes % 16 or ld_scales % 16 or ld_codes < code_bytes or ld_scales < blocks
                or codes.data_ptr() % 16 or scales.data_ptr() % 16):
            raise ValueError(f"MXFP4: rows of codes and of scales must be contiguous and start 16-byte aligned (strides {codes.stride()} "
                             f"and {scales.stride()})")
        self._hold(codes, scales, rows, cols, settled, ld_codes, ld_scales)

    def _hold(self, codes, scales, rows: int, cols: int, settled: bool, ld_codes: int, ld_scales: int) -> None:
        self.codes, self.scales, self.rows, self.cols, self.settled = codes, scales, rows, cols, settled
        self.ld_codes, self.ld_scales = ld_codes, ld_scales

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def nbytes(self) -> int:
        """Bytes of codes and scales, rows' alignment included."""
        return self.rows * (self.ld_codes + self.ld_scales)

    def __repr__(self) -> str:
        return f"MXFP4({self.rows} x {self.cols} on {self.device}{', settled' if self.settled else ''})"

    @classmethod
    def empty(cls, rows: int, cols: int, device: torch.device) -> "MXFP4":
        """Room for a matrix; what a row of scales has behind its last block is never used."""
        blocks = -(-cols // BLOCK)
        ld = -(-blocks // 16) * 16
        q = cls.__new__(cls)
        q._hold(torch.empty_strided((rows, blocks * 16), (blocks * 16, 1), dtype=torch.uint8, device=device),
                torch.empty_strided((rows, blocks), (ld, 1), dtype=torch.uint8, device=device), rows, cols, False, blocks * 16, ld)
        return q
