"""
A matrix held in microscaled 4-bit floating point (the OCP microscaling format MXFP4: E2M1 codes, one E8M0 scale for 32 of them).

A row of `cols` numbers is cut into blocks of 32.  A block has one scale, the power of two 2^(s - 127) held in the byte s (255: the
block is NaN), and 32 codes of four bits, which stand for 0, 0.5, 1, 1.5, 2, 3, 4 and 6 and, eight further on, their negatives.
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

BLOCK = 32


def blocks_of(cols: int) -> int:
    return -(-cols // BLOCK)


@dataclass(frozen=True)
class MXFP4:
    """
    `codes`: uint8 [rows, blocks * 16], two codes a byte, the lower four bits the earlier one, codes behind the last column 0;
    `scales`: uint8 [rows, blocks].  The rows of either start 16-byte aligned (a row of scales is usually a stretch of a wider one).
    `settled`: the codes and scales were written long ago and stay as they are (a loaded model's weights): products may read them before
    the kernels ahead of them on the stream have finished.
    """

    codes: torch.Tensor
    scales: torch.Tensor
    cols: int
    settled: bool = False

    def __post_init__(self) -> None:
        codes, scales = self.codes, self.scales
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8 or codes.dim() != 2 or scales.dim() != 2:
            raise ValueError("MXFP4: codes and scales must be uint8 matrices")
        blocks = blocks_of(self.cols)
        if self.cols <= 0 or codes.shape[1] != blocks * 16 or scales.shape[1] != blocks or codes.shape[0] != scales.shape[0]:
            raise ValueError(f"MXFP4: codes {tuple(codes.shape)} and scales {tuple(scales.shape)} do not hold rows of {self.cols} numbers: "
                             f"{blocks} blocks of 16 bytes and one scale each")
        if codes.device != scales.device:
            raise ValueError(f"MXFP4: codes on {codes.device}, scales on {scales.device}")
        for t, name in ((codes, "codes"), (scales, "scales")):
            if t.shape[1] > 1 and t.stride(1) != 1 or t.shape[0] > 1 and (t.stride(0) % 16 or t.stride(0) < t.shape[1]) or t.data_ptr() % 16:
                raise ValueError(f"MXFP4: rows of {name} must be contiguous and start 16-byte aligned (strides {t.stride()})")

    @property
    def rows(self) -> int:
        return self.codes.shape[0]

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def nbytes(self) -> int:
        """Bytes of codes and scales, rows' alignment included."""
        return self.rows * (self.ld_codes + self.ld_scales)

    @property
    def ld_codes(self) -> int:
        """Bytes from a row of codes to the next (of a single row: what the next one's would be)."""
        return self.codes.stride(0) if self.rows > 1 else self.codes.shape[1]

    @property
    def ld_scales(self) -> int:
        return self.scales.stride(0) if self.rows > 1 else -(-self.scales.shape[1] // 16) * 16

    @staticmethod
    def empty(rows: int, cols: int, device: torch.device) -> "MXFP4":
        """Room for a matrix; what a row of scales has behind its last block is never used."""
        blocks = blocks_of(cols)
        codes = torch.empty((rows, blocks * 16), dtype=torch.uint8, device=device)
        scales = torch.empty((rows, -(-blocks // 16) * 16), dtype=torch.uint8, device=device)
        return MXFP4(codes, scales[:, :blocks], cols)
