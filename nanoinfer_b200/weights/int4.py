"""Matrices of 4-bit weights with a scale for each group of a row: ``w[n, k] = (code[n, k] - 8) * scale[n, k // group]``.

The codes are laid out once, for the product of few tokens (csrc/gemm_int4.cu): tiles of 16 rows and 64 columns, 512 bytes
each, in the order in which the lanes of a warp feed them to the tensor core.
"""
from __future__ import annotations

import torch

GROUPS = (32, 64, 128)


class Int4Matrix:
    """``shape`` (rows, columns), ``group``, and on the device ``packed`` (uint8, half a byte a weight; rows and columns are padded to
    whole tiles) and ``scales`` (bfloat16, for every row of the tiles); neither is replaced afterwards. ``bf16_exact``: every weight is a
    bfloat16 number (no scale has more than 5 significant bits; a code has 3)."""

    def __init__(self, packed: torch.Tensor, scales: torch.Tensor, shape, group: int, bf16_exact: bool):
        if group not in GROUPS:
            raise ValueError(f"groups of {GROUPS} weights are possible, not of {group}")
        n, k = (int(x) for x in shape)
        if n <= 0 or k <= 0 or k % group:
            raise ValueError(f"{n} rows of {k} weights: columns are a multiple of {group}")
        # (the kernels read by ``shape``: what they read has to be there)
        row_tiles, k_tiles = -(-n // 16), -(-k // 64)
        for what, t, dtype, count in (("codes", packed, torch.uint8, row_tiles * k_tiles * 512), ("scales", scales, torch.bfloat16, row_tiles * 16 * (k // group))):
            if t.dtype != dtype or t.numel() != count or not t.is_contiguous() or t.device != packed.device:
                raise ValueError(f"the {what} of {n} x {k} weights in groups of {group} are {count} dense {dtype} on the codes' device; got {t.dtype} "
                                 f"{tuple(t.shape)} on {t.device}")
        self.packed, self.scales, self.shape, self.group, self.bf16_exact = packed, scales, (n, k), int(group), bool(bf16_exact)

    @property
    def device(self) -> torch.device:
        return self.packed.device

    def nbytes(self) -> int:
        return self.packed.numel() + 2 * self.scales.numel()

    @staticmethod
    def from_codes(codes: torch.Tensor, scales: torch.Tensor, group: int) -> "Int4Matrix":
        """``codes`` uint8 [rows, columns] of 0..15, ``scales`` bfloat16 [rows, columns / group], on one device."""
        if group not in GROUPS:
            raise ValueError(f"groups of {GROUPS} weights are possible, not of {group}")
        if codes.dim() != 2 or codes.dtype != torch.uint8 or codes.numel() == 0 or codes.shape[1] % group:
            raise ValueError(f"codes are uint8 [rows, columns], columns a multiple of {group}; got {codes.dtype} {tuple(codes.shape)}")
        n, k = codes.shape
        if scales.dtype != torch.bfloat16 or tuple(scales.shape) != (n, k // group) or scales.device != codes.device:
            raise ValueError(f"scales are bfloat16 {(n, k // group)} on {codes.device}; got {scales.dtype} {tuple(scales.shape)} on {scales.device}")
        if int(codes.max()) > 15:
            raise ValueError("a code of 4 bits is 0..15")
        bits = scales.contiguous().view(torch.int16)
        exact = bool(((bits & 7) == 0).all()) and bool(torch.isfinite(scales).all())
        row_tiles, k_tiles = -(-n // 16), -(-k // 64)
        if row_tiles * 16 != n or k_tiles * 64 != k:
            padded = torch.full((row_tiles * 16, k_tiles * 64), 8, dtype=torch.uint8, device=codes.device)
            padded[:n, :k] = codes
            codes = padded
            wide = torch.zeros((row_tiles * 16, scales.shape[1]), dtype=torch.bfloat16, device=codes.device)
            wide[:n] = scales
            scales = wide
        # [row tile, half, g, k tile, b, t, j, e high, e low] -> [row tile, k tile, g, t, b, j, e low, e high], a byte of the two halves
        c = codes.reshape(row_tiles, 2, 8, k_tiles, 2, 4, 2, 2, 2)
        packed = (c[:, 0] | (c[:, 1] << 4)).permute(0, 2, 1, 4, 3, 5, 7, 6).contiguous().reshape(-1)
        paired = scales.reshape(row_tiles, 2, 8, -1).permute(0, 3, 2, 1).contiguous()
        return Int4Matrix(packed, paired, (n, k), group, exact)

    @staticmethod
    def quantize(w: torch.Tensor, group: int = 64) -> "Int4Matrix":
        """The nearest codes for a matrix of floats; a group's scale is its largest magnitude / 7, rounded up to 5 significant bits, with
        which every weight is a bfloat16 number and the products of few and of many tokens multiply with the same matrix."""
        if group not in GROUPS:
            raise ValueError(f"groups of {GROUPS} weights are possible, not of {group}")
        if w.dim() != 2 or w.numel() == 0 or w.shape[1] % group or not w.is_floating_point():
            raise ValueError(f"a matrix of floats whose columns are a multiple of {group} can be quantized, not {w.dtype} {tuple(w.shape)}")
        n, k = w.shape
        codes, scales = [], []
        for rows in w.split(max(1, (1 << 24) // k)):            # (a large matrix is not copied whole to 32 bits)
            x = rows.float().reshape(-1, k // group, group)
            largest = x.abs().amax(dim=2)
            largest = largest / torch.full_like(largest, 7.0)       # (by a number it is a product with 1/7 on some devices, and another scale)
            if not bool(torch.isfinite(largest).all()):
                raise ValueError("a matrix with undefined or infinite elements cannot be quantized")
            s = ((largest.view(torch.int32) + 0x7FFFF) & ~0x7FFFF).view(torch.float32)
            s = torch.where(s < 2.0 ** -120, torch.zeros_like(s), s)        # (nothing that a product would notice)
            q = torch.round(x / torch.where(s > 0, s, torch.ones_like(s))[:, :, None]).clamp(-8, 7)
            codes.append((torch.where(s[:, :, None] > 0, q, torch.zeros_like(q)) + 8).to(torch.uint8).reshape(-1, k))
            scales.append(s.to(torch.bfloat16))
        return Int4Matrix.from_codes(torch.cat(codes), torch.cat(scales), group)
