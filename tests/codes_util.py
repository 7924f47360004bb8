"""Rows in 8 bits by their definition, in exact rational arithmetic or float64."""

from __future__ import annotations

from fractions import Fraction

import numpy as np
import torch

#: Magnitudes that an e4m3fn code stands for, by code.
E4M3 = [Fraction((8 * (e > 0) + m) * 2**max(e, 1), 2**10) for e in range(16) for m in range(8)][:127]


def nearest(q: Fraction, codes: torch.dtype) -> Fraction:
    """The code's number nearest to q, ties to the even code."""
    grid = [Fraction(i) for i in range(128)] if codes == torch.int8 else E4M3
    size = abs(q)
    best = min(range(len(grid)), key=lambda i: (abs(grid[i] - size), i % 2))
    return grid[best] if q >= 0 else -grid[best]


def rows(x: torch.Tensor, codes: torch.dtype) -> tuple[torch.Tensor, torch.Tensor]:
    """(numbers of the codes in fp64, scales): row by row, with fractions."""
    top = np.float32(127.0 if codes == torch.int8 else 448.0)
    flat = x.detach().cpu().float().reshape(-1, x.shape[-1]).numpy()
    out, scales = np.zeros(flat.shape), np.ones(len(flat), dtype=np.float32)
    for i, row in enumerate(flat):
        if not np.isfinite(row).all():
            scales[i] = np.nan
            continue
        s = np.abs(row).max() * (np.float32(1) / top) if len(row) else np.float32(0)
        scales[i] = s if s > 0 else 1.0
        out[i] = [float(nearest(Fraction(float(v)) / Fraction(float(scales[i])), codes)) for v in row]
    return torch.from_numpy(out).view(x.shape), torch.from_numpy(scales).view(x.shape[:-1])


def hard_rows(dtype: torch.dtype, cols: int = 64, seed: int = 0) -> torch.Tensor:
    """Rows of many sizes, zeros, single values, the type's ends, and values next
    to the middle between two codes."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(24, cols, generator=gen)
    x[1] = 0.0
    x[2] = -0.0
    x[3] = 0.0
    x[3, cols // 2] = -1.5
    x[4] *= 1e-4
    x[5] *= 3e3
    x[6, :] = 1.0
    x[7] = torch.arange(cols) - cols // 2
    x[8] = (torch.arange(cols) % 127 + 0.5) * (1 - 2 * (torch.arange(cols) % 2))
    x[8, 0] = 127.0
    x[9] = (torch.arange(cols) % 127 + 0.5) * 1.37
    x[9, 0] = 127.0 * 1.37
    x = x.to(dtype)
    info = torch.finfo(dtype)
    x[10] = info.max
    x[11, :] = info.tiny
    x[12] = torch.randn(cols, generator=gen).to(dtype) * info.tiny
    x[13, 0] = info.max
    x[14, ::2] = info.smallest_normal / 4
    x[15, 1] = float("nan")
    x[16, 2] = float("inf")
    x[17, 3] = -float("inf")
    if dtype == torch.float32:
        x[18] *= 1e-40
        x[19] *= 1e-30
        x[20] = torch.arange(cols) * 2.0**-149
        x[21] = 190 * 2.0**-149
    return x
