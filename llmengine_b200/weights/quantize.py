"""Weights of 8 and 4 bits: how a matrix is rounded to them, and how 4-bit codes lie in memory.

8 bits: float8_e4m3fn values with one 32-bit scale a row, w[n, k] ~ scales[n] * q[n, k].  4 bits: codes 0..15 with a bfloat16 scale and,
where asked for, a zero point for every `group` neighbouring values of a row, w[n, k] ~ scales[n, g] * (code[n, k] - zeros[n, g]), g = k //
group; without zero points 8 stands in their place.  These are run once, when a model is loaded, with tensor operations on whichever
device holds the matrix; the products that read the results are `CudaOps.linear_e4m3` and `CudaOps.linear_int4`.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

GROUPS = (32, 64, 128)          # values that may share a scale
BLOCK = 128                     # values in one block of codes (64 bytes)
E4M3_LARGEST = 448.0
LEAST = 2.0 ** -100             # a row's largest value counts as at least this


def _finite(w: torch.Tensor) -> torch.Tensor:
    if w.dim() != 2 or not w.is_floating_point():
        raise ValueError(f"weights must be a matrix of floating-point numbers, got {w.dtype} {tuple(w.shape)}")
    w = w.float()
    if not torch.isfinite(w).all():
        raise ValueError("weights with a NaN or an infinity cannot be rounded to fewer bits")
    return w


def quantize_e4m3(w: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(float8_e4m3fn [N, K], 32-bit scales [N]) of w [N, K]: every row over its largest value, rounded to the nearest."""
    w = _finite(w)
    scales = w.abs().amax(1).clamp(min=LEAST) / E4M3_LARGEST if w.shape[1] else torch.full((w.shape[0],), LEAST / E4M3_LARGEST, device=w.device)
    return (w / scales[:, None]).clamp(-E4M3_LARGEST, E4M3_LARGEST).to(torch.float8_e4m3fn), scales


def pack_int4(codes: torch.Tensor) -> torch.Tensor:
    """Codes 0..15 [N, K] as the kernels read them, uint8 [N, ceil(K / 128) * 64].  A row goes in blocks of 128 values, the last one
    filled up with zeros.  Of a block's sixteen 32-bit words word 4 q + j holds values 32 j + 8 q .. + 7: the even ones in the low half,
    the odd ones in the high half, four bits each, in order."""
    if codes.dim() != 2 or codes.is_floating_point():
        raise ValueError(f"codes must be a matrix of integers, got {codes.dtype} {tuple(codes.shape)}")
    if codes.numel() and (int(codes.min()) < 0 or int(codes.max()) > 15):
        raise ValueError("a code is outside 0..15")
    n, k = codes.shape
    v = torch.nn.functional.pad(codes.to(torch.uint8), (0, -k % BLOCK)).view(n, -(-k // BLOCK), 4, 4, 2, 2, 2)     # block, j, q, byte, nibble, odd
    v = v.permute(0, 1, 3, 2, 6, 4, 5)                                                                # block, q, j, odd, byte, nibble
    return (v[..., 0] | (v[..., 1] << 4)).reshape(n, -(-k // BLOCK) * (BLOCK // 2)).contiguous()


def unpack_int4(packed: torch.Tensor, k: int) -> torch.Tensor:
    """The codes [N, k], uint8, of a matrix that `pack_int4` made."""
    n = packed.shape[0]
    if packed.dtype != torch.uint8 or packed.shape[1] != -(-k // BLOCK) * (BLOCK // 2):
        raise ValueError(f"{k} codes a row take uint8 rows of {-(-k // BLOCK) * (BLOCK // 2)}, got {packed.dtype} {tuple(packed.shape)}")
    v = torch.stack([packed & 15, packed >> 4], -1).view(n, -(-k // BLOCK), 4, 4, 2, 2, 2)                        # block, q, j, odd, byte, nibble
    return v.permute(0, 1, 3, 2, 5, 6, 4).reshape(n, -(-k // BLOCK) * BLOCK)[:, :k].contiguous()


def quantize_int4(w: torch.Tensor, group: int = 128, zeros: bool = False) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """(packed codes, bfloat16 scales [N, ceil(K / group)], zero points uint8 of that shape or None) of w [N, K].  Without zero points a
    group's scale takes its largest value to 7 (codes 1..15); with them it takes the span from its least to its largest value, zero
    included, to 15.  The codes are rounded against the scale as it is stored."""
    if group not in GROUPS:
        raise ValueError(f"a group is of {', '.join(map(str, GROUPS))} values, got {group}")
    w = _finite(w)
    n, k = w.shape
    g = torch.nn.functional.pad(w, (0, -k % group)).view(n, -(-k // group), group)
    if zeros:
        least, most = g.amin(2).clamp(max=0.0), g.amax(2).clamp(min=0.0)
        scales = ((most / 2 - least / 2) / 7.5).clamp(min=LEAST).to(torch.bfloat16)        # (halves: a span may be twice the largest number)
        at = (-least / scales.float()).round().clamp(0, 15)
    else:
        scales = (g.abs().amax(2) / 7).clamp(min=LEAST).to(torch.bfloat16)
        at = torch.full_like(scales, 8.0, dtype=torch.float32)
    codes = (g / scales.float()[..., None] + at[..., None]).round().clamp(0, 15)
    return pack_int4(codes.flatten(1)[:, :k].to(torch.uint8)), scales, at.to(torch.uint8) if zeros else None


def dequantize_int4(packed: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor], k: int, group: int) -> torch.Tensor:
    """The 32-bit matrix [N, k] that packed codes, scales and zero points stand for."""
    at = torch.arange(k, device=packed.device) // group
    zero = zeros.float()[:, at] if zeros is not None else 8.0
    return (unpack_int4(packed, k).float() - zero) * scales.float()[:, at]
