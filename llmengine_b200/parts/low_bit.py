"""Weights of 8 and 4 bits in the parts that take them, and the rows that the 8-bit ones multiply.

A part hands its matrix to `hold` when it is loaded and emits its product with `emit_linear`; which kind of product that is follows from
`Runtime.weights`.  Matrices held as they are stay the tensors they were, and their products the records they were.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Union

import torch

from ..engine.plan import Plan
from ..weights.quantize import quantize_e4m3, quantize_int4
from .base import Runtime


@dataclass
class Rows8:
    """Rows of 8-bit numbers: data [T, D] float8_e4m3fn, scales [T] 32-bit."""

    data: torch.Tensor
    scales: torch.Tensor


@dataclass
class E4M3Weight:
    """A matrix [N, K] in 8 bits with a scale for every row."""

    data: torch.Tensor
    scales: torch.Tensor

    def __getitem__(self, rows: slice) -> "E4M3Weight":
        return E4M3Weight(self.data[rows], self.scales[rows])


@dataclass
class Int4Weight:
    """A matrix [N, K] in 4 bits: packed codes, scales and (or None) zero points."""

    codes: torch.Tensor
    scales: torch.Tensor
    zeros: Optional[torch.Tensor]
    group: int

    def __getitem__(self, rows: slice) -> "Int4Weight":
        return Int4Weight(self.codes[rows], self.scales[rows], None if self.zeros is None else self.zeros[rows], self.group)


Weight = Union[torch.Tensor, E4M3Weight, Int4Weight]


def hold(rt: Runtime, w: torch.Tensor, name: str) -> Weight:
    """The matrix as this runtime's products read it; `name` is for the error that says why it cannot be."""
    if rt.weights == "stored":
        return w
    need = 16 if rt.weights == "e4m3" else 8
    if w.shape[1] % need:
        raise ValueError(f"{name}: weights {rt.weights!r} need rows of a multiple of {need} values, this matrix has {w.shape[1]}")
    try:
        if rt.weights == "e4m3":
            return E4M3Weight(*quantize_e4m3(w))
        return Int4Weight(*quantize_int4(w, rt.weight_group, rt.weight_zero_points), rt.weight_group)
    except ValueError as e:
        raise ValueError(f"{name}: {e}") from None


def rows8_place(rt: Runtime, name: str, size: int) -> Rows8:
    return Rows8(rt.workspace(name, size, torch.float8_e4m3fn), rt.workspace(name + "_scales", 1, torch.float32).view(-1))


def emit_linear(plan: Plan, rt: Runtime, h: Union[torch.Tensor, Rows8], w: Weight, out: torch.Tensor, rows_name: str) -> None:
    """out = h w^T.  Rows that are not 8-bit yet become so, in the workspace `rows_name`, where the weights are."""
    if isinstance(w, E4M3Weight):
        if not isinstance(h, Rows8):
            place = rows8_place(rt, rows_name, h.shape[1])
            plan.rows_e4m3(h, place.data, place.scales)
            h = place
        plan.linear_e4m3(h.data, h.scales, w.data, w.scales, out)
    elif isinstance(w, Int4Weight):
        plan.linear_int4(h, w.codes, w.scales, w.zeros, w.group, out)
    else:
        plan.linear(h, w, out)
