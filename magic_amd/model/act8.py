"""Activations kept for the backward pass in 8 bits.

A linear layer keeps its input until its weight gradient is formed.  Where nothing else keeps that matrix, 8 bits save
three quarters of its memory.  ``act8_pack`` stores a float32 matrix as signed 8-bit codes with one
power-of-two scale for every 32 columns of a row (1.03 bytes an element instead of 4), ``act8_unpack`` reads it back,
and ``linear_nobias(x, w, act_bits=8)`` (``gat.py``) forms its weight gradient from the codes.  The rounding is off by
at most half a step, 2^-7.98 of a block's largest magnitude at worst.  No counterpart in the reference, which keeps
float32 activations.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from .. import _lib


class Act8(NamedTuple):
    """``codes`` int8 [N, stride], ``exps`` uint8 [N, ceil(F / 32)], ``cols`` = F."""
    codes: torch.Tensor
    exps: torch.Tensor
    cols: int


def act8_pack(x: torch.Tensor) -> Act8:
    """Codes of a float32 [N, F] matrix on the GPU: x ~ code * 2^(exp - 127), rounded to nearest even.  A block of 32
    columns that holds an infinity or a NaN reads back as NaN."""
    codes, exps = _lib.act8_pack(x)
    return Act8(codes, exps, x.shape[1])


def act8_unpack(a: Act8) -> torch.Tensor:
    """The float32 [N, F] matrix the codes stand for."""
    return _lib.act8_unpack(a.codes, a.exps, a.cols)


def act8_weight_grad(dy: torch.Tensor, a: Act8) -> torch.Tensor:
    """``dy.T @ act8_unpack(a)`` without the unpacked matrix: [M, F] for dy [N, M]."""
    return _lib.act8_weight_grad(dy, a.codes, a.exps, a.cols)
