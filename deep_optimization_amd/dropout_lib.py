"""Dropout operators with a counter-based mask that is never stored: ``torch.ops.act_lib.dropout_add_fwd`` /
``dropout_bwd`` on the gfx950 kernel behind dopt_dropout. No counterparts in the reference.

    dropout_add_fwd(x, residual, p, seed, offset, step) -> y
    dropout_bwd(dy, p, seed, offset, step, out_dtype) -> dx

y = residual + (kept ? x * scale : 0), elementwise in fp32, in residual's type (x's without one). Element i in row-major
order is kept where half-word i % 8 (little endian in the four output words) of Philox4x32-10 with counter {i / 8,
offset + step} (64 bits each) and key ``seed`` is at least T = round(65536 p); scale = 65536 / (65536 - T). The backward
pass computes the same mask from the same arguments. ``step`` (optional) is a one-element int64 device tensor that the
kernel reads: a program that captures its step in a HIP graph counts it up between replays and draws a new mask on each.
The quantizer's Philox rounding uses the same generator: give the two different seeds.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor

from . import _lib
from .act_lib import _DTYPE_CODE, _U64, _op, _require_cuda, _stream


def _launch(what: str, x: Tensor, residual: Optional[Tensor], p: float, seed: int, offset: int, step: Optional[Tensor], y_dtype: torch.dtype) -> Tensor:
    if x.dtype not in _DTYPE_CODE or y_dtype not in _DTYPE_CODE:
        raise RuntimeError(f"{what}: input and output must be float32, float16 or bfloat16, got {x.dtype} and {y_dtype}")
    if not 0.0 <= p <= 1.0:
        raise RuntimeError(f"{what}: p must lie in [0, 1], got {p}")
    if residual is not None and residual.shape != x.shape:
        raise RuntimeError(f"{what}: residual must have x's shape {tuple(x.shape)}, got {tuple(residual.shape)}")
    if step is not None and (step.dtype != torch.int64 or step.numel() != 1):
        raise RuntimeError(f"{what}: step must be a one-element int64 tensor, got {tuple(step.shape)} {step.dtype}")
    _require_cuda(x, residual, step)
    x = x.contiguous()
    residual = None if residual is None else residual.contiguous()
    y = torch.empty(x.shape, dtype=y_dtype, device=x.device)
    rc = _lib.lib().dopt_dropout(x.data_ptr(), _DTYPE_CODE[x.dtype], None if residual is None else residual.data_ptr(), x.numel(),
                                 float(p), seed & _U64, offset & _U64, None if step is None else step.data_ptr(), y.data_ptr(),
                                 _DTYPE_CODE[y_dtype], _stream(x))
    _lib.check(rc, what)
    return y


def _dropout_add_fwd(x: Tensor, residual: Optional[Tensor], p: float, seed: int, offset: int, step: Optional[Tensor]) -> Tensor:
    return _launch("dropout_add_fwd", x, residual, p, seed, offset, step, x.dtype if residual is None else residual.dtype)


def _dropout_bwd(dy: Tensor, p: float, seed: int, offset: int, step: Optional[Tensor], out_dtype: torch.dtype) -> Tensor:
    return _launch("dropout_bwd", dy, None, p, seed, offset, step, out_dtype)


dropout_add_fwd = _op("dropout_add_fwd(Tensor x, Tensor? residual, float p, int seed, int offset, Tensor? step) -> Tensor",
                      _dropout_add_fwd,
                      lambda x, residual, p, seed, offset, step:
                          x.new_empty(x.shape, dtype=x.dtype if residual is None else residual.dtype))
dropout_bwd = _op("dropout_bwd(Tensor dy, float p, int seed, int offset, Tensor? step, ScalarType out_dtype) -> Tensor",
                  _dropout_bwd, lambda dy, p, seed, offset, step, out_dtype: dy.new_empty(dy.shape, dtype=out_dtype))

__all__ = ["dropout_add_fwd", "dropout_bwd"]
