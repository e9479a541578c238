"""Layer norm operators: ``torch.ops.act_lib.layer_norm_fwd`` / ``layer_norm_bwd`` on the gfx950 kernels behind
dopt_layer_norm_forward / dopt_layer_norm_backward. No counterparts in the reference (its Transformer models leave layer
norm to torch; Activation_Compression/layers.py:206-216 has an RMSNorm module in plain torch).

    layer_norm_fwd(x, weight, bias, eps, out_dtype) -> (y, mean, rstd)
    layer_norm_bwd(dy, x, mean, rstd, weight, dresidual, weight_grad, bias_grad) -> (dx, dweight, dbias)

x [..., D] in fp32, fp16 or bf16, normalized over its last axis in fp32; y in ``out_dtype`` (any of the three); mean and
rstd fp32 [...]. weight and bias [D] in any of the three types (the same one where both are given). The backward pass
takes dy in any of them, adds ``dresidual`` (x's shape and type: the gradient that reaches x past the norm, as in
x + f(norm(x))) and returns dx in x's type and fp32 dweight / dbias (None where not asked for).
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor

from . import _lib
from .act_lib import _DTYPE_CODE, _op, _require_cuda, _stream


def _ptr(t: Optional[Tensor]):
    return None if t is None else t.data_ptr()


def _check_params(what: str, D: int, weight: Optional[Tensor], bias: Optional[Tensor]) -> int:
    """The parameters' type code."""
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if p.numel() != D or p.dim() != 1 or p.dtype not in _DTYPE_CODE:
            raise RuntimeError(f"{what}: {name} must be a float32, float16 or bfloat16 vector of {D} values, got {tuple(p.shape)} {p.dtype}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise RuntimeError(f"{what}: weight and bias must have one type, got {weight.dtype} and {bias.dtype}")
    p = weight if weight is not None else bias
    return _lib.F32 if p is None else _DTYPE_CODE[p.dtype]


def _check_x(what: str, x: Tensor) -> int:
    if x.dim() < 1 or x.shape[-1] < 1 or x.dtype not in _DTYPE_CODE:
        raise RuntimeError(f"{what}: x must be a float32, float16 or bfloat16 tensor [..., D] with D >= 1, got {tuple(x.shape)} {x.dtype}")
    return int(x.shape[-1])


def _layer_norm_fwd(x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], eps: float, out_dtype: torch.dtype):
    D = _check_x("layer_norm_fwd", x)
    code = _check_params("layer_norm_fwd", D, weight, bias)
    if out_dtype not in _DTYPE_CODE:
        raise RuntimeError(f"layer_norm_fwd: out_dtype must be float32, float16 or bfloat16, got {out_dtype}")
    _require_cuda(x, weight, bias)
    x = x.contiguous()
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    y = torch.empty(x.shape, dtype=out_dtype, device=x.device)
    mean = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    rstd = torch.empty_like(mean)
    rc = _lib.lib().dopt_layer_norm_forward(x.data_ptr(), _DTYPE_CODE[x.dtype], mean.numel(), D, _ptr(weight), _ptr(bias), code,
                                            float(eps), y.data_ptr(), _DTYPE_CODE[out_dtype], mean.data_ptr(), rstd.data_ptr(), _stream(x))
    _lib.check(rc, "layer_norm_fwd")
    return y, mean, rstd


layer_norm_fwd = _op(
    "layer_norm_fwd(Tensor x, Tensor? weight, Tensor? bias, float eps, ScalarType out_dtype) -> (Tensor, Tensor, Tensor)",
    _layer_norm_fwd,
    lambda x, weight, bias, eps, out_dtype: (x.new_empty(x.shape, dtype=out_dtype), x.new_empty(x.shape[:-1], dtype=torch.float32),
                                             x.new_empty(x.shape[:-1], dtype=torch.float32)))


def _layer_norm_bwd(dy: Tensor, x: Tensor, mean: Tensor, rstd: Tensor, weight: Optional[Tensor], dresidual: Optional[Tensor],
                    weight_grad: bool, bias_grad: bool):
    D = _check_x("layer_norm_bwd", x)
    code = _check_params("layer_norm_bwd", D, weight, None)
    rows = x.numel() // D
    if dy.shape != x.shape or dy.dtype not in _DTYPE_CODE:
        raise RuntimeError(f"layer_norm_bwd: dy must be a float32, float16 or bfloat16 tensor of x's shape {tuple(x.shape)}, got {tuple(dy.shape)} {dy.dtype}")
    for name, t in (("mean", mean), ("rstd", rstd)):
        if t.numel() != rows or t.dtype != torch.float32:
            raise RuntimeError(f"layer_norm_bwd: {name} must hold {rows} float32 values, got {tuple(t.shape)} {t.dtype}")
    if dresidual is not None and (dresidual.shape != x.shape or dresidual.dtype != x.dtype):
        raise RuntimeError(f"layer_norm_bwd: dresidual must have x's shape and type, got {tuple(dresidual.shape)} {dresidual.dtype}")
    _require_cuda(dy, x, mean, rstd, weight, dresidual)
    dy, x, mean, rstd = dy.contiguous(), x.contiguous(), mean.contiguous(), rstd.contiguous()
    weight = None if weight is None else weight.contiguous()
    dresidual = None if dresidual is None else dresidual.contiguous()
    L = _lib.lib()
    dx = torch.empty_like(x)
    dw = torch.empty(D, dtype=torch.float32, device=x.device) if weight_grad else None
    db = torch.empty(D, dtype=torch.float32, device=x.device) if bias_grad else None
    floats = int(L.dopt_layer_norm_workspace_floats(rows, D)) if weight_grad or bias_grad else 0
    ws = torch.empty(floats, dtype=torch.float32, device=x.device) if floats else None
    rc = L.dopt_layer_norm_backward(dy.data_ptr(), _DTYPE_CODE[dy.dtype], x.data_ptr(), _DTYPE_CODE[x.dtype], rows, D,
                                    mean.data_ptr(), rstd.data_ptr(), _ptr(weight), code, _ptr(dresidual), dx.data_ptr(),
                                    _ptr(ws), _ptr(dw), _ptr(db), _stream(x))
    _lib.check(rc, "layer_norm_bwd")
    return dx, dw, db


def _layer_norm_bwd_fake(dy, x, mean, rstd, weight, dresidual, weight_grad, bias_grad):
    D = x.shape[-1]
    return (x.new_empty(x.shape), x.new_empty((D,), dtype=torch.float32) if weight_grad else None,
            x.new_empty((D,), dtype=torch.float32) if bias_grad else None)


layer_norm_bwd = _op(
    "layer_norm_bwd(Tensor dy, Tensor x, Tensor mean, Tensor rstd, Tensor? weight, Tensor? dresidual, bool weight_grad, "
    "bool bias_grad) -> (Tensor, Tensor?, Tensor?)", _layer_norm_bwd, _layer_norm_bwd_fake)

__all__ = ["layer_norm_fwd", "layer_norm_bwd"]
