"""The Linear layer's products with bias, activation and residual in their epilogue: ``torch.ops.act_lib.linear_act_fwd`` /
``linear_act_bwd`` / ``gated_linear_fwd`` / ``gated_linear_bwd`` on the gfx950 MFMA kernels behind dopt_linear_forward,
dopt_linear_input_grad, dopt_linear_weight_grad, dopt_gated_forward and dopt_gated_input_grad. No counterparts in the reference, whose Linear layers call F.linear
(Activation_Compression/modules/ops.py:481) and whose activations are separate modules.

    linear_act_fwd(x, weight, bias, residual, act, save_pre) -> (y, pre)
        z = x weight^T + bias;  y = act(z) + residual;  pre = z (None unless save_pre)
    linear_act_bwd(dy, x, weight, pre, act, in_pre, in_act, input_grad, weight_grad, bias_grad, grad_dtype)
            -> (dx, dweight, dbias)
        dz = dy act'(pre);  dx = (dz weight) in_act'(in_pre);  dweight = dz^T x;  dbias = sum of dz over the rows

x [..., K] and weight [N, K] in bf16 or fp16 (fp32 sums, fp32 epilogue, each result rounded once), ``act`` one of "none",
"relu", "gelu" (the exact one), "gelu_tanh", "silu". bias [N] in bf16, fp16 or fp32; residual [..., N] in x's type or fp32,
y in residual's type (x's without one). pre [..., N] in x's type.

Backward: dy and pre [..., N] in x's type. With ``in_act`` other than "none", x is in_act(in_pre), the output of the
activation that feeds the layer, and dx is the gradient of in_pre [..., K]: an MLP's second layer hands its first one the
gradient of the pre-activation in one pass. dz is rounded to x's type for the products, which read it on matrix instructions of
that type: with an activation dx and dweight are then off by that rounding beside their own (0.0023 of their norm where the one
rounding alone is 0.0017, 2001 rows of 333 -> 1001 in bf16). dz as a sum of two 16-bit terms would keep twice the bits and double the
products: their measured times put 25216 x 768 -> 3072 with GELU at 560 us for 334. dbias is the sum of dz before that rounding.
dweight and dbias come in ``grad_dtype`` (float32 or x's type; both are summed in fp32); what is not asked for is None. The weight gradient's product sums an activation-less dz on its
way; without that product, or with an activation, the launch that writes dz (or one that writes nothing else) makes dbias.

    gated_linear_fwd(x, weight, bias, act, save_pre) -> (h, pre)
        g = x weight[:H]^T + bias[:H],  u = x weight[H:]^T + bias[H:];  h = act(g) u;  pre = g, u beside each other (None unless save_pre)
    gated_linear_bwd(dy, out_weight, pre, act, hidden) -> (dpre, h)
        dh = dy out_weight (out_weight None: dy);  dpre = dh u act'(g), dh act(g) beside each other;  h = act(g) u (None unless hidden)

The gated layer: weight [2 H, K], bias [2 H], h [..., H], pre and dpre [..., 2 H]; both projections, the activation and the product in one
kernel. Its backward pass with the Linear layer behind it (out_weight [N, H], dy [..., N]) is one product too, which makes dpre from its sums, and
h once more for out_weight's gradient, so that a caller who asks for it may keep x and pre only; x's and weight's gradients are linear_act_bwd(dpre, x, weight, None, "none", ..).
h comes from the fp32 sums, rounded once; the backward pass reads g and u as pre holds them, in x's type, and rounds dpre to it: x's and
weight's gradients are then off by 0.003 of their norm where their own rounding alone is 0.0017 (25216 rows of 768 -> 2 x 2048 with
silu in bf16). pre in fp32 would double the 207 MB that are written and read there, some 80 us of 800, and leave dpre's rounding.

Rows may be strided (x[:, 0] of a [B, T, K] tensor) and lie at any element. Where they start at multiples of 16 bytes
and hold whole 16-byte chunks the faster kernels read them; others are read through registers, or copied into
aligned rows first where that is estimated to be faster (dopt_linear_copy_preferred).
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor

from . import _lib
from .act_lib import _DTYPE_CODE, _op, _require_cuda, _stream

_TYPES = (torch.bfloat16, torch.float16)


def _act_code(act: str) -> int:
    try:
        return _lib.LIN_ACTS[act]
    except KeyError:
        raise ValueError(f"act must be one of {', '.join(_lib.LIN_ACTS)}, got {act!r}") from None


def _pad8(n: int) -> int:
    return (n + 7) // 8 * 8


class _Rows:
    """An operand [rows, cols] as the products read it: contiguous rows ``ld`` apart, ``whole`` where they hold whole 16-byte
    chunks. ``copy``: it is going to be laid out again; ``written``: it is an activation's gradient, which is written anyway."""

    def __init__(self, t: Tensor, rows: int, cols: int, written: bool = False):
        t2 = t.reshape(rows, cols) if t.dim() != 2 else t
        if t2.stride(1) != 1 or not cols <= t2.stride(0) < 1 << 21:
            t2 = t2.contiguous()
        self.t, self.rows, self.cols, self.copy, self.written = t2, rows, cols, False, written
        self.ld = cols if rows <= 1 else int(t2.stride(0))
        if written:
            self.whole = cols % 8 == 0
            return
        # (the last row's last chunk must be there too)
        self.whole = self.ld % 8 == 0 and self.ld >= _pad8(cols) and t2.data_ptr() % 16 == 0 and (
            cols % 8 == 0 or (t2.storage_offset() + (rows - 1) * self.ld + _pad8(cols)) * 2 <= t2.untyped_storage().nbytes())

    @property
    def loose(self) -> bool:
        return not (self.whole or self.copy)


def _plan(product: int, M: int, N: int, K: int, a: _Rows, b: _Rows, launched: bool) -> None:
    """Marks the loose ones of a product's operands for a copy into aligned rows, where that is estimated to be faster;
    ``launched``: others are laid out anyway, by the same launch."""
    loose = [r for r in (a, b) if r.loose]
    copies = [r for r in loose if not r.written]
    if loose and _lib.lib().dopt_linear_copy_preferred(product, M, N, K, sum(r.rows * r.cols for r in copies), int(bool(copies) and not launched)):
        for r in loose:
            r.copy = True


def _layout(items, dtype: torch.dtype, stream) -> None:
    """One launch that lays out [(operand, pre, act, sum)]; each then holds its new rows. With an activation the rows become dy act'(pre),
    padded only where a copy is marked; ``sum`` (or None) receives their columns' sums, which is all that an operand gets that is neither
    to be copied nor written."""
    if not items:
        return
    rows, kept = (_lib.LinearRows * len(items))(), []
    for d, (r, pre, act, total) in zip(rows, items):
        width = _pad8(r.cols) if r.copy else r.cols if r.written else 0
        out = torch.empty((r.rows, width), dtype=dtype, device=r.t.device) if width else None
        n, cols, src, dst = r.rows, r.cols, r.ld, width
        space = None
        if total is not None:
            floats = int(_lib.lib().dopt_linear_layout_workspace_floats(n, cols))
            space = torch.empty(floats, dtype=torch.float32, device=r.t.device) if floats else None
            d.sum, d.sum_dtype, d.workspace = total.data_ptr(), _DTYPE_CODE[total.dtype], None if space is None else space.data_ptr()
        elif width == cols == r.ld:  # a contiguous matrix as one row
            n, cols, src, dst = 1, n * cols, n * cols, n * cols
        # (what the launch reads lives until then: the next result could take its memory)
        kept.append((r.t, space))
        d.src, d.ld_src, d.pre, d.rows, d.cols, d.dst, d.ld_dst, d.act = (r.t.data_ptr(), src, None if pre is None else pre.data_ptr(), n,
                                                                          cols, None if out is None else out.data_ptr(), dst, act)
        if out is not None:
            r.t, r.ld, r.whole, r.copy = out, width, width % 8 == 0, False
    _lib.check(_lib.lib().dopt_linear_layout(rows, len(items), _DTYPE_CODE[dtype], stream), "linear_act")


def _check_operands(what: str, x: Tensor, weight: Tensor):
    """(rows, N, K)"""
    if x.dtype not in _TYPES or weight.dtype != x.dtype or x.dim() < 1 or weight.dim() != 2 or weight.shape[1] != x.shape[-1]:
        raise RuntimeError(f"{what}: x [..., K] and weight [N, K] must both be bfloat16 or float16, got {tuple(x.shape)} {x.dtype} and "
                           f"{tuple(weight.shape)} {weight.dtype}")
    rows = 1
    for n in x.shape[:-1]:
        rows *= int(n)
    return rows, int(weight.shape[0]), int(weight.shape[1])


def _check_like(what: str, name: str, t: Tensor, shape, dtypes) -> None:
    if tuple(t.shape) != tuple(shape) or t.dtype not in dtypes:
        raise RuntimeError(f"{what}: {name} must be {tuple(shape)} in {' or '.join(str(d) for d in dtypes)}, got {tuple(t.shape)} {t.dtype}")


def _linear_act_fwd(x: Tensor, weight: Tensor, bias: Optional[Tensor], residual: Optional[Tensor], act: str, save_pre: bool):
    what = "linear_act_fwd"
    code = _act_code(act)
    M, N, K = _check_operands(what, x, weight)
    shape = (*x.shape[:-1], N)
    if bias is not None:
        _check_like(what, "bias", bias, (N,), tuple(_DTYPE_CODE))
    if residual is not None:
        _check_like(what, "residual", residual, shape, (x.dtype, torch.float32))
    _require_cuda(x, weight, bias, residual)
    a, b = _Rows(x, M, K), _Rows(weight, N, K)
    if M and N and K:
        _plan(0, M, N, K, a, b, False)
        _layout([(r, None, 0, None) for r in (a, b) if r.copy], x.dtype, _stream(x))
    bias = None if bias is None else bias.contiguous()
    residual = None if residual is None else residual.contiguous()
    y = torch.empty(shape, dtype=x.dtype if residual is None else residual.dtype, device=x.device)
    pre = torch.empty(shape, dtype=x.dtype, device=x.device) if save_pre else None
    rc = _lib.lib().dopt_linear_forward(
        a.t.data_ptr(), a.ld, b.t.data_ptr(), b.ld, _DTYPE_CODE[x.dtype], M, N, K, None if bias is None else bias.data_ptr(),
        _lib.F32 if bias is None else _DTYPE_CODE[bias.dtype], None if residual is None else residual.data_ptr(), code,
        y.data_ptr(), _DTYPE_CODE[y.dtype], None if pre is None else pre.data_ptr(), _stream(x))
    _lib.check(rc, what)
    return y, pre


def _linear_act_fwd_fake(x, weight, bias, residual, act, save_pre):
    shape = (*x.shape[:-1], weight.shape[0])
    return x.new_empty(shape, dtype=x.dtype if residual is None else residual.dtype), (x.new_empty(shape) if save_pre else None)


linear_act_fwd = _op(
    "linear_act_fwd(Tensor x, Tensor weight, Tensor? bias, Tensor? residual, str act, bool save_pre) -> (Tensor, Tensor?)",
    _linear_act_fwd, _linear_act_fwd_fake)


def _linear_act_bwd(dy: Tensor, x: Tensor, weight: Tensor, pre: Optional[Tensor], act: str, in_pre: Optional[Tensor], in_act: str,
                    input_grad: bool, weight_grad: bool, bias_grad: bool, grad_dtype: torch.dtype):
    what = "linear_act_bwd"
    code, in_code = _act_code(act), _act_code(in_act)
    M, N, K = _check_operands(what, x, weight)
    _check_like(what, "dy", dy, (*x.shape[:-1], N), (x.dtype,))
    if grad_dtype not in (torch.float32, x.dtype):
        raise RuntimeError(f"{what}: grad_dtype must be float32 or x's type, got {grad_dtype}")
    if (code != 0) != (pre is not None):
        raise RuntimeError(f"{what}: pre goes with an activation (act {act!r}, pre {'given' if pre is not None else 'missing'})")
    if (in_code != 0) != (in_pre is not None):
        raise RuntimeError(f"{what}: in_pre goes with in_act (in_act {in_act!r}, in_pre {'given' if in_pre is not None else 'missing'})")
    if pre is not None:
        _check_like(what, "pre", pre, dy.shape, (x.dtype,))
    if in_pre is not None:
        _check_like(what, "in_pre", in_pre, x.shape, (x.dtype,))
    _require_cuda(dy, x, weight, pre, in_pre)
    L, dt, stream = _lib.lib(), _DTYPE_CODE[x.dtype], _stream(x)
    empty = M == 0 or N == 0 or K == 0
    # dz is dy, or written by the launch that lays out the operands whose rows the products do better to read aligned;
    # that launch makes its sums where no product does, or only once it is rounded
    db = torch.empty(N, dtype=grad_dtype, device=x.device) if bias_grad else None
    summed = db is not None and (code != 0 or not weight_grad or K == 0 or M == 0)
    z = code != 0 and M > 0 and N > 0 and (input_grad or weight_grad)
    dz, w, xr = _Rows(dy, M, N, z), _Rows(weight, N, K), _Rows(x, M, K)
    if not empty:
        if input_grad:
            _plan(1, M, N, K, dz, w, z or summed)
        if weight_grad:
            _plan(2, M, N, K, dz, xr, z or summed or dz.copy or w.copy)
    pre = None if pre is None else pre.contiguous()
    _layout([(r, p, a, s) for r, p, a, s in ((dz, pre, code, db if summed else None), (w, None, 0, None), (xr, None, 0, None))
             if r.copy or r.written or s is not None], x.dtype, stream)
    dx = dw = None
    dx_args = dw_args = ()
    if input_grad:
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        in_pre = None if in_pre is None else in_pre.contiguous()
        dx_args = (None if in_pre is None else in_pre.data_ptr(), in_code, dx.data_ptr())
    K8 = K
    if weight_grad:
        # the kernels that split the sum write whole chunks of a row
        if K % 8 and N and dz.whole and xr.whole and L.dopt_linear_tile(2, M, N, _pad8(K), 0) == 100:
            K8 = _pad8(K)
        dw = torch.empty((N, K8), dtype=grad_dtype, device=x.device)
        if N and K:
            ws = torch.empty(max(int(L.dopt_linear_weight_grad_workspace_floats(M, N, K8)), 4), dtype=torch.float32, device=x.device)
            f32 = grad_dtype == torch.float32
            dbp = None if db is None or summed else db.data_ptr()
            dw_args = (ws.data_ptr(), dw.data_ptr() if f32 else None, None if f32 else dw.data_ptr(), dbp if f32 else None, None if f32 else dbp)
    if dx_args and dw_args and K8 == K:
        _lib.check(L.dopt_linear_backward(dz.t.data_ptr(), dz.ld, xr.t.data_ptr(), xr.ld, w.t.data_ptr(), w.ld, dt, M, N, K, *dx_args, *dw_args,
                                          stream), what)
    else:
        if dx_args:
            _lib.check(L.dopt_linear_input_grad(dz.t.data_ptr(), dz.ld, w.t.data_ptr(), w.ld, dt, M, N, K, *dx_args, stream), what)
        if dw_args:
            _lib.check(L.dopt_linear_weight_grad(dz.t.data_ptr(), dz.ld, xr.t.data_ptr(), xr.ld, dt, M, N, K8, *dw_args, stream), what)
    if K8 != K:
        dw = dw[:, :K].contiguous()
    return dx, dw, db


def _linear_act_bwd_fake(dy, x, weight, pre, act, in_pre, in_act, input_grad, weight_grad, bias_grad, grad_dtype):
    return (x.new_empty(x.shape) if input_grad else None, weight.new_empty(weight.shape, dtype=grad_dtype) if weight_grad else None,
            weight.new_empty((weight.shape[0],), dtype=grad_dtype) if bias_grad else None)


linear_act_bwd = _op(
    "linear_act_bwd(Tensor dy, Tensor x, Tensor weight, Tensor? pre, str act, Tensor? in_pre, str in_act, bool input_grad, "
    "bool weight_grad, bool bias_grad, ScalarType grad_dtype) -> (Tensor?, Tensor?, Tensor?)", _linear_act_bwd, _linear_act_bwd_fake)



def _gated_linear_fwd(x: Tensor, weight: Tensor, bias: Optional[Tensor], act: str, save_pre: bool):
    what = "gated_linear_fwd"
    code = _act_code(act)
    M, N, K = _check_operands(what, x, weight)
    if N % 2:
        raise RuntimeError(f"{what}: weight must hold as many rows for the gate as for the up projection, got {tuple(weight.shape)}")
    if bias is not None:
        _check_like(what, "bias", bias, (N,), tuple(_DTYPE_CODE))
    _require_cuda(x, weight, bias)
    a, b = _Rows(x, M, K), _Rows(weight, N, K)
    if M and N and K:
        _plan(0, M, N, K, a, b, False)
        _layout([(r, None, 0, None) for r in (a, b) if r.copy], x.dtype, _stream(x))
    bias = None if bias is None else bias.contiguous()
    h = torch.empty((*x.shape[:-1], N // 2), dtype=x.dtype, device=x.device)
    pre = torch.empty((*x.shape[:-1], N), dtype=x.dtype, device=x.device) if save_pre else None
    rc = _lib.lib().dopt_gated_forward(
        a.t.data_ptr(), a.ld, b.t.data_ptr(), b.ld, _DTYPE_CODE[x.dtype], M, N // 2, K, None if bias is None else bias.data_ptr(),
        _lib.F32 if bias is None else _DTYPE_CODE[bias.dtype], code, h.data_ptr(), None if pre is None else pre.data_ptr(), _stream(x))
    _lib.check(rc, what)
    return h, pre


def _gated_linear_fwd_fake(x, weight, bias, act, save_pre):
    N = weight.shape[0]
    return x.new_empty((*x.shape[:-1], N // 2)), (x.new_empty((*x.shape[:-1], N)) if save_pre else None)


gated_linear_fwd = _op(
    "gated_linear_fwd(Tensor x, Tensor weight, Tensor? bias, str act, bool save_pre) -> (Tensor, Tensor?)",
    _gated_linear_fwd, _gated_linear_fwd_fake)


def _gated_linear_bwd(dy: Tensor, out_weight: Optional[Tensor], pre: Tensor, act: str, hidden: bool):
    what = "gated_linear_bwd"
    code = _act_code(act)
    if pre.dtype not in _TYPES or pre.dim() < 1 or pre.shape[-1] % 2:
        raise RuntimeError(f"{what}: pre [..., 2 H] must be bfloat16 or float16, got {tuple(pre.shape)} {pre.dtype}")
    H = int(pre.shape[-1]) // 2
    if out_weight is not None and (out_weight.dim() != 2 or out_weight.dtype != pre.dtype or out_weight.shape[1] != H):
        raise RuntimeError(f"{what}: out_weight must be [N, {H}] in pre's type, got {tuple(out_weight.shape)} {out_weight.dtype}")
    N = H if out_weight is None else int(out_weight.shape[0])
    _check_like(what, "dy", dy, (*pre.shape[:-1], N), (pre.dtype,))
    _require_cuda(dy, out_weight, pre)
    M = 1
    for n in pre.shape[:-1]:
        M *= int(n)
    a, b = _Rows(dy, M, N), None if out_weight is None else _Rows(out_weight, N, H)
    if b is not None and M and N and H:
        _plan(1, M, N, H, a, b, False)
        _layout([(r, None, 0, None) for r in (a, b) if r.copy], pre.dtype, _stream(pre))
    pre = pre.contiguous()
    dpre = torch.empty_like(pre)
    h = torch.empty((*pre.shape[:-1], H), dtype=pre.dtype, device=pre.device) if hidden else None
    # (an out_weight without rows has no address of its own: any but null says that there is one)
    weight = None if b is None else b.t.data_ptr() if N else pre.data_ptr()
    rc = _lib.lib().dopt_gated_input_grad(a.t.data_ptr(), a.ld, weight, 0 if b is None else b.ld, _DTYPE_CODE[pre.dtype],
                                          M, N, H, pre.data_ptr(), code, dpre.data_ptr(), None if h is None else h.data_ptr(), _stream(pre))
    _lib.check(rc, what)
    return dpre, h


def _gated_linear_bwd_fake(dy, out_weight, pre, act, hidden):
    return pre.new_empty(pre.shape), (pre.new_empty((*pre.shape[:-1], pre.shape[-1] // 2)) if hidden else None)


gated_linear_bwd = _op(
    "gated_linear_bwd(Tensor dy, Tensor? out_weight, Tensor pre, str act, bool hidden) -> (Tensor, Tensor?)",
    _gated_linear_bwd, _gated_linear_bwd_fake)

__all__ = ["linear_act_fwd", "linear_act_bwd", "gated_linear_fwd", "gated_linear_bwd"]
