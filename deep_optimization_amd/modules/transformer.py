"""Layers of a pre-norm transformer block on the layer norm, dropout and linear operators (``ln_lib``, ``dropout_lib``,
``linear_lib``). No counterparts in the reference, whose transformer models use torch's modules.

Functional forms on the GPU, differentiable once in reverse mode (forward mode and second derivatives raise):

    layer_norm(x, weight, bias, eps)                      in the autocast dtype under autocast, else in x's
    layer_norm_residual(x, weight, bias, eps)             (layer_norm(x), x); its backward adds the gradient that reaches x
                                                          past the norm while it writes the norm's own
    linear_act(x, weight, bias, residual, act)            act(x weight^T + bias) + residual
    mlp(x, w1, b1, w2, b2, residual, act)                 act(x w1^T + b1) w2^T + b2 + residual; its backward hands the first
                                                          layer the gradient of its pre-activation in one pass
    dropout_add(x, residual, p, seed, offset, step)       residual + dropout(x)

and as modules with torch's parameter names: LayerNorm, LinearAct, Mlp, DropoutAdd (with DropoutRng, the count that gives
every pass of a model its own masks). Products run in bf16 or fp16: of that type, or under autocast.

Gradients between the operators are in the products' type, as torch's are under autocast: mlp hands its first layer dz in 16 bits, so
b1's gradient sums rounded terms (linear_act's sums fp32 ones), and an fp32 gradient that comes in (of an fp32
residual's sum) is rounded to 16 bits for the products and the bias, while the residual gets it as it is. Each term of such a sum is off by
up to 2^-9 of itself in bf16, independently of the others. Parameters in fp32 get fp32 sums.
"""
from __future__ import annotations

import functools
from typing import Optional

import torch
from torch import Tensor, nn
from torch.amp import custom_bwd, custom_fwd
from torch.autograd import forward_ad
from torch.autograd import Function

from .. import dropout_lib, linear_lib, ln_lib  # noqa: F401  (registers torch.ops.act_lib.*)
from .ops import _compute_dtype

_U63 = (1 << 63) - 1


def _differentiated(*tensors: Optional[Tensor]) -> bool:
    """Whether a call on these goes through its autograd Function: one that does not would lose the tangents of forward mode, which
    ask for no gradient (the Functions refuse them, and functorch's transforms). Inside a level of dual numbers every call does: asking
    each tensor would be half of what a call on one token takes here."""
    if forward_ad._current_level >= 0 or torch._C._are_functorch_transforms_active():
        return True
    if not torch.is_grad_enabled():
        return False
    for t in tensors:
        if t is not None and t.requires_grad:
            return True
    return False


def _first_order(backward):
    """For the backward of a Function: the operators that compute it have no derivatives, so a graph of it (create_graph) is refused, as
    is a tangent that comes in. Not an error that waits until the results are differentiated, as torch's once_differentiable: a
    search for some tensors' gradients would pass that by, and add nothing."""
    @functools.wraps(backward)
    def guarded(ctx, *grads):
        if forward_ad._current_level >= 0 and any(g is not None and forward_ad.unpack_dual(g).tangent is not None for g in grads):
            raise NotImplementedError("the transformer layers' gradients have no forward-mode derivatives")
        if not torch.is_grad_enabled():
            return backward(ctx, *grads)
        with torch.no_grad():
            out = backward(ctx, *grads)
        if any(g is not None and not any(g is d for d in grads) for g in out):  # (an incoming one that is handed on has its own graph)
            raise RuntimeError("the transformer layers' gradients cannot be differentiated again (create_graph=True)")
        return out

    return guarded


def _to(t: Optional[Tensor], dtype: torch.dtype) -> Optional[Tensor]:
    return None if t is None else t.to(dtype)


def _product_operands(x: Tensor, *weights: Tensor):
    """x and weights in the products' type: the autocast dtype, else x's."""
    dt = _compute_dtype() or x.dtype
    return (x.to(dt), *(w.to(dt) for w in weights))


def _grad_dtype(operand: Tensor, *params) -> torch.dtype:
    """What a product's parameter gradients come in, of (parameter's type, whether it needs one): the operands' type where
    all that need one have it, else fp32, so that none is rounded to fewer bits than its parameter has."""
    return operand.dtype if all(dtype == operand.dtype for dtype, need in params if need) else torch.float32


class _LayerNorm(Function):
    @staticmethod
    @custom_fwd(device_type="cuda")
    def forward(ctx, x, weight, bias, eps, residual):
        y, mean, rstd = torch.ops.act_lib.layer_norm_fwd(x, weight, bias, eps, _compute_dtype() or x.dtype)
        ctx.save_for_backward(x, mean, rstd, weight)
        ctx.bias_dtype = None if bias is None else bias.dtype
        ctx.set_materialize_grads(False)
        return (y, x.view_as(x)) if residual else y

    @staticmethod
    @custom_bwd(device_type="cuda")
    @_first_order
    def backward(ctx, dy, dresidual=None):
        x, mean, rstd, weight = ctx.saved_tensors
        _, need_w, need_b, _, _ = ctx.needs_input_grad
        if dy is None:
            return dresidual, None, None, None, None
        dx, dw, db = torch.ops.act_lib.layer_norm_bwd(dy, x, mean, rstd, weight, dresidual, need_w, need_b)
        return dx, _to(dw, weight.dtype) if need_w else None, _to(db, ctx.bias_dtype) if need_b else None, None, None


def layer_norm(x: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None, eps: float = 1e-5) -> Tensor:
    return _LayerNorm.apply(x, weight, bias, eps, False)


def layer_norm_residual(x: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None, eps: float = 1e-5):
    return _LayerNorm.apply(x, weight, bias, eps, True)


class _LinearAct(Function):
    @staticmethod
    @custom_fwd(device_type="cuda")
    def forward(ctx, x, weight, bias, residual, act):
        xc, wc = _product_operands(x, weight)
        y, pre = torch.ops.act_lib.linear_act_fwd(xc, wc, bias, residual, act, act != "none")
        ctx.save_for_backward(xc, wc, pre)
        ctx.act, ctx.x_dtype, ctx.param = act, x.dtype, (weight.dtype, None if bias is None else bias.dtype)
        return y

    @staticmethod
    @custom_bwd(device_type="cuda")
    @_first_order
    def backward(ctx, dy):
        x, weight, pre = ctx.saved_tensors
        need_x, need_w, need_b, need_r, _ = ctx.needs_input_grad
        dx, dw, db = torch.ops.act_lib.linear_act_bwd(dy.to(x.dtype), x, weight, pre, ctx.act, None, "none", need_x, need_w, need_b,
                                                      _grad_dtype(x, (ctx.param[0], need_w), (ctx.param[1], need_b)))
        return (_to(dx, ctx.x_dtype), _to(dw, ctx.param[0]), _to(db, ctx.param[1]) if need_b else None, dy if need_r else None, None)


def linear_act(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, residual: Optional[Tensor] = None, act: str = "none") -> Tensor:
    if not _differentiated(x, weight, bias, residual):
        xc, wc = _product_operands(x, weight)
        return torch.ops.act_lib.linear_act_fwd(xc, wc, bias, residual, act, False)[0]
    return _LinearAct.apply(x, weight, bias, residual, act)


class _Mlp(Function):
    @staticmethod
    @custom_fwd(device_type="cuda")
    def forward(ctx, x, w1, b1, w2, b2, residual, act):
        xc, w1c, w2c = _product_operands(x, w1, w2)
        h, pre = torch.ops.act_lib.linear_act_fwd(xc, w1c, b1, None, act, act != "none")
        y, _ = torch.ops.act_lib.linear_act_fwd(h, w2c, b2, residual, "none", False)
        ctx.save_for_backward(xc, w1c, w2c, h, pre)
        ctx.act, ctx.x_dtype = act, x.dtype
        ctx.param = tuple(None if t is None else t.dtype for t in (w1, b1, w2, b2))
        return y

    @staticmethod
    @custom_bwd(device_type="cuda")
    @_first_order
    def backward(ctx, dy):
        x, w1, w2, h, pre = ctx.saved_tensors
        need_x, need_w1, need_b1, need_w2, need_b2, need_r, _ = ctx.needs_input_grad
        t1, u1, t2, u2 = ctx.param
        first = need_x or need_w1 or need_b1
        dz, dw2, db2 = torch.ops.act_lib.linear_act_bwd(dy.to(x.dtype), h, w2, None, "none", pre, ctx.act, first, need_w2, need_b2,
                                                        _grad_dtype(x, (t2, need_w2), (u2, need_b2)))
        dx = dw1 = db1 = None
        if first:
            dx, dw1, db1 = torch.ops.act_lib.linear_act_bwd(dz, x, w1, None, "none", None, "none", need_x, need_w1, need_b1,
                                                            _grad_dtype(x, (t1, need_w1), (u1, need_b1)))
        return (_to(dx, ctx.x_dtype), _to(dw1, t1), _to(db1, u1) if need_b1 else None, _to(dw2, t2), _to(db2, u2) if need_b2 else None,
                dy if need_r else None, None)


def mlp(x: Tensor, w1: Tensor, b1: Optional[Tensor], w2: Tensor, b2: Optional[Tensor], residual: Optional[Tensor] = None,
        act: str = "gelu") -> Tensor:
    if not _differentiated(x, w1, b1, w2, b2, residual):
        xc, w1c, w2c = _product_operands(x, w1, w2)
        h = torch.ops.act_lib.linear_act_fwd(xc, w1c, b1, None, act, False)[0]
        return torch.ops.act_lib.linear_act_fwd(h, w2c, b2, residual, "none", False)[0]
    return _Mlp.apply(x, w1, b1, w2, b2, residual, act)


class _DropoutAdd(Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, offset, step):
        ctx.save_for_backward(step)
        ctx.args, ctx.x_dtype = (p, seed, offset), x.dtype
        return torch.ops.act_lib.dropout_add_fwd(x, residual, p, seed, offset, step)

    @staticmethod
    @_first_order
    def backward(ctx, dy):
        (step,) = ctx.saved_tensors
        need_x, need_r = ctx.needs_input_grad[:2]
        dx = torch.ops.act_lib.dropout_bwd(dy, *ctx.args, step, ctx.x_dtype) if need_x else None
        return dx, dy if need_r else None, None, None, None, None


def dropout_add(x: Tensor, residual: Optional[Tensor], p: float, seed: int, offset: int = 0, step: Optional[Tensor] = None) -> Tensor:
    return _DropoutAdd.apply(x, residual, p, seed, offset, step)


def _bare(m: nn.Module, cls: type) -> bool:
    """Whether calling m does what cls.forward does and nothing else, so that a fused call may read its parameters instead: a layer that
    was replaced, has a forward of its own or hooks (pruning sets the weight in one) is called."""
    if not isinstance(m, cls) or type(m).forward is not cls.forward:
        return False
    d = m.__dict__
    return not ("forward" in d or d["_forward_hooks"] or d["_forward_pre_hooks"] or d["_backward_hooks"] or d["_backward_pre_hooks"]
                or nn.modules.module._has_any_global_hook())


def norm_residual(norm: nn.Module, x: Tensor):
    """(norm(x), x) for x + f(norm(x)): by layer_norm_residual where norm is a LayerNorm of this module."""
    if _bare(norm, LayerNorm):
        return layer_norm_residual(x, norm.weight, norm.bias, norm.eps)
    return norm(x), x


class LayerNorm(nn.LayerNorm):
    """torch.nn.LayerNorm over the last axis. ``residual(x)`` is (norm(x), x) for x + f(norm(x))."""

    def __init__(self, dim: int, eps: float = 1e-5, **kw):
        super().__init__(dim, eps, **kw)
        if len(self.normalized_shape) != 1:
            raise ValueError(f"LayerNorm normalizes the last axis only, got {self.normalized_shape}")

    def forward(self, x):
        return layer_norm(x, self.weight, self.bias, self.eps)

    def residual(self, x):
        return norm_residual(self, x)


class LinearAct(nn.Module):
    """act(x weight^T + bias) + residual with torch.nn.Linear's parameters and initialisation."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True, act: str = "none", device=None, dtype=None):
        super().__init__()
        linear_lib._act_code(act)
        plain = nn.Linear(in_features, out_features, bias, device=device, dtype=dtype)
        self.in_features, self.out_features, self.act = in_features, out_features, act
        self.weight, self.bias = plain.weight, plain.bias

    def forward(self, x, residual=None):
        return linear_act(x, self.weight, self.bias, residual, self.act)

    def extra_repr(self):
        return f"{self.in_features}, {self.out_features}, bias={self.bias is not None}, act={self.act!r}"


class DropoutRng(nn.Module):
    """The masks of a model's dropout layers: a seed, and a count of passes that lies on the device, so that a captured
    step draws new masks on every replay. Call it once at the start of a pass, on the input: it returns that and steps the
    count. Every layer has an offset of its own (``site``). ``step`` is part of the state dict; the seed is not: ranks that
    train on different data each give their own (default: from torch's initial seed). One process per GPU: the layers refuse to run
    in nn.DataParallel's replicas. The layers take the count of the latest call: call it outside of what activation checkpointing
    recomputes, and recompute a pass before the next one begins."""

    def __init__(self, seed: Optional[int] = None):
        super().__init__()
        # (not the quantizer's default key: both use the same generator)
        self.seed = (torch.initial_seed() ^ 0x64726F70 if seed is None else seed) & _U63
        self.register_buffer("step", torch.zeros(1, dtype=torch.int64))
        self.current = None
        self.sites = 0

    def site(self) -> int:
        self.sites += 1
        return (self.sites - 1) << 40

    def forward(self, x):
        if self.training:
            # (a tensor of its own, which the pass's backward reads whatever passes follow)
            self.current = self.step + 1
            self.step.copy_(self.current)
        return x


class DropoutAdd(nn.Module):
    """residual + dropout(x), in residual's type (x's without one)."""

    def __init__(self, p: float, rng: DropoutRng):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"p must lie in [0, 1], got {p}")
        self.p, self.offset = float(p), rng.site()
        self._rng = (rng,)  # (not a submodule of every layer)

    def forward(self, x, residual=None):
        if not self.training or self.p == 0.0:
            return x if residual is None else residual + x.to(residual.dtype)
        rng = self._rng[0]
        if getattr(self, "_is_replica", False):
            raise RuntimeError("DropoutAdd does not run in nn.DataParallel replicas, whose DropoutRng it would not see: use one process per GPU")
        if rng.current is None:
            raise RuntimeError("DropoutAdd: call the model's DropoutRng at the start of the pass")
        return dropout_add(x, residual, self.p, rng.seed, self.offset, rng.current)

    def extra_repr(self):
        return f"p={self.p}"


class Mlp(nn.Module):
    """fc2(act(fc1(x))) + residual; with a dropout rate after the activation and after fc2."""

    def __init__(self, dim: int, hidden: int, act: str = "gelu", drop: float = 0.0, rng: Optional[DropoutRng] = None):
        super().__init__()
        self.fc1 = LinearAct(dim, hidden, act=act)
        self.fc2 = LinearAct(hidden, dim)
        if drop:
            if rng is None:
                raise ValueError("Mlp: a dropout rate needs a DropoutRng")
            self.drop1, self.drop2 = DropoutAdd(drop, rng), DropoutAdd(drop, rng)
        else:
            self.drop1 = self.drop2 = None

    def forward(self, x, residual=None):
        if self.drop1 is not None and self.training:
            return self.drop2(self.fc2(self.drop1(self.fc1(x))), residual)
        if not (_bare(self.fc1, LinearAct) and _bare(self.fc2, LinearAct) and self.fc2.act == "none"):
            return self.fc2(self.fc1(x), residual)
        return mlp(x, self.fc1.weight, self.fc1.bias, self.fc2.weight, self.fc2.bias, residual, self.fc1.act)


__all__ = ["layer_norm", "layer_norm_residual", "linear_act", "mlp", "dropout_add", "norm_residual", "LayerNorm", "LinearAct", "DropoutRng",
           "DropoutAdd", "Mlp"]
