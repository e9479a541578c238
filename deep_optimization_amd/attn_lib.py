"""Attention operators: ``torch.ops.act_lib.attention_fwd`` / ``attention_bwd`` / ``attention_qkv_bwd`` on the gfx950 MFMA kernels behind
dopt_attention_forward and dopt_attention_backward. No counterparts in the reference, whose Transformer models call torch's attention.

    attention_fwd(q, k, v, lengths, scale, causal, save_lse) -> (out, lse)
    attention_bwd(dout, q, k, v, out, lse, lengths, scale, causal) -> (dq, dk, dv)
    attention_qkv_bwd(dout, qkv, heads, out, lse, lengths, scale, causal) -> dqkv

q [B, Lq, H, D], k and v [B, Lk, G, D] in bf16 or fp16, D a multiple of 8 up to 128; H is a multiple of G, and query head h reads key
head h / (H / G). Query i of sequence b sees key j where j < lengths[b] (int32 or int64 [B]; all keys without it; values outside 0..Lk count
as those ends) and, with ``causal``, j <= i + Lk - Lq: the last query sees every key, as new tokens at the end of a cache do.

    s = scale q k^T (scale from 2^-100 to 2^100),  out = softmax(s) v,  lse = log sum exp s   (a query that sees no key: out 0, lse -inf)

out [B, Lq, H, D] contiguous in q's type, lse fp32 [B, H, Lq] (None unless save_lse). Scores, softmax and sums are fp32; the
probabilities, and in the backward pass ds, are rounded to q's type for the products that read them on matrix instructions (in fp16 times powers of two that
keep them in its range, whatever the size of dout); delta is of out as it
was returned, rounded to q's type (felt where a query sees a few keys only: 0.0039 of dq's norm at two keys in bf16, 0.0024 at many). What lies in k and v
past a sequence's length is never used (NaN and infinities included) and has zero gradients. What ``causal`` hides is multiplied by probabilities of 0: a value
or key that is not finite makes NaN of earlier queries of its tile too, and a query's q or dout of later keys' gradients. attention_qkv_bwd is attention_bwd
for q, k and v that are the parts of one tensor qkv [B, L, H + 2 G, D], ``heads`` = H: its gradient in one tensor.

Any strides whose last one is 1; the kernels read where tokens lie at multiples of 16 bytes, at least D and less than 2^23 elements apart,
other layouts are copied. Sums have the order that the sizes give them: the same inputs give the same bits.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch
from torch import Tensor

from . import _lib
from .act_lib import _DTYPE_CODE, _op, _require_cuda, _stream

_TYPES = (torch.bfloat16, torch.float16)


def _check(what: str, q: Tensor, k: Tensor, v: Tensor, lengths: Optional[Tensor], scale: float) -> None:
    if q.dtype not in _TYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise RuntimeError(f"{what}: q, k and v must all be bfloat16 or float16, got {q.dtype}, {k.dtype} and {v.dtype}")
    if (q.dim() != 4 or k.dim() != 4 or v.shape != k.shape or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3]
            or (q.shape[2] == 0 or q.shape[2] % k.shape[2] if k.shape[2] else q.shape[2])):
        raise RuntimeError(f"{what}: q [B, Lq, H, D] and k, v [B, Lk, G, D] with H a multiple of G (0 only with 0), got {tuple(q.shape)}, {tuple(k.shape)} and "
                           f"{tuple(v.shape)}")
    if not 0 < q.shape[3] <= 128 or q.shape[3] % 8:
        raise RuntimeError(f"{what}: a head must have a multiple of 8 elements, 8 to 128, got {q.shape[3]}")
    if lengths is not None and (lengths.dtype not in (torch.int32, torch.int64) or lengths.shape != q.shape[:1]):
        raise RuntimeError(f"{what}: lengths must be int32 or int64 of shape [{q.shape[0]}], got {tuple(lengths.shape)} {lengths.dtype}")
    if not 2.0 ** -100 <= scale <= 2.0 ** 100:
        raise RuntimeError(f"{what}: scale must lie between 2^-100 and 2^100, got {scale}")


def _readable(t: Tensor) -> Tensor:
    """t, or a copy in a layout that the kernels read."""
    ok = t.data_ptr() % 16 == 0 and t.stride(3) == 1
    for d in (0, 1, 2):
        ok = ok and (t.shape[d] <= 1 or (t.stride(d) >= 0 and t.stride(d) % 8 == 0))
    if ok and (t.shape[1] <= 1 or t.shape[3] <= t.stride(1) < 1 << 23):
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _lengths(lengths: Optional[Tensor], Lk: int) -> Optional[Tensor]:
    if lengths is not None and lengths.dtype != torch.int32:
        lengths = lengths.clamp(0, Lk).to(torch.int32)
    return None if lengths is None else lengths.contiguous()


def _view(t: Tensor) -> _lib.AttentionTensor:
    return _lib.AttentionTensor(t.data_ptr(), t.stride(0), t.stride(1), t.stride(2))


def _call(q: Tensor, k: Tensor, v: Tensor, out: Tensor, lse: Optional[Tensor], lengths: Optional[Tensor], scale: float, causal: bool) -> _lib.Attention:
    B, Lq, H, D = q.shape
    a = _lib.Attention(batch=B, heads=H, kv_heads=k.shape[2], q_len=Lq, k_len=k.shape[1], dim=D, scale=scale, causal=int(causal),
                       dtype=_DTYPE_CODE[q.dtype])
    a.q, a.k, a.v, a.out = _view(q), _view(k), _view(v), _view(out)
    a.lse = None if lse is None else lse.data_ptr()
    a.lengths = None if lengths is None else lengths.data_ptr()
    return a


def _attention_fwd(q: Tensor, k: Tensor, v: Tensor, lengths: Optional[Tensor], scale: float, causal: bool, save_lse: bool):
    what = "attention_fwd"
    _check(what, q, k, v, lengths, scale)
    _require_cuda(q, k, v, lengths)
    stream = _stream(q)
    q, k, v, lengths = _readable(q), _readable(k), _readable(v), _lengths(lengths, k.shape[1])
    B, Lq, H, D = q.shape
    out = torch.empty((B, Lq, H, D), dtype=q.dtype, device=q.device)
    lse = torch.empty((B, H, Lq), dtype=torch.float32, device=q.device) if save_lse else None
    a = _call(q, k, v, out, lse, lengths, scale, causal)
    L = _lib.lib()
    floats = int(L.dopt_attention_workspace_floats(ctypes.byref(a)))
    ws = torch.empty(floats, dtype=torch.float32, device=q.device) if floats else None
    a.workspace = None if ws is None else ws.data_ptr()
    _lib.check(L.dopt_attention_forward(ctypes.byref(a), stream), what)
    return out, lse


def _attention_fwd_fake(q, k, v, lengths, scale, causal, save_lse):
    B, Lq, H, D = q.shape
    return q.new_empty((B, Lq, H, D)), (q.new_empty((B, H, Lq), dtype=torch.float32) if save_lse else None)


attention_fwd = _op(
    "attention_fwd(Tensor q, Tensor k, Tensor v, Tensor? lengths, float scale, bool causal, bool save_lse) -> (Tensor, Tensor?)",
    _attention_fwd, _attention_fwd_fake)


def _backward(what: str, dout: Tensor, q: Tensor, k: Tensor, v: Tensor, out: Tensor, lse: Tensor, lengths: Optional[Tensor], scale: float, causal: bool,
              dq: Tensor, dk: Tensor, dv: Tensor) -> None:
    B, Lq, H, D = q.shape
    for name, t in (("dout", dout), ("out", out)):
        if t.shape != q.shape or t.dtype != q.dtype:
            raise RuntimeError(f"{what}: {name} must have q's shape {tuple(q.shape)} and type, got {tuple(t.shape)} {t.dtype}")
    if lse.shape != (B, H, Lq) or lse.dtype != torch.float32:
        raise RuntimeError(f"{what}: lse must be float32 of shape {(B, H, Lq)}, got {tuple(lse.shape)} {lse.dtype}")
    _require_cuda(dout, q, k, v, out, lse, lengths)
    stream = _stream(q)
    q, k, v, out, dout, lse = _readable(q), _readable(k), _readable(v), _readable(out), _readable(dout), lse.contiguous()
    lengths = _lengths(lengths, k.shape[1])
    a = _call(q, k, v, out, lse, lengths, scale, causal)
    a.dout, a.dq, a.dk, a.dv = _view(dout), _view(dq), _view(dk), _view(dv)
    L = _lib.lib()
    floats = int(L.dopt_attention_backward_workspace_floats(ctypes.byref(a)))
    ws = torch.empty(floats, dtype=torch.float32, device=q.device) if floats else None
    a.workspace = None if ws is None else ws.data_ptr()
    _lib.check(L.dopt_attention_backward(ctypes.byref(a), stream), what)


def _attention_bwd(dout: Tensor, q: Tensor, k: Tensor, v: Tensor, out: Tensor, lse: Tensor, lengths: Optional[Tensor], scale: float, causal: bool):
    what = "attention_bwd"
    _check(what, q, k, v, lengths, scale)
    dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
    _backward(what, dout, q, k, v, out, lse, lengths, scale, causal, dq, dk, dv)
    return dq, dk, dv


attention_bwd = _op(
    "attention_bwd(Tensor dout, Tensor q, Tensor k, Tensor v, Tensor out, Tensor lse, Tensor? lengths, float scale, bool causal) "
    "-> (Tensor, Tensor, Tensor)", _attention_bwd,
    lambda dout, q, k, v, out, lse, lengths, scale, causal: (q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape)))


def _split_qkv(what: str, qkv: Tensor, heads: int):
    if qkv.dim() != 4 or not 0 <= heads <= qkv.shape[2] or (qkv.shape[2] - heads) % 2:
        raise RuntimeError(f"{what}: qkv must be [B, L, H + 2 G, D] with H = {heads}, got {tuple(qkv.shape)}")
    kv = (qkv.shape[2] - heads) // 2
    return qkv.split((heads, kv, kv), dim=2)


def _attention_qkv_bwd(dout: Tensor, qkv: Tensor, heads: int, out: Tensor, lse: Tensor, lengths: Optional[Tensor], scale: float, causal: bool):
    what = "attention_qkv_bwd"
    q, k, v = _split_qkv(what, qkv, heads)
    _check(what, q, k, v, lengths, scale)
    dqkv = torch.empty(qkv.shape, dtype=qkv.dtype, device=qkv.device)
    _backward(what, dout, q, k, v, out, lse, lengths, scale, causal, *_split_qkv(what, dqkv, heads))
    return dqkv


attention_qkv_bwd = _op(
    "attention_qkv_bwd(Tensor dout, Tensor qkv, int heads, Tensor out, Tensor lse, Tensor? lengths, float scale, bool causal) -> Tensor",
    _attention_qkv_bwd, lambda dout, qkv, heads, out, lse, lengths, scale, causal: qkv.new_empty(qkv.shape))

__all__ = ["attention_fwd", "attention_bwd", "attention_qkv_bwd"]
