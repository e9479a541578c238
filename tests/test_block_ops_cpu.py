"""The layer norm, dropout and linear operators without a GPU: fake kernels, refusals of the C entries that come before any
launch, and the fused ViT's names and trace."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import deep_optimization_amd  # noqa: F401
from deep_optimization_amd import _lib
from deep_optimization_amd.controller import Controller
from deep_optimization_amd.modules import transformer
from deep_optimization_amd.vit import VisionTransformer

ops = torch.ops.act_lib
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def test_fake_shapes():
    with FakeTensorMode():
        x = torch.empty((2, 5, 24), dtype=BF16, device="cuda")
        w = torch.empty((40, 24), dtype=BF16, device="cuda")
        y, mean, rstd = ops.layer_norm_fwd(x, None, None, 1e-5, F32)
        assert y.shape == x.shape and y.dtype == F32 and mean.shape == rstd.shape == (2, 5) and mean.dtype == F32
        dx, dw, db = ops.layer_norm_bwd(y, x, mean, rstd, None, x, True, False)
        assert dx.shape == x.shape and dx.dtype == BF16 and dw.shape == (24,) and dw.dtype == F32 and db is None
        assert ops.dropout_add_fwd(x, y, 0.1, 0, 0, None).dtype == F32 and ops.dropout_add_fwd(x, None, 0.1, 0, 0, None).dtype == BF16
        assert ops.dropout_bwd(y, 0.1, 0, 0, None, F16).dtype == F16
        r = torch.empty((2, 5, 40), dtype=F32, device="cuda")
        y, pre = ops.linear_act_fwd(x, w, None, r, "gelu", True)
        assert y.shape == pre.shape == (2, 5, 40) and y.dtype == F32 and pre.dtype == BF16
        assert ops.linear_act_fwd(x, w, None, None, "gelu", False)[1] is None
        dx, dw, db = ops.linear_act_bwd(pre, x, w, pre, "gelu", None, "none", True, True, True, F32)
        assert dx.shape == x.shape and dx.dtype == BF16 and dw.shape == (40, 24) and dw.dtype == F32 and db.shape == (40,)
        assert ops.linear_act_bwd(pre, x, w, None, "none", None, "none", False, True, False, BF16)[0::2] == (None, None)


def test_cpu_tensors_are_refused():
    x, w = torch.zeros((2, 8), dtype=BF16), torch.zeros((8, 8), dtype=BF16)
    for call in (lambda: ops.layer_norm_fwd(x, None, None, 1e-5, F32), lambda: ops.dropout_add_fwd(x, None, 0.1, 0, 0, None),
                 lambda: ops.linear_act_fwd(x, w, None, None, "none", False)):
        with pytest.raises(NotImplementedError):
            call()


BUF = ctypes.create_string_buffer(4096)
AT = (ctypes.addressof(BUF) + 255) // 256 * 256  # an address that no refused call reads
ODD = AT + 1


def _refused(rc):
    assert rc in (_lib.EINVAL, _lib.EUNSUPPORTED) and _lib.lib().dopt_last_error()


def test_c_entries_refuse_before_any_launch():
    L = _lib.lib()
    BF, FP, I8 = _lib.BF16, _lib.F32, 99
    ln = lambda **k: L.dopt_layer_norm_forward(*{**dict(x=AT, xd=BF, rows=2, dim=8, w=None, b=None, pd=FP, eps=1e-5, y=AT, yd=BF, mean=AT, rstd=AT, s=None), **k}.values())  # noqa: E731
    for k in (dict(x=None), dict(xd=I8), dict(rows=-1), dict(dim=0), dict(y=None), dict(yd=I8), dict(mean=None), dict(rstd=None), dict(w=AT, pd=I8)):
        _refused(ln(**k))
    lb = lambda **k: L.dopt_layer_norm_backward(*{**dict(dy=AT, dyd=BF, x=AT, xd=BF, rows=2, dim=8, mean=AT, rstd=AT, w=None, pd=FP, res=None, dx=AT, ws=AT, dw=AT, db=AT, s=None), **k}.values())  # noqa: E731
    for k in (dict(dy=None), dict(dyd=I8), dict(x=None), dict(rows=-1), dict(dim=0), dict(mean=None), dict(dx=None), dict(rows=5000, ws=None)):
        _refused(lb(**k))
    dr = lambda **k: L.dopt_dropout(*{**dict(x=AT, xd=BF, res=None, n=8, p=0.5, seed=0, off=0, step=None, y=AT, yd=BF, s=None), **k}.values())  # noqa: E731
    for k in (dict(x=None), dict(xd=I8), dict(n=-1), dict(p=-0.1), dict(p=1.5), dict(p=float("nan")), dict(y=None), dict(yd=I8)):
        _refused(dr(**k))
    fw = lambda **k: L.dopt_linear_forward(*{**dict(x=AT, ldx=8, w=AT, ldw=8, dt=BF, M=2, N=4, K=8, b=None, bd=FP, res=None, act=0, y=AT, yd=BF, pre=None, s=None), **k}.values())  # noqa: E731
    for k in (dict(x=None), dict(w=None), dict(x=ODD), dict(ldx=7), dict(ldw=7), dict(dt=FP), dict(M=-1), dict(N=-1), dict(K=-1), dict(act=5), dict(act=-1),
              dict(y=None), dict(yd=I8), dict(b=AT, bd=I8), dict(ldx=1 << 21), dict(K=1 << 28, ldx=1 << 28, ldw=1 << 28)):
        _refused(fw(**k))
    dg = lambda **k: L.dopt_linear_input_grad(*{**dict(dz=AT, ldz=8, w=AT, ldw=8, dt=BF, M=2, N=8, K=8, ip=None, act=0, dx=AT, s=None), **k}.values())  # noqa: E731
    for k in (dict(dz=None), dict(w=None), dict(ldz=7), dict(ldw=7), dict(dt=FP), dict(M=-1), dict(act=2), dict(act=9), dict(dx=None)):
        _refused(dg(**k))
    wg = lambda **k: L.dopt_linear_weight_grad(*{**dict(dz=AT, ldz=8, x=AT, ldx=8, dt=BF, M=2, N=8, K=8, ws=AT, dw=AT, dw16=None, db=None, db16=None, s=None), **k}.values())  # noqa: E731
    for k in (dict(dz=None), dict(x=None), dict(ldz=7), dict(ldx=7), dict(dt=FP), dict(M=-1), dict(N=0), dict(dw=None), dict(dw16=AT), dict(db=AT, db16=AT)):
        _refused(wg(**k))
    def lay(n=1, dt=BF, **k):
        r = _lib.LinearRows(*{**dict(src=AT, ld=8, pre=AT, rows=2, cols=8, dst=AT, ldd=8, act=2, sdt=BF, sum=AT, ws=AT), **k}.values())
        return L.dopt_linear_layout(ctypes.byref(r), n, dt, None)

    for k in (dict(src=None), dict(dst=None), dict(pre=None), dict(ld=7), dict(ldd=7), dict(act=7), dict(act=-1), dict(dt=FP),
              dict(rows=-1), dict(cols=-1), dict(n=5), dict(n=-1), dict(src=ODD), dict(pre=ODD), dict(dst=ODD),
              dict(rows=1 << 40, ld=32, ldd=32), dict(rows=5000, ws=None), dict(sdt=I8), dict(sdt=_lib.F16), dict(cols=1 << 26, ld=1 << 26, ldd=1 << 26)):
        _refused(lay(**k))
    _refused(L.dopt_linear_layout(None, 1, BF, None))
    assert lay(n=0) == 0 and lay(rows=0, src=None, dst=None, sum=None) == 0
    # nothing to do is no error
    assert ln(rows=0, x=None, y=None, mean=None, rstd=None) == 0 and dr(n=0, x=None, y=None) == 0 and fw(M=0, y=None) == 0 and dg(M=0, dx=None) == 0


def test_fused_vit_names_and_initialisation():
    kw = dict(img_size=32, patch_size=8, num_classes=7, embed_dim=64, depth=2, num_heads=2)
    torch.manual_seed(0)
    plain = VisionTransformer(**kw)
    torch.manual_seed(0)
    fused = VisionTransformer(**kw, fused=True)
    a, b = plain.state_dict(), fused.state_dict()
    assert list(a) == list(b) and all(torch.equal(a[n], b[n]) for n in a)
    dropped = VisionTransformer(**kw, fused=True, drop_rate=0.1)
    assert set(dropped.state_dict()) - set(a) == {"dropout_rng.step"}
    sites = [m.offset for m in dropped.modules() if isinstance(m, transformer.DropoutAdd)]
    assert len(sites) == 1 + 3 * 2 and len(set(sites)) == len(sites)


def test_controller_traces_the_fused_vit():
    model = VisionTransformer(img_size=32, patch_size=8, num_classes=7, embed_dim=64, depth=1, num_heads=2, fused=True, drop_rate=0.1)
    c = Controller(model, {"batch_size": 2, "default_bits": 2}, input_shape=(3, 32, 32), device="cpu")
    from deep_optimization_amd.controller import _Tracer

    nodes = [n.target for n in _Tracer.make()[0].trace(c.model).nodes]
    assert {"dropout_rng", "drop", "blocks.0", "norm", "head"} <= set(nodes)
