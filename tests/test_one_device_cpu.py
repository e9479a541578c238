"""Tensors of two GPUs in one call are refused before anything reads them: fake tensors through the Python implementations (which
the native operators follow), and the native operators where two GPUs are there."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import deep_optimization_amd  # noqa: F401
from deep_optimization_amd import act_lib, dropout_lib, dw_lib, linear_lib, ln_lib

F32, BF16 = torch.float32, torch.bfloat16


def _calls(make):
    """(name, implementation, arguments, which of them lies elsewhere); make(shape, dtype, elsewhere)."""
    t = lambda *shape, dt=BF16: (shape, dt)  # noqa: E731
    x, w, dy, v, rows, step = t(4, 8), t(6, 8), t(4, 6), t(8), t(4, dt=F32), t(1, dt=torch.int64)
    table = [("layer_norm_fwd", ln_lib._layer_norm_fwd, (x, v, v, 1e-5, BF16), (1, 2)),
             ("layer_norm_bwd", ln_lib._layer_norm_bwd, (x, x, rows, rows, v, x, True, True), (0, 2, 3, 4, 5)),
             ("dropout_add_fwd", dropout_lib._dropout_add_fwd, (x, x, 0.5, 0, 0, step), (1, 5)),
             ("dropout_bwd", dropout_lib._dropout_bwd, (x, 0.5, 0, 0, step, BF16), (4,)),
             ("linear_act_fwd", linear_lib._linear_act_fwd, (x, w, t(6), dy, "none", False), (1, 2, 3)),
             ("linear_act_bwd", linear_lib._linear_act_bwd, (dy, x, w, dy, "gelu", x, "gelu", True, True, True, F32), (0, 2, 3, 5)),
             ("dw_gemm_any", dw_lib._dw_gemm_any, (dy, x, False, F32), (1,)),
             ("fp8_gemm_nt", act_lib._fp8_gemm_nt, (t(32, 32, dt=torch.float8_e4m3fn), t(32, 32, dt=torch.float8_e4m3fn), 1.0), (1,))]
    for name, f, args, others in table:
        for k in others:
            yield name, f, [make(*a, i == k) if isinstance(a, tuple) else a for i, a in enumerate(args)]


def test_the_python_operators_refuse_tensors_of_two_devices(monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    with FakeTensorMode():
        calls = list(_calls(lambda shape, dt, elsewhere: torch.empty(shape, dtype=dt, device=f"cuda:{int(elsewhere)}")))
        assert len(calls) > 15
        for name, f, args in calls:
            with pytest.raises(RuntimeError, match="one device"):
                f(*args)


@pytest.mark.gpu
@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="two GPUs")
def test_the_native_operators_refuse_tensors_of_two_devices():
    for name, _, args in _calls(lambda shape, dt, elsewhere: torch.zeros(shape, device=f"cuda:{int(elsewhere)}").to(dt)):
        with pytest.raises(RuntimeError, match="one device"):
            getattr(torch.ops.act_lib, name)(*args)
