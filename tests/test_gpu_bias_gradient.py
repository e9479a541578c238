"""linear_act_bwd where the weight's gradient is not asked for: the bias gradient is a sum of columns alone."""
import ctypes

import pytest
import torch

import deep_optimization_amd  # noqa: F401
from deep_optimization_amd import _lib, linear_lib
from tests import block_reference as ref
from tests.test_gpu_linear_act import check_bwd

DEV = "cuda"
ops = torch.ops.act_lib
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
gpu = pytest.mark.gpu


def _rand(seed, shape, dtype=BF16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(shape, generator=g, device=DEV).to(dtype)


@gpu
@pytest.mark.parametrize("dt", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("M,N", [(0, 40), (1, 8), (3, 13), (512, 2048), (513, 1001), (20000, 40), (5000, 2311)])
def test_sums_alone(M, N, dt):
    """Within the fp32 sums' bound, whole rows or rows as they lie in a larger tensor, with the input's gradient or without; the
    operand stays as it is."""
    for grad in (F32, dt):
        for act in ("none", "silu"):
            check_bwd(M, 24, N, dt, act, grad=grad, parts=(False, False, True))
            check_bwd(M, 24, N, dt, act, "gelu", grad=grad, parts=(True, False, True))
    wide, x, w = _rand(M + N, (M, N + 5), dt), _rand(1, (M, 24), dt), _rand(2, (N, 24), dt)
    before = wide.clone()
    for dy in (wide[:, 2:N + 2], wide[:, 5:]):
        for parts in ((False, False, True), (True, False, True)):
            db = ops.linear_act_bwd(dy, x, w, None, "none", None, "none", *parts, F32)[2]
            ref.close(db, dy.double().sum(0), (M + 8) * ref.E * dy.double().abs().sum(0), "dbias")
            assert torch.equal(db, linear_lib._linear_act_bwd(dy, x, w, None, "none", None, "none", *parts, F32)[2])
    assert torch.equal(wide, before)


@gpu
@pytest.mark.parametrize("call", [ops.linear_act_bwd, linear_lib._linear_act_bwd], ids=["native", "python"])
def test_no_weight_gradient_is_computed(call):
    """Its 128 MB (and, with an activation, a dz that nothing reads) are not allocated."""
    M, N, K = 600, 8192, 8192
    dy, x, w = _rand(0, (M, N)), _rand(1, (M, K)), _rand(2, (N, K))
    for act, pre in (("none", None), ("gelu", dy)):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        dx, dw, db = call(dy, x, w, pre, act, None, "none", False, False, True, F32)
        assert dx is None and dw is None and db.shape == (N,)
        assert torch.cuda.max_memory_allocated() - before < 2 * M * N


def test_layout_takes_sums_alone():
    """The C entry: no dst goes with ld_dst 0 and a sum only."""
    buf = ctypes.create_string_buffer(4096)
    at = (ctypes.addressof(buf) + 255) // 256 * 256

    def lay(**k):
        r = _lib.LinearRows(*{**dict(src=at, ld=8, pre=None, rows=2, cols=8, dst=None, ldd=0, act=0, sdt=_lib.BF16, sum=at, ws=None), **k}.values())
        return _lib.lib().dopt_linear_layout(ctypes.byref(r), 1, _lib.BF16, None)

    for k in (dict(sum=None), dict(ldd=8), dict(dst=at), dict(src=None), dict(ld=7), dict(act=2), dict(rows=5000)):
        assert lay(**k) == _lib.EINVAL, k
