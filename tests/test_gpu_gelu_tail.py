"""The exact GELU's negative side relative to itself, in 32 bits and as one rounding to 16: erf-based forms lose it below -4.

The kernels' Q(a) = 1 - Phi(a) is a fit within 1.9e-6 of Q, and its fp32 evaluation adds: rcp and exp2 of 1 ulp (1.2e-7 each), three
products and the polynomial's last sums (5e-7 together), the exponent a^2 / 2, whose three roundings move it by a^2 / 2 * 2.5 * 2^-24
(8e-8 a^2). gelu = -a Q for z < 0, act' = Q - a phi: within 3e-6 + 1e-7 z^2 of a Q and of Q + a phi. Down to z = -12.5, where e^(-z^2 / 2)
is a normal number."""
import math

import pytest
import torch

import deep_optimization_amd  # noqa: F401
from tests import block_reference as ref

pytestmark = pytest.mark.gpu
ops = torch.ops.act_lib
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _arguments(dt):
    return torch.cat([-torch.linspace(4, 12.5, 4000), -torch.linspace(0.01, 4, 4000)]).to(dt).unique().to("cuda")


def _rel(z):
    return 3e-6 + 1e-7 * z * z


@pytest.mark.parametrize("dt", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("rows", [1, 300], ids=["token", "rows"])  # (the kernel of few rows, and the tiles)
def test_values(dt, rows):
    """z = x: a weight of 1 and no bias; an fp32 residual of zeros for a result in 32 bits."""
    z = _arguments(dt)
    x = torch.ones((rows, 1), device="cuda", dtype=dt)
    w = z.view(-1, 1)
    want = ref.act(z.double(), "gelu").expand(rows, -1)
    tol = _rel(z.double()) * want.abs()
    y, _ = ops.linear_act_fwd(x, w, None, torch.zeros((rows, z.numel()), device="cuda"), "gelu", False)
    assert y.dtype == F32
    ref.close(y, want, tol, "fp32")
    y, _ = ops.linear_act_fwd(x, w, None, None, "gelu", False)
    ref.close(y, want, tol, "16 bits")


@pytest.mark.parametrize("dt", [BF16, F16], ids=["bf16", "f16"])
def test_derivatives(dt):
    """The bias gradient of one row of ones is act'(pre) in 32 bits; dx through the activation that feeds the layer, in 16."""
    z = _arguments(dt).view(1, -1)
    n = z.numel()
    one, x = torch.ones((1, n), device="cuda", dtype=dt), torch.zeros((1, 8), device="cuda", dtype=dt)
    zd = z.double()
    want = ref.act_grad(zd, "gelu")
    tol = _rel(zd) * (0.5 * torch.special.erfc(-zd * 2 ** -0.5) - zd * torch.exp(-zd * zd / 2) / math.sqrt(2 * math.pi))
    db = ops.linear_act_bwd(one, x, torch.zeros((n, 8), device="cuda", dtype=dt), z, "gelu", None, "none", False, False, True, F32)[2]
    ref.close(db, want[0], tol[0], "fp32")
    for rows in (1, 300):
        dx = ops.linear_act_bwd(torch.ones((rows, 1), device="cuda", dtype=dt), z.expand(rows, n), one, None, "none", z.expand(rows, n).contiguous(), "gelu",
                                True, False, False, dt)[0]
        ref.close(dx, want.expand(rows, n), tol.expand(rows, n), "16 bits")
