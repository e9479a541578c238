"""Attention in fp16 where probabilities, their gradients or the scores' lie far from 1: against the formulas in 64 bits
(tests/attention_reference.py), in the norm of the error, which sees what falls out of fp16's range.

Bounds: u = 2^-11. A gradient is a sum of terms that each carry one rounding of at most u of themselves, independently: their errors' norm is at
most u times the norm of the terms, which for random operands is the sum's own. The result's rounding to fp16 is computed, not bounded: for
small gradients it is one to subnormal numbers."""
import pytest
import torch

import deep_optimization_amd  # noqa: F401
from tests import attention_reference as ref
from tests.block_reference import close

pytestmark = pytest.mark.gpu
DEV = "cuda"
ops = torch.ops.act_lib
F16 = torch.float16
U16 = 2.0 ** -11


def _rand(gen, shape, scale=1.0):
    return (torch.randn(shape, generator=gen, device=DEV) * scale).to(F16)


def _gradients(q, k, v, dout, scale, causal, names=("dq", "dk", "dv")):
    """Each within its own rounding and one of its terms (half as much again for what delta feels of out's)."""
    out, lse = ops.attention_fwd(q, k, v, None, scale, causal, True)
    grads = ops.attention_bwd(dout, q, k, v, out, lse, None, scale, causal)
    torch.cuda.synchronize()
    o64, lse64 = ref.forward(q, k, v, None, scale, causal)[:2]
    want = ref.backward(dout, q, k, v, o64, lse64, None, scale, causal)[:3]
    for name, got, w in zip(("dq", "dk", "dv"), grads, want):
        if name in names:
            own, size, off = float((w.to(F16).double() - w).norm()), float(w.norm()), float((got.double() - w).norm())
            print(f"[attention f16] {name}: off by {off / size:.3g} of its norm, {own / size:.3g} its rounding", flush=True)
            assert off <= 1.05 * own + 1.5 * U16 * size, name


@pytest.mark.parametrize("size", [1e-5, 1e-4, 1e-3, 1.0, 1e3])
@pytest.mark.parametrize("B,H,G,L,D,causal", [(1, 2, 1, 1024, 64, False), (1, 2, 2, 500, 80, True), (1, 4, 2, 700, 128, True), (1, 2, 1, 33, 128, False), (64, 4, 4, 100, 64, False)])
def test_gradients_of_any_size(B, H, G, L, D, causal, size):
    gen = torch.Generator(device=DEV).manual_seed(L)
    q, k, v = _rand(gen, (B, L, H, D)), _rand(gen, (B, L, G, D)), _rand(gen, (B, L, G, D))
    _gradients(q, k, v, _rand(gen, (B, L, H, D), size), D ** -0.5, causal)


@pytest.mark.parametrize("D", [64, 80, 128])
@pytest.mark.parametrize("B", [1, 60])
def test_score_gradients_past_the_largest_number(B, D):
    """ds passes 65504 on its way to gradients that do not."""
    gen = torch.Generator(device=DEV).manual_seed(D)
    q, k, v = _rand(gen, (B, 40, 4, D), 0.02), _rand(gen, (B, 40, 4, D), 0.02), _rand(gen, (B, 40, 4, D), 60.0)
    dout = _rand(gen, (B, 40, 4, D), 6000.0)
    ds = dout.double().norm(dim=3).max() * v.double().norm(dim=3).max() / 40
    assert ds > 65504
    _gradients(q, k, v, dout, D ** -0.5, False, ("dq", "dk"))


@pytest.mark.parametrize("D", [64, 80, 128])
def test_gradients_that_grow_along_the_sequence(D):
    """Rows of dout from 1e-6 to 1e4 and back: each query's gradient and each key's is held to its own largest terms."""
    gen = torch.Generator(device=DEV).manual_seed(3)
    L = 640
    q, k, v = _rand(gen, (1, L, 2, D)), _rand(gen, (1, L, 2, D)), _rand(gen, (1, L, 2, D), 0.1)
    for flip in (False, True):
        size = torch.logspace(-6, 3, L, device=DEV)
        dout = (torch.randn((1, L, 2, D), generator=gen, device=DEV) * (size.flip(0) if flip else size)[None, :, None, None]).to(F16)
        _gradients(q, k, v, dout, D ** -0.5, True)


@pytest.mark.parametrize("D", [64, 80, 128])
def test_gradients_of_probabilities_below_the_smallest_normal_number(D):
    gen = torch.Generator(device=DEV).manual_seed(4)
    Lq, Lk = 70, 131072
    _gradients(_rand(gen, (1, Lq, 1, D)), _rand(gen, (1, Lk, 1, D)), _rand(gen, (1, Lk, 1, D)), _rand(gen, (1, Lq, 1, D)), D ** -0.5, False)


@pytest.mark.parametrize("Lq", [1, 40])
@pytest.mark.parametrize("D", [64, 80, 128])
def test_many_small_probabilities_beside_a_large_one(Lq, D):
    """One key has all but 0.3 % of the probability and no value, so that the output is the other keys' alone."""
    gen = torch.Generator(device=DEV).manual_seed(5)
    Lk = 131072
    q, k = torch.zeros((1, Lq, 1, D), device=DEV, dtype=F16), torch.zeros((1, Lk, 1, D), device=DEV, dtype=F16)
    q[..., 0] = 1
    k[:, 0, :, 0] = 17.7
    k[:, 1:, :, 0] = _rand(gen, (1, Lk - 1, 1), 0.3)
    v = (1 + 0.1 * torch.randn((1, Lk, 1, D), generator=gen, device=DEV)).to(F16)
    v[:, 0] = 0
    out, lse = ops.attention_fwd(q, k, v, None, 1.0, False, True)
    torch.cuda.synchronize()
    want, wlse, tol, tlse = ref.forward(q, k, v, None, 1.0, False)
    assert 0.002 < float(want.max()) < 0.004
    close(out, want, tol, "out")
    close(lse, wlse, tlse, "lse")


@pytest.mark.parametrize("shift", [0.0, 30.0, -200.0])
@pytest.mark.parametrize("Lq", [2, 70])
def test_scores_far_from_zero_and_growing_maxima(Lq, shift):
    gen = torch.Generator(device=DEV).manual_seed(6)
    q, k, v = _rand(gen, (1, Lq, 2, 64)), _rand(gen, (1, 1500, 2, 64)), _rand(gen, (1, 1500, 2, 64))
    q[..., 0] = 8
    k[..., 0] = (torch.linspace(0, 10, 1500, device=DEV) + shift).to(F16)[None, :, None]
    out, lse = ops.attention_fwd(q, k, v, None, 1.0, False, True)
    want, wlse, tol, tlse = ref.forward(q, k, v, None, 1.0, False)
    close(out, want, tol, "out")
    close(lse, wlse, tlse, "lse")


@pytest.mark.parametrize("Lq,Lk", [(1, 1), (40, 1), (50, 50), (5, 700)])
def test_a_query_of_one_key_returns_its_value(Lq, Lk):
    gen = torch.Generator(device=DEV).manual_seed(7)
    q, k, v = _rand(gen, (3, Lq, 2, 64), 3.0), _rand(gen, (3, Lk, 2, 64), 3.0), _rand(gen, (3, Lk, 2, 64))
    n = torch.ones(3, dtype=torch.int32, device=DEV)
    assert torch.equal(ops.attention_fwd(q, k, v, n, 0.5, False, False)[0], v[:, :1].expand(3, Lq, 2, 64))
