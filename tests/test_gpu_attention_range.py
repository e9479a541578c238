"""Attention where values are very small, very large or not finite: against the formulas in 64 bits (tests/attention_reference.py)."""
import math

import pytest
import torch

import deep_optimization_amd  # noqa: F401

pytestmark = pytest.mark.gpu
DEV = "cuda"
ops = torch.ops.act_lib
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
DT = pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])


def _rand(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device=DEV) * scale).to(dtype)


@DT
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("B,H,G,Lq,Lk,D", [(70, 6, 3, 40, 100, 64), (100, 4, 4, 7, 33, 40), (2, 4, 2, 40, 200, 80), (2, 4, 2, 40, 200, 128)])
def test_keys_past_a_length_have_zero_gradients_whatever_the_queries_hold(B, H, G, Lq, Lk, D, bad, dtype):
    """A query's q or dout that is not finite makes gradients of the keys that it sees; those past the length have zeros all the same."""
    gen = torch.Generator(device=DEV).manual_seed(1)
    q, k, v = _rand(gen, (B, Lq, H, D), dtype), _rand(gen, (B, Lk, G, D), dtype), _rand(gen, (B, Lk, G, D), dtype)
    lens = torch.tensor([(7 * i + 3) % (Lk + 1) for i in range(B)], dtype=torch.int32, device=DEV)
    out, lse = ops.attention_fwd(q, k, v, lens, 0.125, False, True)
    dout = _rand(gen, q.shape, dtype)
    dout[:, 3, :, 5] = bad
    past = torch.arange(Lk, device=DEV) >= lens[:, None]
    for name, t in zip(("dk", "dv"), ops.attention_bwd(dout, q, k, v, out, lse, lens, 0.125, False)[1:]):
        assert bool((t[past] == 0).all()), name
        assert not t[~past].isfinite().all(), name
