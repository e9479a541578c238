"""Attention of few queries where there are more workgroups than CUs (of 2 waves each): against the formulas in 64 bits."""
import pytest
import torch

import deep_optimization_amd  # noqa: F401
from tests import attention_reference as ref
from tests.block_reference import close

pytestmark = pytest.mark.gpu
DEV = "cuda"
ops = torch.ops.act_lib


@pytest.mark.parametrize("D", [40, 64, 80, 96, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
@pytest.mark.parametrize("B,H,G,Lq,Lk,causal", [(40, 16, 8, 1, 300, False), (33, 35, 7, 3, 1100, True), (300, 1, 1, 32, 33, True)])
def test_many_heads_of_few_queries(B, H, G, Lq, Lk, causal, D, dtype):
    gen = torch.Generator(device=DEV).manual_seed(Lk + D)
    q, k, v = (torch.randn(s, generator=gen, device=DEV).to(dtype) for s in ((B, Lq, H, D), (B, Lk, G, D), (B, Lk, G, D)))
    for lengths in (None, torch.tensor([(37 * i) % (Lk + 1) for i in range(B)], dtype=torch.int32, device=DEV)):
        out, lse = ops.attention_fwd(q, k, v, lengths, D ** -0.5, causal, True)
        want, wlse, tol, tlse = ref.forward(q, k, v, lengths, D ** -0.5, causal)
        close(out, want, tol, "out")
        close(lse, wlse, tlse, "lse")
        if lengths is not None:
            assert not out[0].any() and (lse[0] == -torch.inf).all()
