"""Attention's gradients where queries see a few keys, against the exact ones: of the exact output, not of the rounded one that attention_bwd is
given (which tests/test_gpu_attention.py holds it to).

The expected error, in norms, from the roundings that the operator states, each independent and off by r of its value (r as measured of the output's
rounding): the result's own; one of every term of its sum (ds, for its product); and delta = dout . out of an out whose probabilities and whose
result were rounded, off by r times the root of the sums of (p dp)^2 and (dout out)^2, which each of the query's keys feels by its probability. Where a
query sees two keys, dp - delta is a small difference and the last is the largest. Twice the expected variance is allowed for."""
import pytest
import torch

import deep_optimization_amd  # noqa: F401
from tests import attention_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
ops = torch.ops.act_lib
F16, BF16 = torch.float16, torch.bfloat16


def _exact(q, k, v, dout, lengths, scale, causal):
    """(q, k, dout, out, p, dp, ds) in 64 bits, heads first."""
    H = q.shape[2]
    mask = ref.seen(q.shape[0], q.shape[1], k.shape[1], lengths, causal, q.device)
    q, k, v, do = (ref._heads(t, H) for t in (q, k, v, dout))
    s = (q @ k.transpose(2, 3).contiguous() * scale).masked_fill(~mask, -torch.inf)
    p = torch.where(mask, torch.exp(s - torch.logsumexp(s, 3, keepdim=True)), 0.0)
    out = p @ v
    dp = do @ v.transpose(2, 3).contiguous()
    return q, k, do, out, p, dp, p * (dp - (do * out).sum(3, keepdim=True))


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("B,H,G,Lq,Lk,D,causal,keys", [(64, 8, 8, 2, 2, 64, False, None), (400, 4, 4, 16, 16, 64, True, None), (30, 4, 2, 90, 100, 64, False, (2, 16)),
                                                       (300, 2, 1, 40, 60, 40, False, (2, 6)), (60, 4, 4, 30, 150, 80, False, (2, 3)), (40, 4, 2, 16, 16, 128, True, None),
                                                       (40, 4, 2, 50, 300, 128, False, (2, 5))])
def test_gradients_of_queries_that_see_a_few_keys(B, H, G, Lq, Lk, D, causal, keys, dtype):
    gen = torch.Generator(device=DEV).manual_seed(Lk)
    q, k, v, dout = (torch.randn(s, generator=gen, device=DEV).to(dtype) for s in ((B, Lq, H, D), (B, Lk, G, D), (B, Lk, G, D), (B, Lq, H, D)))
    lengths = None if keys is None else torch.randint(keys[0], keys[1] + 1, (B,), generator=gen, device=DEV, dtype=torch.int32)
    scale = D ** -0.5
    out, lse = ops.attention_fwd(q, k, v, lengths, scale, causal, True)
    got_q, got_k, _ = ops.attention_bwd(dout, q, k, v, out, lse, lengths, scale, causal)
    torch.cuda.synchronize()
    qh, kh, do, o, p, dp, ds = _exact(q, k, v, dout, lengths, scale, causal)
    r = float((o.to(dtype).double() - o).norm() / o.norm())
    delta = r * ((p * dp).square().sum(3) + (do * o).square().sum(3)).sqrt()
    dst, pt = ds.transpose(2, 3).contiguous(), p.transpose(2, 3).contiguous()
    for name, got, want, terms, felt in (
            ("dq", got_q, ref._back(scale * (ds @ kh)), (ds.square() @ kh.square()).sum(), (delta * (p @ kh).norm(dim=3)).square().sum()),
            ("dk", got_k, ref._back(scale * (dst @ qh), G), (dst.square() @ qh.square()).sum(), ((pt * delta[:, :, None]).square() @ qh.square()).sum())):
        own = float((want.to(dtype).double() - want).norm())
        off, size = float((got.double() - want).norm()), float(want.norm())
        expected = (own ** 2 + scale ** 2 * (r ** 2 * float(terms) + float(felt))) ** 0.5
        print(f"[few keys] {name}: off by {off / size:.3g} of its norm, expected {expected / size:.3g}, its own rounding {own / size:.3g}", flush=True)
        assert off <= 2 ** 0.5 * expected, name
