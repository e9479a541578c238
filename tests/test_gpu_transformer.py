"""The transformer block layers (modules/transformer.py) and the ViT built from them: their gradients against the operators',
against differences, and against the plain model in 32 bits; dropout's masks over passes and graph replays."""
import copy

import pytest
import torch
import torch.nn.functional as F

from deep_optimization_amd.graph import graph_module_in_place
from deep_optimization_amd.modules import transformer as T
from deep_optimization_amd.vit import VisionTransformer
from tests import block_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
ops = torch.ops.act_lib
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _rand(seed, shape, dtype=BF16, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def _leaf(seed, shape, dtype=BF16, scale=1.0):
    return _rand(seed, shape, dtype, scale).requires_grad_(True)


@pytest.mark.parametrize("autocast", [False, True])
@pytest.mark.parametrize("dt", [BF16, F16], ids=["bf16", "f16"])
def test_functions_return_the_operators_gradients(dt, autocast):
    """Each function's result and gradients are the operators' on the same arguments, cast to the leaves' types."""
    pt = F32 if autocast else dt
    x, w1, b1 = _leaf(0, (3, 50, 72), dt), _leaf(1, (136, 72), pt, 0.1), _leaf(2, (136,), pt)
    w2, b2, res = _leaf(3, (72, 136), pt, 0.1), _leaf(4, (72,), pt), _leaf(5, (3, 50, 72), dt)
    dy = _rand(6, (3, 50, 72), dt)
    gd = F32 if autocast else dt
    with torch.autocast("cuda", dtype=dt, enabled=autocast):
        y = T.mlp(x, w1, b1, w2, b2, res, "gelu")
    y.backward(dy)
    with torch.no_grad():
        h, pre = ops.linear_act_fwd(x, w1.to(dt), b1, None, "gelu", True)
        want, _ = ops.linear_act_fwd(h, w2.to(dt), b2, res, "none", False)
        dz, dw2, db2 = ops.linear_act_bwd(dy, h, w2.to(dt), None, "none", pre, "gelu", True, True, True, gd)
        dx, dw1, db1 = ops.linear_act_bwd(dz, x, w1.to(dt), None, "none", None, "none", True, True, True, gd)
    assert torch.equal(y, want) and torch.equal(res.grad, dy)
    for leaf, g in ((x, dx), (w1, dw1), (b1, db1), (w2, dw2), (b2, db2)):
        assert leaf.grad.dtype == leaf.dtype and torch.equal(leaf.grad, g)
    with torch.no_grad(), torch.autocast("cuda", dtype=dt, enabled=autocast):
        assert torch.equal(T.mlp(x, w1, b1, w2, b2, res, "gelu"), want)

    x, w, b, res = _leaf(7, (40, 72), dt), _leaf(8, (56, 72), pt, 0.1), None, _leaf(9, (40, 56), F32)
    dy = _rand(10, (40, 56), F32)
    with torch.autocast("cuda", dtype=dt, enabled=autocast):
        y = T.linear_act(x, w, b, res, "silu")
    y.backward(dy)
    with torch.no_grad():
        want, pre = ops.linear_act_fwd(x, w.to(dt), None, res, "silu", True)
        dx, dw, _ = ops.linear_act_bwd(dy.to(dt), x, w.to(dt), pre, "silu", None, "none", True, True, False, gd)
    assert y.dtype == F32 and torch.equal(y, want) and torch.equal(res.grad, dy) and torch.equal(x.grad, dx) and torch.equal(w.grad, dw)

    x, w, b = _leaf(11, (5, 7, 96), dt), _leaf(12, (96,), pt), _leaf(13, (96,), pt)
    dy, dr = _rand(14, (5, 7, 96), dt), _rand(15, (5, 7, 96), dt)
    with torch.autocast("cuda", dtype=dt, enabled=autocast):
        y, same = T.layer_norm_residual(x, w, b, 1e-6)
    torch.autograd.backward([y, same], [dy, dr])
    with torch.no_grad():
        want, mean, rstd = ops.layer_norm_fwd(x, w, b, 1e-6, dt)
        dx, dw, db = ops.layer_norm_bwd(dy, x, mean, rstd, w, dr, True, True)
    assert torch.equal(y, want) and torch.equal(same, x) and torch.equal(x.grad, dx)
    assert torch.equal(w.grad, dw.to(pt)) and torch.equal(b.grad, db.to(pt))

    x.grad = None
    _, same = T.layer_norm_residual(x, w, b, 1e-6)
    same.backward(dr)
    assert torch.equal(x.grad, dr)
    x.grad = None
    T.layer_norm(x, None, None).backward(dy)
    y, mean, rstd = ops.layer_norm_fwd(x.detach(), None, None, 1e-5, dt)
    assert torch.equal(x.grad, ops.layer_norm_bwd(dy, x.detach(), mean, rstd, None, None, False, False)[0])


@pytest.mark.parametrize("act", ["none", "relu", "gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("what", ["x", "weight", "bias"])
def test_linear_gradients_against_differences(act, what):
    """(L(v + d) - L(v - d)) / 2 against <grad L, d> for L = <y, g>, y in fp32 (an fp32 residual of zeros). v lies on a grid of
    2^-4 below 4 and d is +-2^-4, so v +- d are exact in bf16. Bounds: y's fp32 sums (ref.linear_fwd), the cubic term of the
    difference (|act'''| <= 1.6; a kink of relu moves by |delta| where |z| < |delta|), the gradient's roundings: pre to bf16
    (|act''| <= 1.2), dz to bf16, the result once."""
    M, K, N = 24, 40, 56
    grid = lambda seed, shape: ((_rand(seed, shape, F32) * 16).round() / 16).clamp(-3.9, 3.9).to(BF16)  # noqa: E731
    v = {"x": grid(0, (M, K)), "weight": grid(1, (N, K)), "bias": grid(2, (N,))}
    g = _rand(3, (M, N), F32)
    d = torch.where(_rand(4, v[what].shape, F32) > 0, 2.0 ** -4, -(2.0 ** -4)).to(BF16)
    zero = torch.zeros((M, N), device=DEV)

    def loss(shift):
        a = {k: (t.float() + shift * d.float() if k == what else t).to(BF16) for k, t in v.items()}
        y = T.linear_act(a["x"], a["weight"], a["bias"], zero, act)
        return (y.double() * g.double()).sum(), ref.linear_fwd(a["x"], a["weight"], a["bias"], zero, act)

    (up, rup), (down, rdown) = loss(1.0), loss(-1.0)
    leaves = {k: t.clone().requires_grad_(k == what) for k, t in v.items()}
    gb = g.to(BF16)
    T.linear_act(leaves["x"], leaves["weight"], leaves["bias"], zero, act).backward(gb.float())
    got = (leaves[what].grad.double() * d.double()).sum()
    z = v["x"].double() @ v["weight"].double().t() + v["bias"].double()
    delta = (d.double() @ v["weight"].double().t() if what == "x" else v["x"].double() @ d.double().t() if what == "weight" else
             d.double().expand(M, N)).abs()
    u, ga = ref.U[BF16], g.abs().double()
    tol = (ga * (rup[2] + rdown[2] + (ref.U[F32]) * (rup[0].abs() + rdown[0].abs()))).sum() / 2
    tol += ((g - gb.float()).abs().double() * 1.2 * delta).sum()  # the gradient that the function was given
    if act == "relu":
        tol += (ga * delta * (z.abs() <= delta + u * z.abs())).sum()
    elif act != "none":
        tol += (ga * delta ** 3 * 1.6 / 6).sum() + (ga * delta * (1.2 * u * z.abs() + ref.ACT_ERR)).sum()
    # |dz| <= 1.2 |g|, rounded, times the other operand; then the result's own rounding
    tol += (1.2 * ga * u * delta).sum() * 1.01
    tol += (u * leaves[what].grad.double().abs() * d.double().abs()).sum() + 1e-6 * (ga * delta).sum()
    assert abs((up - down) / 2 - got) <= tol, (float((up - down) / 2), float(got), float(tol))


def _vit(**kw):
    torch.manual_seed(0)
    return VisionTransformer(img_size=32, patch_size=8, num_classes=11, embed_dim=64, depth=2, num_heads=2, **kw).to(DEV)


def _grads(model, x, y, autocast=True):
    model.zero_grad()
    with torch.autocast("cuda", dtype=BF16, enabled=autocast):
        out = model(x)
        loss = F.cross_entropy(out.float(), y)
    loss.backward()
    return out.detach().float(), {n: p.grad.float().clone() for n, p in model.named_parameters()}


def test_fused_vit_is_the_plain_vit():
    """The same parameters by name, and results no further from the 32-bit model's than twice the plain bf16 model's (both
    round to bf16 at each layer; the fused one at fewer places)."""
    plain, fused = _vit(), _vit(fused=True)
    with torch.no_grad():  # (biases and norms that count)
        for i, p in enumerate(plain.parameters()):
            p.add_(_rand(i, p.shape, F32, 0.05))
    assert not any(fused.load_state_dict(plain.state_dict()))
    x, y = _rand(100, (6, 3, 32, 32), F32), torch.arange(6, device=DEV)
    cpu = copy.deepcopy(plain).cpu()
    cpu_out = cpu(x.cpu())
    F.cross_entropy(cpu_out, y.cpu()).backward()
    want = {n: p.grad.to(DEV) for n, p in cpu.named_parameters()}
    want["out"] = cpu_out.detach().to(DEV)
    off = {}
    for name, m in (("plain", plain), ("fused", fused)):
        out, g = _grads(m, x, y)
        off[name] = {n: float((v - want[n]).norm() / want[n].norm()) for n, v in (*g.items(), ("out", out))}
    for n in want:
        assert off["fused"][n] <= 2 * off["plain"][n] + 2.0 ** -8, (n, off["fused"][n], off["plain"][n])


def test_fused_vit_in_bf16_without_autocast_and_in_eval():
    model = _vit(fused=True, drop_rate=0.25).to(BF16)
    x = _rand(0, (4, 3, 32, 32))
    model.eval()
    with torch.no_grad():
        assert torch.equal(model(x), model(x)) and int(model.dropout_rng.step) == 0
    model.train()
    out, g = _grads(model, x, torch.arange(4, device=DEV), autocast=False)
    assert int(model.dropout_rng.step) == 1 and torch.isfinite(out).all() and all(torch.isfinite(v).all() and v.any() for v in g.values())
    assert not torch.equal(model(x).float(), out)


def test_dropout_masks_of_layers_and_passes_differ_and_the_backward_has_the_forwards():
    rng = T.DropoutRng(seed=5).to(DEV)
    layers = [T.DropoutAdd(0.5, rng) for _ in range(2)]
    x = torch.ones(4096, device=DEV, requires_grad=True)
    masks, held = [], []
    for _ in range(3):
        rng(x)
        for layer in layers:
            y = layer(x, torch.zeros_like(x))
            masks.append(y.detach())
            held.append(y)
    for i in range(6):
        for j in range(i):
            assert 0.4 < float((masks[i] == masks[j]).float().mean()) < 0.6
    for y, m in reversed(list(zip(held, masks))):  # backward passes after all the forwards
        x.grad = None
        y.backward(torch.ones_like(y))
        assert torch.equal(x.grad, m)
    for layer in layers:
        layer.eval()
    assert torch.equal(layers[0](x, x), x + x) and layers[0](x) is x


def test_fused_vit_with_dropout_in_a_captured_graph():
    """Replays of the captured step equal the eager model's passes with the same count, and differ from each other."""
    eager = _vit(fused=True, drop_rate=0.2, dropout_seed=3)
    graphed = copy.deepcopy(eager)
    graph_module_in_place(graphed)
    x, y = _rand(0, (4, 3, 32, 32), F32), torch.arange(4, device=DEV)
    outs = []
    for _ in range(4):
        out, g = _grads(graphed, x, y)
        torch.cuda.synchronize()
        eager.dropout_rng.step.copy_(graphed.dropout_rng.step - 1)
        want, gw = _grads(eager, x, y)
        assert torch.equal(eager.dropout_rng.step, graphed.dropout_rng.step)
        # (attention's own kernels need not be the same ones; masks that differed would be off by far more)
        assert (out - want).norm() <= 2.0 ** -7 * want.norm()
        for n in g:
            assert (g[n] - gw[n]).norm() <= 2.0 ** -5 * gw[n].norm() + 1e-6, n
        outs.append(out)
    assert not torch.equal(outs[0], outs[1]) and not torch.equal(outs[2], outs[3])


def test_refusals():
    with pytest.raises(ValueError):
        VisionTransformer(img_size=32, patch_size=8, embed_dim=64, depth=1, num_heads=2, drop_rate=0.1)
    with pytest.raises(ValueError):
        T.Mlp(8, 16, drop=0.1)
    with pytest.raises(ValueError):
        T.LinearAct(8, 16, act="tanh")
    with pytest.raises(ValueError):
        T.LayerNorm((4, 8))
    with pytest.raises(ValueError):
        T.DropoutAdd(1.5, T.DropoutRng(0))
    drop = T.DropoutAdd(0.5, T.DropoutRng(0).to(DEV))
    with pytest.raises(RuntimeError):
        drop(torch.ones(8, device=DEV))
    with pytest.raises(RuntimeError):  # products in fp32
        T.LinearAct(8, 16).to(DEV)(torch.ones(2, 8, device=DEV))
