"""Every tile of the linear products with every epilogue that weighs in its choice, at sizes that dopt_linear_epilogue_tile says take it (the
choice of the call itself), with sums of whole slabs (64 terms) and with a remainder. The persistent tiles (160 and 256 high) at
sizes where workgroups go on to further tiles: prefetch of the next tile, counted waits over the epilogue's stores, the alternating
bias rows."""
import itertools

import pytest
import torch

import deep_optimization_amd  # noqa: F401
from deep_optimization_amd import _lib
from tests import block_reference as ref
from tests.test_gpu_linear_act import check_bwd, check_fwd

DEV = "cuda"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
FORWARD, INPUT_GRAD, WEIGHT_GRAD = 0, 1, 2
# indexes of the cost table in csrc/linear_gemm.hip: 32 x 64, 64 x 64 in four stages and in two, 128 x 64, 128 x 128, 160 and 256 x 256; then those of
# rows at any element, 32 x 64 and 64 x 64; 100: the split weight gradient
SMALL, BIG, REG = {0, 1, 2, 3, 4}, {5: 160, 6: 256}, {7, 8}
# (activation, residual, pre, fp32 result) of the forward product
EPILOGUES = {"plain": (0, 0, 0, 0), "act": (1, 0, 0, 0), "act_pre": (1, 0, 1, 0), "res": (0, 1, 0, 0), "act_pre_res": (1, 1, 1, 0),
             "res_f32": (0, 1, 0, 1), "act_pre_res_f32": (1, 1, 1, 1)}
gpu = pytest.mark.gpu
DT = pytest.mark.parametrize("dt", [BF16, F16], ids=["bf16", "f16"])


def _tile(product, M, K, N, any_rows=0, act=0, side=0, pre=0, y_f32=0):
    return _lib.lib().dopt_linear_epilogue_tile(product, M, N, K, any_rows, act, side, pre, y_f32)


def _sum(product, M, K, N):
    return {FORWARD: K, INPUT_GRAD: N, WEIGHT_GRAD: M}[product]


def _result(product, M, K, N):
    return {FORWARD: (M, N), INPUT_GRAD: (M, K), WEIGHT_GRAD: (N, K)}[product]


def _sizes(product, n_cu, odd=0, **epilogue):
    """{(tile, whether the sum has whole slabs only): the cheapest (M, K, N) that takes it}; the persistent tiles' with more of them than CUs."""
    rows = (17, 64, 130, 320, 1500, 3008, 6000, 9000, 12032, 16300, 20000)
    cols = (72, 128, 264, 320, 520, 776, 1536, 1544, 2040, 3008) if not odd else (73, 129, 265, 777, 1537)
    found = {}
    for M, K, N in sorted(itertools.product(rows, cols, cols), key=lambda s: s[0] * s[1] * s[2]):
        tile = _tile(product, M, K, N, odd, **epilogue)
        if tile in BIG:
            m, n = _result(product, M, K, N)
            if -(-m // BIG[tile]) * -(-n // 256) <= n_cu:
                continue
        found.setdefault((tile, _sum(product, M, K, N) % 64 == 0), (M, K, N))
    return found


def _wanted(tiles, whole=(True, False)):
    return {(t, w) for t in tiles for w in whole}


def _epilogue_args(name):
    act, side, pre, f32 = EPILOGUES[name]
    return dict(act=act, side=side, pre=pre, y_f32=f32)


@pytest.mark.parametrize("name", EPILOGUES)
def test_there_are_sizes_for_every_tile(name):
    """At 256 CUs, which is what the choice assumes without a GPU (the tests below ask for the GPU's own)."""
    if torch.cuda.is_available():
        pytest.skip("asks for the GPU's own CUs below")
    e = _epilogue_args(name)
    assert set(_sizes(FORWARD, 256, **e)) == _wanted(SMALL | (set() if e["y_f32"] else set(BIG)))
    assert set(_sizes(FORWARD, 256, odd=1, **e)) == _wanted(REG, (False,))
    if name in ("plain", "act"):
        assert set(_sizes(INPUT_GRAD, 256, act=e["act"])) == _wanted(SMALL | set(BIG))
        assert set(_sizes(INPUT_GRAD, 256, odd=1, act=e["act"])) == _wanted(REG, (False,))
    if name == "plain":
        assert set(_sizes(WEIGHT_GRAD, 256)) == _wanted(SMALL | {100})
        assert set(_sizes(WEIGHT_GRAD, 256, odd=1)) == _wanted(REG)


def _cus():
    return torch.cuda.get_device_properties(0).multi_processor_count


@gpu
@DT
@pytest.mark.parametrize("name", EPILOGUES)
def test_forward(name, dt):
    e = _epilogue_args(name)
    found = _sizes(FORWARD, _cus(), **e)
    assert set(found) == _wanted(SMALL | (set() if e["y_f32"] else set(BIG)))
    for (tile, _), (M, K, N) in found.items():
        acts = ("none",) if not e["act"] else ("relu", "gelu", "gelu_tanh", "silu") if tile in BIG else ("gelu",)  # (instances of their own)
        for i, act in enumerate(acts):
            assert _tile(FORWARD, M, K, N, act=_lib.LIN_ACTS[act], side=e["side"], pre=e["pre"], y_f32=e["y_f32"]) == tile
            check_fwd(M, K, N, dt, act, bias=(F32, dt, None)[i % 3], res=None if not e["side"] else F32 if e["y_f32"] else dt, pre=bool(e["pre"]), seed=tile)


@gpu
@DT
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "gelu_tanh", "silu"])
def test_input_gradient(act, dt):
    found = _sizes(INPUT_GRAD, _cus(), act=_lib.LIN_ACTS[act])
    assert set(found) == _wanted(SMALL | set(BIG))
    for (tile, _), (M, K, N) in found.items():
        check_bwd(M, K, N, dt, "none", act, parts=(True, False, False), seed=tile)


@gpu
@DT
def test_weight_gradient(dt):
    found = _sizes(WEIGHT_GRAD, _cus())
    assert set(found) == _wanted(SMALL | {100})
    for M, K, N in found.values():
        check_bwd(M, K, N, dt, grad=F32, parts=(False, True, True))
        check_bwd(M, K, N, dt, grad=dt, parts=(False, True, True))
        check_bwd(M, K, N, dt, grad=dt, parts=(False, True, False))


def _rand(seed, shape, dt, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dt)


@gpu
@DT
@pytest.mark.parametrize("name", EPILOGUES)
def test_rows_at_any_element(name, dt):
    """The C entries, which copy nothing."""
    L, code, stream = _lib.lib(), {BF16: _lib.BF16, F16: _lib.F16}[dt], torch.cuda.current_stream().cuda_stream
    e = _epilogue_args(name)
    found = _sizes(FORWARD, _cus(), odd=1, **e)
    assert set(found) == _wanted(REG, (False,))
    for (tile, _), (M, K, N) in found.items():
        print(f"[linear tiles] forward at any element {M} x {K} x {N} {dt} {name}", flush=True)
        yt = F32 if e["y_f32"] else dt
        x, w, b = _rand(0, (M, K), dt), _rand(1, (N, K), dt, K ** -0.5), _rand(2, (N,), F32)
        r = _rand(3, (M, N), yt) if e["side"] else None
        y, pre = torch.empty((M, N), device=DEV, dtype=yt), torch.empty((M, N), device=DEV, dtype=dt) if e["pre"] else None
        act = "gelu" if e["act"] else "none"
        _lib.check(L.dopt_linear_forward(x.data_ptr(), K, w.data_ptr(), K, code, M, N, K, b.data_ptr(), _lib.F32, None if r is None else r.data_ptr(),
                                         _lib.LIN_ACTS[act], y.data_ptr(), _lib.F32 if e["y_f32"] else code, None if pre is None else pre.data_ptr(),
                                         stream), "linear")
        wy, wz, ty, tz = ref.linear_fwd(x, w, b, r, act)
        ref.close(y, wy, ty, f"tile {tile}")
        if pre is not None:
            ref.close(pre, wz, tz, f"tile {tile} pre")
    if name not in ("plain", "act"):
        return
    for (tile, _), (M, K, N) in _sizes(INPUT_GRAD, _cus(), odd=1, act=e["act"]).items():
        print(f"[linear tiles] input gradient at any element {M} x {K} x {N} {dt} {name}", flush=True)
        dz, w, z = _rand(0, (M, N), dt), _rand(1, (N, K), dt, N ** -0.5), _rand(2, (M, K), dt) if e["act"] else None
        dx = torch.empty((M, K), device=DEV, dtype=dt)
        act = "silu" if e["act"] else "none"
        _lib.check(L.dopt_linear_input_grad(dz.data_ptr(), N, w.data_ptr(), K, code, M, N, K, None if z is None else z.data_ptr(), _lib.LIN_ACTS[act],
                                            dx.data_ptr(), stream), "linear")
        want, _, _, tol, _, _ = ref.linear_bwd(dz, torch.zeros((M, K), device=DEV, dtype=dt), w, None, "none", z, act)
        ref.close(dx, want, tol, f"tile {tile}")


@gpu
@DT
def test_the_vit_mlp_over_many_tiles(dt):
    """ViT-B/16's MLP at batch 128: its products take the persistent tiles, several to a workgroup."""
    M = 128 * 197
    assert _tile(FORWARD, M, 768, 3072, act=2, pre=1) in BIG and _tile(FORWARD, M, 3072, 768, side=1) in BIG and _tile(INPUT_GRAD, M, 3072, 768, act=2) in BIG
    check_fwd(M, 768, 3072, dt, "gelu", bias=dt, pre=True)
    check_fwd(M, 768, 3072, dt, "gelu", bias=F32, pre=True, res=dt)
    check_fwd(M, 3072, 768, dt, "none", bias=dt, res=dt)
    check_bwd(M, 3072, 768, dt, "none", "gelu", parts=(True, False, False))
