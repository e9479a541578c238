"""The layer norm, dropout and linear operators as the framework runs them: the native operators against the Python ones bit for
bit, torch.library.opcheck, other streams, captured graphs, and every tile that the linear products choose from."""
import pytest
import torch

import deep_optimization_amd  # noqa: F401
from deep_optimization_amd import _lib, dropout_lib, linear_lib, ln_lib
from tests import block_reference as ref
from tests.test_gpu_linear_act import check_bwd, check_fwd
from tests.test_gpu_native_ops import same
from tests.test_gpu_opcheck import TESTS

pytestmark = pytest.mark.gpu
DEV = "cuda"
ops = torch.ops.act_lib
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _rand(seed, shape, dtype=BF16, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def _calls(dt=BF16, M=70, K=88, N=56):
    """(operator, arguments) of each, with and without the optional ones."""
    x, w, b, dy = _rand(0, (M, K), dt), _rand(1, (N, K), dt, 0.1), _rand(2, (N,), F32), _rand(3, (M, N), dt)
    step = torch.tensor([4], device=DEV)
    ln_w = _rand(4, (K,), F32)
    _, mean, rstd = ops.layer_norm_fwd(x, None, None, 1e-5, dt)
    return [("layer_norm_fwd", (x, ln_w, ln_w, 1e-5, dt)), ("layer_norm_fwd", (x, None, None, 1e-6, F32)),
            ("layer_norm_bwd", (x, x, mean, rstd, ln_w, x, True, True)), ("layer_norm_bwd", (x, x, mean, rstd, None, None, False, False)),
            ("layer_norm_bwd", (x, x, mean, rstd, None, None, False, True)),
            ("dropout_add_fwd", (x, x.float(), 0.3, 5, 7, step)), ("dropout_add_fwd", (x, None, 0.5, -1, 0, None)),
            ("dropout_bwd", (x, 0.3, 5, 7, step, F32)), ("dropout_bwd", (x, 0.3, 5, 7, None, dt)),
            ("linear_act_fwd", (x, w, b, dy.float(), "gelu", True)), ("linear_act_fwd", (x, w, None, None, "none", False)),
            ("linear_act_bwd", (dy, x, w, dy, "silu", x, "gelu", True, True, True, F32)),
            ("linear_act_bwd", (dy, x, w, None, "none", None, "none", True, True, True, dt)),
            ("linear_act_bwd", (dy, x, w, None, "none", None, "none", False, False, True, dt)),
            ("linear_act_bwd", (dy, x, w, None, "none", None, "none", True, False, False, F32))]


PYTHON = {"layer_norm_fwd": ln_lib._layer_norm_fwd, "layer_norm_bwd": ln_lib._layer_norm_bwd, "dropout_add_fwd": dropout_lib._dropout_add_fwd,
          "dropout_bwd": dropout_lib._dropout_bwd, "linear_act_fwd": linear_lib._linear_act_fwd, "linear_act_bwd": linear_lib._linear_act_bwd}


@pytest.mark.parametrize("dt", [BF16, F16], ids=["bf16", "f16"])
def test_native_operators_are_the_python_ones(dt):
    for sizes in ((70, 88, 56), (70, 87, 57), (3000, 333, 1001), (1, 64, 1000), (5000, 136, 2056)):
        for name, args in _calls(dt, *sizes):
            print(f"[block ops] {name} {dt} {sizes}", flush=True)
            same(getattr(ops, name)(*args), PYTHON[name](*args))


def test_native_refusals_are_the_python_ones():
    x, w, dy = _rand(0, (4, 64)), _rand(1, (32, 64)), _rand(2, (4, 32))
    _, mean, rstd = ops.layer_norm_fwd(x, None, None, 1e-5, BF16)
    for name, args in (("layer_norm_fwd", (x, w, None, 1e-5, BF16)), ("layer_norm_fwd", (x, None, None, 1e-5, torch.int32)),
                       ("layer_norm_fwd", (x, x[0], x[0].float(), 1e-5, BF16)), ("layer_norm_fwd", (x[0, 0], None, None, 1e-5, BF16)),
                       ("layer_norm_bwd", (dy, x, mean, rstd, None, None, True, True)), ("layer_norm_bwd", (x, x, mean[:3], rstd, None, None, True, True)),
                       ("layer_norm_bwd", (x, x, mean, rstd, None, x.float(), True, True)),
                       ("dropout_add_fwd", (x, None, 1.5, 0, 0, None)), ("dropout_add_fwd", (x, dy, 0.5, 0, 0, None)),
                       ("dropout_add_fwd", (x.double(), None, 0.5, 0, 0, None)), ("dropout_add_fwd", (x, None, 0.5, 0, 0, mean)),
                       ("dropout_bwd", (x, 0.5, 0, 0, None, torch.float64)),
                       ("linear_act_fwd", (x, w, None, None, "tanh", False)), ("linear_act_fwd", (x, w.half(), None, None, "none", False)),
                       ("linear_act_fwd", (x, w, x[0], None, "none", False)), ("linear_act_fwd", (x, w, None, dy[:3], "none", False)),
                       ("linear_act_bwd", (dy[:3], x, w, None, "none", None, "none", True, True, True, F32)),
                       ("linear_act_bwd", (dy, x, w, None, "gelu", None, "none", True, True, True, F32)),
                       ("linear_act_bwd", (dy, x, w, None, "none", None, "gelu", True, True, True, F32)),
                       ("linear_act_bwd", (dy, x, w, None, "none", None, "none", True, True, True, F16))):
        with pytest.raises((RuntimeError, ValueError)) as native:
            getattr(ops, name)(*args)
        with pytest.raises((RuntimeError, ValueError)) as python:
            PYTHON[name](*args)
        assert isinstance(native.value, ValueError) == isinstance(python.value, ValueError), (name, native.value, python.value)


@pytest.mark.parametrize("i", range(15))
def test_opcheck(i):
    name, args = _calls()[i]
    torch.library.opcheck(getattr(ops, name).default, args, test_utils=TESTS)


def test_on_another_stream():
    """Work that a side stream's inputs wait for: a launch on any other stream would read them before they are written."""
    want = [getattr(ops, n)(*a) for n, a in _calls()]
    busy = torch.randn((4096, 4096), device=DEV)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(4):
            busy = busy @ busy * 1e-3
        got = [getattr(ops, n)(*a) for n, a in _calls()]  # (the inputs are made on the side stream, behind that)
    side.synchronize()
    same(got, want)


def test_in_a_captured_graph():
    """Replays on new inputs give the eager results, with eager work between them."""
    cases = _calls(M=600, K=264, N=520)
    x = cases[0][1][0]
    for _ in range(2):
        [getattr(ops, n)(*a) for n, a in cases]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        outs = [getattr(ops, n)(*a) for n, a in cases]
    for i in range(4):
        x.copy_(_rand(50 + i, x.shape))
        g.replay()
        torch.cuda.synchronize()
        same(outs, [getattr(ops, n)(*a) for n, a in cases])
        torch.cuda.synchronize()


# sizes (M, K, N) of the layer that each product gives each of its tiles (include/dopt.h: DOPT_LIN_*; indexes of the cost table in
# csrc/linear_gemm.hip; -1 the kernel of at most 16 rows, 100 the split weight gradient); found by asking dopt_linear_tile
FORWARD, INPUT_GRAD, WEIGHT_GRAD = 0, 1, 2
CANDIDATES = [(M, K, N) for M in (17, 64, 300, 1500, 3000, 6000, 12000) for K in (72, 264, 776, 1544) for N in (72, 264, 776, 1544)]
ODD_CANDIDATES = [(M, K + 1, N + 1) for M, K, N in CANDIDATES]
TILES = {FORWARD: {-1, 0, 1, 2, 3, 4, 5, 6}, INPUT_GRAD: {0, 1, 2, 3, 4, 5, 6}, WEIGHT_GRAD: {0, 1, 2, 3, 4, 100}}
REG_TILES = {7, 8}


def _sizes_of(product, odd):
    found = {}
    if product == FORWARD:
        found[-1] = (9, 264 + odd, 72 + odd)
    for M, K, N in (ODD_CANDIDATES if odd else CANDIDATES):
        found.setdefault(_lib.lib().dopt_linear_tile(product, M, N, K, int(odd)), (M, K, N))
    return found


@pytest.mark.parametrize("dt", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("product", [FORWARD, INPUT_GRAD, WEIGHT_GRAD], ids=["forward", "input_grad", "weight_grad"])
def test_every_tile(product, dt):
    """Each tile of each product, whole and remaining slabs of the sum, with each epilogue that the tile has kernels of its own for."""
    found = _sizes_of(product, False)
    missing = TILES[product] - set(found)
    print(f"[linear tiles] product {product}: {found}; no size here takes {missing}", flush=True)
    assert len(missing) <= 2
    for tile, (M, K, N) in sorted(found.items()):
        whole = tuple(64 * ((v + 63) // 64) for v in (M, K, N)) if tile >= 0 else (M, 320, 64)
        for m, k, n in ((M, K, N), whole):
            if product == FORWARD:
                for act in ("none", "relu", "gelu", "gelu_tanh", "silu"):
                    check_fwd(m, k, n, dt, act, pre=True, res=dt)
            elif product == INPUT_GRAD:
                for act in ("none", "relu", "gelu", "gelu_tanh", "silu"):
                    check_bwd(m, k, n, dt, "none", act, parts=(True, False, False))
            else:
                for grad in (F32, dt):
                    check_bwd(m, k, n, dt, "none", "none", grad, parts=(False, True, True))
                check_bwd(m, k, n, dt, "none", "none", dt, parts=(False, True, False))


@pytest.mark.parametrize("dt", [BF16, F16], ids=["bf16", "f16"])
@pytest.mark.parametrize("product", [FORWARD, INPUT_GRAD, WEIGHT_GRAD], ids=["forward", "input_grad", "weight_grad"])
def test_every_tile_of_rows_at_any_element(product, dt):
    """The C entries on rows of odd lengths, as they are (the operators may copy them into aligned rows first)."""
    L, code = _lib.lib(), {BF16: _lib.BF16, F16: _lib.F16}[dt]
    for tile, (M, K, N) in sorted(_sizes_of(product, True).items()):
        print(f"[linear tiles] product {product} {dt} tile {tile}: {M} x {K} x {N}", flush=True)
        x, w, dz = _rand(0, (M, K), dt), _rand(1, (N, K), dt, K ** -0.5), _rand(2, (M, N), dt)
        if product == FORWARD:
            y = torch.empty((M, N), device=DEV, dtype=dt)
            rc = L.dopt_linear_forward(x.data_ptr(), K, w.data_ptr(), K, code, M, N, K, None, _lib.F32, None, 0, y.data_ptr(), code, None,
                                       torch.cuda.current_stream().cuda_stream)
            want, _, tol, _ = ref.linear_fwd(x, w, None, None, "none")
        elif product == INPUT_GRAD:
            y = torch.empty((M, K), device=DEV, dtype=dt)
            rc = L.dopt_linear_input_grad(dz.data_ptr(), N, w.data_ptr(), K, code, M, N, K, None, 0, y.data_ptr(),
                                          torch.cuda.current_stream().cuda_stream)
            want, _, _, tol, _, _ = ref.linear_bwd(dz, x, w, None, "none", None, "none")
        else:
            y = torch.empty((N, K), device=DEV, dtype=F32)
            rc = L.dopt_linear_weight_grad(dz.data_ptr(), N, x.data_ptr(), K, code, M, N, K, None, y.data_ptr(), None, None, None,
                                           torch.cuda.current_stream().cuda_stream)
            _, want, _, _, tol, _ = ref.linear_bwd(dz, x, w, None, "none", None, "none")
        _lib.check(rc, "linear")
        ref.close(y, want, tol, f"tile {tile}")
