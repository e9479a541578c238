"""act_lib::linear_act_fwd / linear_act_bwd against the formulas in 64 bits (tests/block_reference.py), within bounds from the
sums' lengths and the roundings."""
import pytest
import torch

import deep_optimization_amd  # noqa: F401
from tests import block_reference as ref

DEV = "cuda"
ops = torch.ops.act_lib
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
IDS = {F32: "f32", F16: "f16", BF16: "bf16"}
ACTS = ("none", "relu", "gelu", "gelu_tanh", "silu")
gpu = pytest.mark.gpu


def _rand(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device=DEV) * scale).to(dtype)


def check_fwd(M, K, N, dt, act="none", bias=F32, res=None, pre=False, seed=0, x=None, weight=None):
    print(f"[linear] forward {M} x {K} x {N} {dt} {act} bias {bias} residual {res} pre {pre}", flush=True)
    gen = torch.Generator(device=DEV).manual_seed(seed + M + K + N)
    x = _rand(gen, (M, K), dt) if x is None else x
    w = _rand(gen, (N, K), dt, max(K, 1) ** -0.5) if weight is None else weight
    b = _rand(gen, (N,), bias) if bias is not None else None
    r = _rand(gen, (*x.shape[:-1], N), res) if res is not None else None
    y, z = ops.linear_act_fwd(x, w, b, r, act, pre)
    wy, wz, ty, tz = ref.linear_fwd(x, w, b, r, act)
    assert y.dtype == (res or dt) and (z is None) == (not pre)
    ref.close(y, wy, ty, "y")
    if pre:
        assert z.dtype == dt
        ref.close(z, wz, tz, "pre")


def check_bwd(M, K, N, dt, act="none", in_act="none", grad=None, seed=0, parts=(True, True, True), dy=None, x=None):
    print(f"[linear] backward {M} x {K} x {N} {dt} {act} {in_act} gradients {grad} {parts}", flush=True)
    gen = torch.Generator(device=DEV).manual_seed(seed + M + K + N + 1)
    in_pre = _rand(gen, (M, K), dt) if in_act != "none" else None
    if x is None:
        x = _rand(gen, (M, K), dt) if in_pre is None else ref.act(in_pre.double(), in_act).to(dt)
    w = _rand(gen, (N, K), dt, max(K, 1) ** -0.5)
    pre = _rand(gen, (M, N), dt) if act != "none" else None
    dy = _rand(gen, (M, N), dt) if dy is None else dy
    grad = grad or dt
    dx, dw, db = ops.linear_act_bwd(dy, x, w, pre, act, in_pre, in_act, *parts, grad)
    wx, ww, wb, tx, tw, tb = ref.linear_bwd(dy, x, w, pre, act, in_pre, in_act)
    for got, want, tol, asked, kind, what in ((dx, wx, tx, parts[0], dt, "dx"), (dw, ww, tw, parts[1], grad, "dweight"),
                                              (db, wb, tb, parts[2], grad, "dbias")):
        assert (got is not None) == asked
        if asked:
            assert got.dtype == kind
            ref.close(got, want, tol, what)


# the smallest, odd and whole sizes: single tokens, edges of every tile, K of a few slabs and their remainders
SIZES = [(1, 8, 8), (1, 768, 1000), (2, 24, 3), (16, 64, 16), (16, 1000, 33), (17, 72, 31), (31, 128, 64), (33, 40, 65), (64, 64, 64),
         (100, 192, 200), (129, 256, 127), (197, 768, 768), (300, 520, 1000), (985, 384, 1536), (2000, 333, 129), (77, 1, 5), (5, 5, 1),
         (130, 13, 258), (1, 1, 1), (40, 4097, 24), (1, 777, 10), (4100, 136, 2056), (3000, 1000, 1000), (2600, 2504, 1000), (700, 999, 1001),
         (6000, 1001, 2047), (8200, 520, 776), (8200, 3000, 264), (12000, 64, 264), (5000, 72, 1544), (30000, 24, 40), (20000, 9, 17),
         (64, 100, 3000), (600, 3001, 600), (73, 73, 73), (72, 71, 70), (513, 65, 66)]


@gpu
@pytest.mark.parametrize("M,K,N", SIZES)
@pytest.mark.parametrize("dt", [BF16, F16], ids=IDS.get)
def test_sizes(M, K, N, dt):
    check_fwd(M, K, N, dt, "gelu", pre=True, res=dt)
    check_bwd(M, K, N, dt, "silu", "gelu")
    check_bwd(M, K, N, dt)


@gpu
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M,K,N", [(3, 64, 40), (150, 96, 100), (2500, 256, 3000)])
@pytest.mark.parametrize("dt", [BF16, F16], ids=IDS.get)
def test_epilogues(act, M, K, N, dt):
    for bias in (None, F32, F16, BF16):
        check_fwd(M, K, N, dt, act, bias=bias, res=None, pre=bias is None)
    check_fwd(M, K, N, dt, act, bias=dt, res=F32, pre=True)
    check_fwd(M, K, N, dt, act, bias=None, res=dt)
    check_bwd(M, K, N, dt, act, "none", F32)
    check_bwd(M, K, N, dt, "none", act)
    check_bwd(M, K, N, dt, act, act)


@gpu
@pytest.mark.parametrize("dt", [BF16, F16], ids=IDS.get)
def test_the_vit_layers(dt):
    for K, N in ((768, 2304), (768, 768), (768, 3072), (3072, 768)):
        check_fwd(1576, K, N, dt, "gelu" if N == 3072 else "none", pre=N == 3072, res=dt if N == 768 else None)
        check_bwd(1576, K, N, dt, "none", "gelu" if K == 3072 else "none")


@gpu
def test_parts_of_the_backward():
    for parts in ((True, False, False), (False, True, False), (False, False, True), (True, True, False), (False, True, True), (False, False, False)):
        check_bwd(200, 72, 130, BF16, "relu", parts=parts)
        check_bwd(200, 70, 131, F16, "none", parts=parts, grad=F32)


@gpu
@pytest.mark.parametrize("dt", [BF16, F16], ids=IDS.get)
def test_empty_sizes(dt):
    for M, K, N in ((0, 64, 64), (5, 0, 64), (5, 64, 0), (0, 0, 0)):
        check_fwd(M, K, N, dt, "gelu", res=dt, pre=True)
        check_bwd(M, K, N, dt, "silu")
        check_bwd(M, K, N, dt, grad=F32)


@gpu
def test_strided_rows_and_odd_addresses():
    gen = torch.Generator(device=DEV).manual_seed(4)
    tokens = _rand(gen, (40, 7, 64), BF16)
    flat = _rand(gen, (40 * 72 + 3,), BF16)
    for x in (tokens[:, 0], tokens[:, 3], tokens[:, 0, 8:40], tokens[:, 0, 1:33], tokens[:, 0, :13], flat[3:3 + 40 * 72].view(40, 72),
              tokens[:, 0].t()[:40].t(), tokens[:, :1, :1].expand(40, 1, 16).reshape(40, 16)[:, :16]):
        check_fwd(x.shape[0], x.shape[1], 50, BF16, x=x)
        check_bwd(x.shape[0], x.shape[1], 50, BF16, x=x)
    dy = _rand(gen, (40, 100), BF16)
    for d in (dy[:, :56], dy[:, 4:60], dy[:, 1:57], dy[:, :1].expand(40, 56)):
        check_bwd(40, 64, 56, BF16, dy=d)
        check_bwd(40, 64, 56, BF16, "gelu", dy=d)
    w = _rand(gen, (100, 64), BF16)
    check_fwd(9, 100, 64, BF16, weight=w.t())
    check_fwd(9, 32, 100, BF16, weight=w[:, 16:48])
    x3 = _rand(gen, (2, 3, 5, 64), BF16)
    y, _ = ops.linear_act_fwd(x3, w, None, None, "none", False)
    assert torch.equal(y.reshape(30, 100), ops.linear_act_fwd(x3.reshape(30, 64), w, None, None, "none", False)[0])


@gpu
@pytest.mark.parametrize("M,K,N", [(1, 64, 16), (70, 72, 90), (3000, 192, 2000)])
def test_nan_and_infinity_stay_in_their_rows_and_columns(M, K, N):
    """A bad row of x, a bad row of the weight: only their results, through every tile's edges (what lies past M, N and K must not come in)."""
    gen = torch.Generator(device=DEV).manual_seed(5)
    x, w = _rand(gen, (M, K), BF16), _rand(gen, (N, K), BF16)
    clean, _ = ops.linear_act_fwd(x, w, None, None, "gelu", False)
    bw = w.clone()
    bw[N // 2, K - 1] = float("nan")
    y, _ = ops.linear_act_fwd(x, bw, None, None, "gelu", False)
    cols = [n for n in range(N) if n != N // 2]
    assert torch.isnan(y[:, N // 2]).all() and torch.equal(y[:, cols], clean[:, cols])
    if M > 1:
        bx = x.clone()
        bx[M // 2, 0] = float("nan")
        y, _ = ops.linear_act_fwd(bx, w, None, None, "gelu", False)
        rows = [m for m in range(M) if m != M // 2]
        assert torch.isnan(y[M // 2]).all() and torch.equal(y[rows], clean[rows])
        dx, dw, db = ops.linear_act_bwd(bx[:, :1].expand(M, N).contiguous(), x, w, None, "none", None, "none", True, True, True, F32)
        assert torch.isnan(dx[M // 2]).all() and torch.isfinite(dx[rows].float()).all() and torch.isnan(dw).all()


@gpu
def test_activations_at_the_ends():
    """Large arguments, zeros, infinities and NaN through each activation and its derivative (K = 1, weight 1: z = x)."""
    v = [0.0, -0.0, 1e-4, -1e-4, 0.5, -0.5, 3.0, -3.0, 6.0, -6.0, 12.0, -12.0, 40.0, -40.0, 1e4, -1e4, float("inf"), float("nan")]
    x = torch.tensor(v, device=DEV, dtype=BF16).view(-1, 1)
    one = torch.ones((1, 1), device=DEV, dtype=BF16)
    for act in ACTS:
        y, z = ops.linear_act_fwd(x, one, None, None, act, True)
        assert torch.equal(z[:-1], x[:-1]) and torch.isnan(z[-1])
        want = ref.act(x.double(), act)
        ref.close(y, want, ref.ACT_ERR, act)
        finite = x[:16]
        dx, _, _ = ops.linear_act_bwd(torch.ones_like(finite), torch.ones_like(finite), one, finite, act if act != "none" else "relu", None, "none",
                                      True, False, False, BF16)
        ref.close(dx, ref.act_grad(finite.double(), act if act != "none" else "relu"), ref.ACT_ERR + 2 ** -8 * 1.2, act)


@gpu
def test_the_same_bits_every_time():
    gen = torch.Generator(device=DEV).manual_seed(6)
    x, w, dy = _rand(gen, (5000, 520), BF16), _rand(gen, (640, 520), BF16), _rand(gen, (5000, 640), BF16)
    y0, _ = ops.linear_act_fwd(x, w, None, None, "silu", False)
    g0 = ops.linear_act_bwd(dy, x, w, None, "none", None, "none", True, True, True, F32)
    for _ in range(3):
        assert torch.equal(ops.linear_act_fwd(x, w, None, None, "silu", False)[0], y0)
        assert all(torch.equal(a, b) for a, b in zip(ops.linear_act_bwd(dy, x, w, None, "none", None, "none", True, True, True, F32), g0))


def test_the_reference_derivatives_against_differences():
    """act_grad of tests/block_reference.py is the derivative of its act: central differences in 64 bits."""
    z = torch.linspace(-7, 7, 1401, dtype=torch.float64) + 0.003
    for act in ACTS:
        num = (ref.act(z + 1e-5, act) - ref.act(z - 1e-5, act)) / 2e-5
        assert (num - ref.act_grad(z, act)).abs().max() < 1e-9, act


@gpu
def test_refusals():
    x, w = torch.randn((4, 64), device=DEV).to(BF16), torch.randn((32, 64), device=DEV).to(BF16)
    dy = torch.randn((4, 32), device=DEV).to(BF16)
    fwd, bwd = ops.linear_act_fwd, ops.linear_act_bwd
    with pytest.raises(ValueError):
        fwd(x, w, None, None, "tanh", False)
    with pytest.raises(ValueError):
        bwd(dy, x, w, None, "none", None, "swish", True, True, True, F32)
    for call in (lambda: fwd(x.float(), w.float(), None, None, "none", False), lambda: fwd(x, w.half(), None, None, "none", False),
                 lambda: fwd(x[:, :32], w, None, None, "none", False), lambda: fwd(x, w.view(32, 64, 1), None, None, "none", False),
                 lambda: fwd(x, w, dy[0, :31], None, "none", False), lambda: fwd(x, w, None, dy[:3], "none", False),
                 lambda: fwd(x, w, None, dy.half(), "none", False), lambda: fwd(x, w.cpu(), None, None, "none", False),
                 lambda: bwd(dy[:3], x, w, None, "none", None, "none", True, True, True, F32),
                 lambda: bwd(dy.float(), x, w, None, "none", None, "none", True, True, True, F32),
                 lambda: bwd(dy, x, w, None, "gelu", None, "none", True, True, True, F32),
                 lambda: bwd(dy, x, w, dy, "none", None, "none", True, True, True, F32),
                 lambda: bwd(dy, x, w, None, "none", None, "gelu", True, True, True, F32),
                 lambda: bwd(dy, x, w, None, "none", x, "none", True, True, True, F32),
                 lambda: bwd(dy, x, w, None, "none", x[:3], "gelu", True, True, True, F32),
                 lambda: bwd(dy, x, w, None, "none", None, "none", True, True, True, F16)):
        with pytest.raises(RuntimeError):
            call()


@gpu
@pytest.mark.parametrize("M,N", [(1, 8), (3, 13), (64, 2048), (333, 1001), (20000, 40), (5000, 2311), (9, 9000)])
@pytest.mark.parametrize("dt", [BF16, F16], ids=IDS.get)
def test_the_bias_gradient_is_the_sum_before_rounding(M, N, dt):
    """With an activation, dbias in fp32 is within the fp32 sums' bound, which the sum of a rounded dz is not; rows as they lie in
    a larger tensor, too."""
    gen = torch.Generator(device=DEV).manual_seed(M + N)
    x, w = _rand(gen, (M, 16), dt), _rand(gen, (N, 16), dt)
    wide, pre = _rand(gen, (M, N + 5), dt), _rand(gen, (M, N), dt)
    for dy in (wide[:, :N].contiguous(), wide[:, 2:N + 2]):
        for act in ("gelu", "silu", "relu"):
            db = ops.linear_act_bwd(dy, x, w, pre, act, None, "none", False, False, True, F32)[2]
            terms = dy.double() * ref.act_grad(pre.double(), act)
            ref.close(db, terms.sum(0), (M + 8) * ref.E * terms.abs().sum(0) + ref.ACT_ERR * dy.double().abs().sum(0), act)
            full = ops.linear_act_bwd(dy, x, w, pre, act, None, "none", True, True, True, F32)
            assert torch.equal(full[2], db)


@gpu
@pytest.mark.parametrize("M,K,N", [(1, 8, 8), (9, 117, 128), (33, 64, 64), (70, 200, 72), (197, 384, 384), (394, 768, 768), (985, 384, 1536), (640, 1000, 77),
                                   (300, 301, 303), (61, 1537, 63)])
@pytest.mark.parametrize("dt", [BF16, F16], ids=IDS.get)
def test_small_backward_products_together(M, K, N, dt):
    """Both products of a small layer go out in one launch: their results, with every epilogue, and in fp32."""
    for act, in_act in (("none", "none"), ("none", "gelu"), ("relu", "silu")):
        for grad in (F32, dt):
            check_bwd(M, K, N, dt, act, in_act, grad)
    check_bwd(M, K, N, dt, "none", "gelu_tanh", dt, parts=(True, True, False))


# sizes (M rows, columns of the result, terms of the sum) that take the persistent 160- and 256-high tiles (5 and 6 of the launchers'
# table) whatever their epilogue: a tile for each CU, a remainder of 8 terms; and two tiles and whole slabs
LARGE = {5: [(2624, 3592, 264), (5264, 1544, 264)], 6: [(4736, 2824, 264), (6144, 4096, 512)]}


@gpu
@pytest.mark.parametrize("tile", sorted(LARGE))
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dt", [BF16, F16], ids=IDS.get)
def test_large_tiles(tile, act, dt):
    from deep_optimization_amd import _lib

    taken = []
    for M, N, K in LARGE[tile]:
        taken += [_lib.lib().dopt_linear_tile(0, M, N, K, 0), _lib.lib().dopt_linear_tile(1, M, K, N, 0)]
        check_fwd(M, K, N, dt, act, bias=dt, pre=True, res=dt)
        check_fwd(M, K, N, dt, act, bias=F32)
        check_bwd(M, N, K, dt, "none", act, parts=(True, False, False))
    assert taken.count(tile) >= 2, taken


@gpu
@pytest.mark.parametrize("dt", [BF16, F16], ids=IDS.get)
def test_the_128_high_tiles_with_a_remainder(dt):
    check_fwd(1000, 776, 1032, dt, bias=None)


@gpu
@pytest.mark.parametrize("dt", [BF16, F16], ids=IDS.get)
def test_large_tiles_cut_rows_that_end_inside_a_chunk(dt):
    """Rows of 261 (and 515) in a pitch of whole chunks, NaN in what lies between them."""
    gen = torch.Generator(device=DEV).manual_seed(8)
    for M, N, K in ((2624, 3592, 261), (4736, 2824, 261), (6144, 4096, 515), (300, 200, 77), (1000, 1032, 773), (40, 64, 13)):
        pitch = (K + 7) // 8 * 8
        x, w = _rand(gen, (M, pitch), dt), _rand(gen, (N, pitch), dt, K ** -0.5)
        x[:, K:], w[:, K:] = float("nan"), float("nan")
        check_fwd(M, K, N, dt, "none", bias=None, x=x[:, :K], weight=w[:, :K])
        dy = _rand(gen, (M, pitch), dt)
        dy[:, K:] = float("nan")
        check_bwd(M, N, K, dt, parts=(True, False, False), dy=dy[:, :K])


@gpu
def test_past_32_bit_element_offsets():
    """x and dx of more than 2^31 elements: the last rows' results, and a weight gradient to which only the last row gives."""
    M, K, N = 2_800_001, 768, 64
    gen = torch.Generator(device=DEV).manual_seed(9)
    x = torch.zeros((M, K), device=DEV, dtype=BF16)
    x[-300:] = _rand(gen, (300, K), BF16)
    w, dy = _rand(gen, (N, K), BF16, K ** -0.5), _rand(gen, (M, N), BF16)
    y, pre = ops.linear_act_fwd(x, w, None, None, "gelu", True)
    wy, wz, ty, tz = ref.linear_fwd(x[-300:], w, None, None, "gelu")
    ref.close(y[-300:], wy, ty, "y")
    ref.close(pre[-300:], wz, tz, "pre")
    assert not y[:-300].any()
    x[:-1] = 0
    dx, dw, db = ops.linear_act_bwd(dy, x, w, None, "none", x, "relu", True, True, True, F32)
    rows = dy[-300:].double() @ w.double()
    assert not dx[:-1].any()
    ref.close(dx[-1:], rows[-1:] * (x[-1:] > 0), (N + 8) * ref.E * (dy[-1:].double().abs() @ w.double().abs()), "dx")
    ref.close(dw, dy[-1:].double().t() @ x[-1:].double(), 0.0, "dweight")
    ref.close(db, dy.double().sum(0), (M + 8) * ref.E * dy.double().abs().sum(0), "dbias")
    del x, dx
    dz = ops.linear_act_bwd(torch.ones((M, K), device=DEV, dtype=BF16), torch.zeros((M, 8), device=DEV, dtype=BF16),
                            torch.zeros((K, 8), device=DEV, dtype=BF16), torch.ones((M, K), device=DEV, dtype=BF16), "relu", None, "none",
                            False, False, True, F32)[2]
    assert (dz == M).all()  # (sums of ones, exact in fp32)
