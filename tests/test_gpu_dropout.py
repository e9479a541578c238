"""act_lib::dropout_add_fwd / dropout_bwd: the mask bit for bit against Philox4x32-10 computed on the host
(tests/block_reference.py; its generator against published vectors below), the values bit for bit against the same two
fp32 operations in torch."""
import numpy as np
import pytest
import torch

import deep_optimization_amd  # noqa: F401
from tests import block_reference as ref

DEV = "cuda"
ops = torch.ops.act_lib
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
IDS = {F32: "f32", F16: "f16", BF16: "bf16"}
gpu = pytest.mark.gpu


def test_the_reference_generator_against_published_vectors():
    """Random123's known answers for Philox4x32-10."""
    assert ref.philox([0] * 4, [0] * 2) == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    assert ref.philox([0xffffffff] * 4, [0xffffffff] * 2) == [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]
    assert ref.philox([0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344], [0xa4093822, 0x299f31d0]) == \
        [0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1]
    # and the vectorised form against it
    seed, ctr = 0x299f31d0a4093822, 0x0370734413198a2e
    words = ref.philox([3, 0, ctr & 0xffffffff, ctr >> 32], [seed & 0xffffffff, seed >> 32])
    halves = [h for w in words for h in (w & 0xffff, w >> 16)]
    for p in (0.25, 0.5, 0.9):
        assert ref.kept(32, p, seed, ctr)[24:].tolist() == [h >= ref.threshold(p) for h in halves]


def _want(x, residual, p, seed, counter, out_dtype):
    keep = torch.from_numpy(ref.kept(x.numel(), p, seed, counter)).to(x.device).reshape(x.shape)
    y = torch.where(keep, x.float() * torch.tensor(ref.scale(p), dtype=F32, device=x.device), torch.zeros((), device=x.device))
    if residual is not None:
        y = y + residual.float()
    return y.to(out_dtype)


@gpu
@pytest.mark.parametrize("x_dt", [F32, F16, BF16], ids=IDS.get)
@pytest.mark.parametrize("y_dt", [F32, F16, BF16], ids=IDS.get)
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 0.97, 1.0])
def test_every_pair_of_types(x_dt, y_dt, p):
    gen = torch.Generator(device=DEV).manual_seed(1)
    for shape in ((1,), (7,), (8,), (9,), (3, 5, 197), (100, 768)):
        print(f"[dropout] {shape} {x_dt} -> {y_dt} p {p}", flush=True)
        x = torch.randn(shape, generator=gen, device=DEV).to(x_dt)
        r = torch.randn(shape, generator=gen, device=DEV).to(y_dt)
        assert torch.equal(ops.dropout_add_fwd(x, r, p, 11, 5, None), _want(x, r, p, 11, 5, y_dt))
        assert torch.equal(ops.dropout_bwd(x, p, 11, 5, None, y_dt), _want(x, None, p, 11, 5, y_dt))
    assert torch.equal(ops.dropout_add_fwd(x, None, p, 11, 5, None), _want(x, None, p, 11, 5, x_dt))


@gpu
@pytest.mark.parametrize("seed,offset,step", [(0, 0, 0), (1 << 40, 3, 5), (-1, -1, 0), (2 ** 63 - 1, 2 ** 32 - 1, 1), (5, -3, 3), (9, 1 << 50, -(1 << 49))])
def test_seeds_offsets_and_steps_are_64_bits(seed, offset, step):
    x = torch.ones(4000, device=DEV)
    t = torch.tensor([step], dtype=torch.int64, device=DEV)
    want = _want(x, None, 0.3, seed, offset + step, F32)
    assert torch.equal(ops.dropout_add_fwd(x, None, 0.3, seed, offset, t), want)
    if step == 0:
        assert torch.equal(ops.dropout_add_fwd(x, None, 0.3, seed, offset, None), want)


@gpu
def test_the_share_kept_and_the_mean():
    """Over n = 2^24 elements the count kept lies within 6 standard deviations of its expectation, the mean of ones likewise."""
    n = 1 << 24
    x = torch.ones(n, device=DEV)
    for p in (0.05, 0.1, 0.5, 1 / 65536, 0.3 / 65536):
        y = ops.dropout_add_fwd(x, None, p, 77, 0, None).double()
        q = 1 - ref.threshold(p) / 65536
        sd = (n * q * (1 - q)) ** 0.5
        assert abs(float((y != 0).sum()) - n * q) <= 6 * sd
        assert abs(float(y.mean()) - 1) <= 6 * sd / (n * q) + 1e-7


@gpu
def test_dropped_values_leave_nothing():
    """NaN and infinities at dropped places give 0 (or the residual), at kept places themselves."""
    x = torch.full((4096,), float("nan"), device=DEV)
    x[::3] = float("inf")
    keep = torch.from_numpy(ref.kept(4096, 0.5, 3, 0)).to(DEV)
    y = ops.dropout_add_fwd(x, None, 0.5, 3, 0, None)
    assert torch.equal(y[~keep], torch.zeros_like(y[~keep])) and not torch.isfinite(y[keep]).any()
    r = torch.randn(4096, device=DEV)
    assert torch.equal(ops.dropout_add_fwd(x, r, 0.5, 3, 0, None)[~keep], r[~keep])
    assert torch.equal(ops.dropout_add_fwd(x, r, 1.0, 3, 0, None), r)


@gpu
def test_views_strides_and_odd_addresses():
    gen = torch.Generator(device=DEV).manual_seed(2)
    big = torch.randn((64, 200), generator=gen, device=DEV).to(BF16)
    for x in (big[:, 3:100], big.t(), big[::2], big.reshape(-1)[5:5 + 1001]):
        r = torch.randn(x.shape, generator=gen, device=DEV).to(BF16)
        assert torch.equal(ops.dropout_add_fwd(x, r, 0.2, 4, 0, None), _want(x.contiguous(), r, 0.2, 4, 0, BF16))
    assert torch.equal(ops.dropout_add_fwd(big, big[:, :1].expand(64, 200), 0.2, 4, 0, None), _want(big, big[:, :1].expand(64, 200), 0.2, 4, 0, BF16))


@gpu
def test_empty():
    x = torch.empty((0, 768), device=DEV, dtype=BF16)
    assert ops.dropout_add_fwd(x, x, 0.1, 0, 0, None).shape == (0, 768)
    assert ops.dropout_bwd(x, 0.1, 0, 0, None, F32).dtype == F32


@gpu
def test_past_32_bit_element_offsets():
    """2^32 + 1000 bf16 elements: the windows around element 2^32, at the start and at the end."""
    n = (1 << 32) + 1000
    print(f"[dropout] {n} elements", flush=True)
    x = torch.ones(n, device=DEV, dtype=BF16)
    y = ops.dropout_add_fwd(x, None, 0.5, 21, 9, None)
    for start in (0, (1 << 32) - 512, n - 1000):
        idx = np.arange(start // 8, start // 8 + 64)
        want = []
        for i in idx.tolist():
            words = ref.philox([i & 0xffffffff, i >> 32, 9, 0], [21, 0])
            want += [2.0 if h >= 32768 else 0.0 for w in words for h in (w & 0xffff, w >> 16)]
        got = y[start // 8 * 8: start // 8 * 8 + 512].float().cpu().tolist()
        assert got == want[:len(got)], start
    del x, y
    torch.cuda.empty_cache()


@gpu
def test_a_captured_graph_draws_a_new_mask_on_each_replay():
    from deep_optimization_amd.graph import finalize

    x = torch.randn((300, 768), device=DEV).to(BF16)
    step = torch.zeros(1, dtype=torch.int64, device=DEV)
    ops.dropout_add_fwd(x, None, 0.4, 6, 0, step)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        y = ops.dropout_add_fwd(x, None, 0.4, 6, 0, step)
        dx = ops.dropout_bwd(x, 0.4, 6, 0, step, BF16)
    finalize(graph)
    for k in range(4):
        step.fill_(k)
        graph.replay()
        torch.cuda.synchronize()
        want = _want(x, None, 0.4, 6, k, BF16)
        assert torch.equal(y, want) and torch.equal(dx, want), k
        (x.float() @ x.float().t()).sum().item()  # the program's own work between replays


@gpu
def test_refusals():
    x = torch.randn((4, 64), device=DEV)
    for call in (lambda: ops.dropout_add_fwd(x, None, -0.1, 0, 0, None), lambda: ops.dropout_add_fwd(x, None, 1.1, 0, 0, None),
                 lambda: ops.dropout_add_fwd(x, None, float("nan"), 0, 0, None), lambda: ops.dropout_add_fwd(x.double(), None, 0.1, 0, 0, None),
                 lambda: ops.dropout_add_fwd(x, x[:3], 0.1, 0, 0, None), lambda: ops.dropout_add_fwd(x, x.double(), 0.1, 0, 0, None),
                 lambda: ops.dropout_add_fwd(x, None, 0.1, 0, 0, torch.zeros(1, device=DEV)),
                 lambda: ops.dropout_add_fwd(x, None, 0.1, 0, 0, torch.zeros(2, dtype=torch.int64, device=DEV)),
                 lambda: ops.dropout_add_fwd(x, x.cpu(), 0.1, 0, 0, None), lambda: ops.dropout_bwd(x, 0.1, 0, 0, None, torch.int8)):
        with pytest.raises(RuntimeError):
            call()
