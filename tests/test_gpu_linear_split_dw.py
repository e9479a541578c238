"""The weight gradient's kernels that split the sum, in fp16 and bf16: every tile (128 x 128, 128 x 256, 256 x 256), one split that writes
the result itself and every width of the join, fp32 and 16-bit results, with the bias's gradient and without."""
import pytest
import torch

import deep_optimization_amd  # noqa: F401
from deep_optimization_amd import _lib
from tests.test_gpu_linear_act import check_bwd

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
SPLIT = 100  # dopt_linear_tile's answer for them
# (M rows, K in, N out features) by (tile rows, tile columns, splits): the smallest of a grid of sizes that take it
SIZES = {(128, 128, "5-8"): (9000, 72, 4096), (128, 128, "9-16"): (6000, 72, 2048), (128, 128, ">16"): (3008, 72, 72),
         (128, 256, "5-8"): (6000, 4096, 130), (128, 256, "9-16"): (6000, 768, 256), (128, 256, ">16"): (3008, 256, 72),
         (256, 256, "1"): (33, 5000, 1544), (256, 256, "2-4"): (4001, 2056, 2048), (256, 256, "5-8"): (6000, 12000, 130),
         (256, 256, "9-16"): (20000, 72, 5000)}


def _taken(M, K, N):
    """(tile rows, tile columns, splits) from the sizes and the workspace that they ask for; None: another kernel's."""
    L = _lib.lib()
    if L.dopt_linear_tile(2, M, N, K, 0) != SPLIT:
        return None
    floats = L.dopt_linear_weight_grad_workspace_floats(M, N, K)
    splits = floats // (N * K + N) if floats else 1
    rows = 128 if -(-N // 256) * -(-K // 256) <= 16 else 256
    cols = 128 if rows == 128 and 0 < K % 256 <= 128 else 256
    return rows, cols, "1" if splits == 1 else "2-4" if splits <= 4 else "5-8" if splits <= 8 else "9-16" if splits <= 16 else ">16"


@pytest.mark.parametrize("key", SIZES, ids=["x".join(map(str, k[:2])) + "_" + k[2] for k in SIZES])
def test_the_sizes_take_what_they_are_here_for(key):
    """With 256 CUs, which is what the choice assumes without a GPU and what the part has."""
    assert _taken(*SIZES[key]) == key


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("key", SIZES, ids=["x".join(map(str, k[:2])) + "_" + k[2] for k in SIZES])
def test_split_weight_gradients(key, dt):
    M, K, N = SIZES[key]
    assert _taken(M, K, N) == key
    for grad in (F32, dt):
        for bias in (True, False):
            check_bwd(M, K, N, dt, grad=grad, parts=(False, True, bias))
