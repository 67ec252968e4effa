"""Calls of the layer operators that once went wrong."""
import pytest
import torch

import layer_plain as plain
from test_gpu_layer_ops import BF16, F32, around, padded, rand

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from gateddeltanet_b200 import build
    build.build()
    from gateddeltanet_b200 import ops
    return ops


@pytest.mark.parametrize("starts", [[0, 2, 1, 400], [2, 1, 400], [0, 1, 0, 400], [0, 2, 0, 2, 400], [0, 200, 199, 201, 400], [400, 2, 1, 400], [0, 400]],
                         ids=str)
@pytest.mark.parametrize("width", [2, 4])
@pytest.mark.parametrize("x_type", [BF16, F32], ids=str)
def test_conv_decreasing_starts_of_wide_rows(ops, starts, width, x_type):
    """Tiles of four tokens and more, in which the walk comes to a sequence behind its begin: the call stays in its tensors
    and ends, and the next call is right. (tests/test_conv_walk_cpu.py holds the indices themselves.)"""
    tokens, channels = 400, 6144
    x, weight = rand(tokens, channels, dtype=x_type), rand(channels, width, seed=2)
    out, big = padded(torch.zeros(tokens, channels, device="cuda", dtype=x_type), 5, 0)
    tails, pool = padded(rand(len(starts) - 1, width - 1, channels), 2, 0, 0)
    ops.short_conv(x, weight, tails, starts=torch.tensor(starts, dtype=torch.int32, device="cuda"), out=out)
    torch.cuda.synchronize()
    assert around(big, out) and around(pool, tails)
    index = torch.tensor(sorted(starts), dtype=torch.int32, device="cuda")
    tails.copy_(rand(len(starts) - 1, width - 1, channels, seed=3))
    want, after, off = plain.conv(x, weight, tails, starts=index)
    plain.check(ops.short_conv(x, weight, tails, starts=index, out=out), want, off)
    assert torch.equal(tails.cpu().double(), after) and around(big, out) and around(pool, tails)
