"""Calls of the layer operators that once went wrong."""
import pytest
import torch

import layer_plain as plain
from test_gpu_layer_ops import BF16, E4M3, F32, around, check_eight, padded, rand

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


@pytest.mark.parametrize("dim", [2048, 2044, 100, 77, 16384])
@pytest.mark.parametrize("x_type,res_type,out_type", [(BF16, None, BF16), (F32, None, F32), (F32, F32, BF16), (BF16, F32, E4M3), (F32, None, E4M3)],
                         ids=str)
def test_norm_rows_whose_squares_overflow(ops, dim, x_type, res_type, out_type):
    """NaN throughout, the scale too, and nothing in the rows beside them."""
    x = rand(9, dim, dtype=x_type)
    # over FP32's 3.4e38: a square, the sum of dim squares, an infinity, a square
    x[1, dim // 2], x[3], x[5, dim - 1], x[7, 0] = 1e20, -1e19, float("-inf"), 2e19
    residual = None if res_type is None else rand(9, dim, seed=2, dtype=res_type)
    want, h = plain.norm(x, residual=residual)
    got = ops.rms_norm(x, residual=residual, dtype=out_type)
    keep, bad = [0, 2, 4, 6, 8], [1, 3, 5, 7]
    if residual is not None:
        plain.check(residual, h, plain.U * h.abs(), "residual")
    if out_type == E4M3:
        assert bool(got[1][bad].isnan().all()) and bool(got[0].float()[bad].isnan().all())
        check_eight((got[0][keep], got[1][keep]), want[keep], plain.norm_error(None) * want[keep].abs())
        return
    assert bool(got[bad].isnan().all())
    plain.check(got[keep], want[keep], plain.norm_error(None) * want[keep].abs())


def test_norm_of_heads_whose_squares_overflow(ops):
    """A head by itself in 16 bits, its whole token in 8."""
    x = rand(3, 4, 64, dtype=BF16)
    x[1, 2, 5] = 3e19
    y = ops.rms_norm(x).isnan()
    assert bool(y[1, 2].all()) and int(y.sum()) == 64
    y, scales = ops.rms_norm(x, dtype=E4M3)
    assert scales.isnan().tolist() == [False, True, False] and bool(y.float()[1].isnan().all())


def test_norm_by_a_root_off_by_its_rounding(ops):
    """Of 1 + eps, exact in FP32, with all that follows exact: the product in Newton's step is off by U, which counts half, and
    the sum after it by U; errors of the instruction's own value come in squared."""
    one, eps = torch.ones(1, 1, device="cuda"), torch.arange(1, 2 ** 20, 2 ** 10 - 3).double() / 2 ** 20 * 3
    got = torch.cat([ops.rms_norm(one, eps=e) for e in eps.tolist()])[:, 0].cpu().double()
    want = (1 + eps) ** -0.5
    assert float(((got - want).abs() / want).max()) <= 1.51 * plain.U
