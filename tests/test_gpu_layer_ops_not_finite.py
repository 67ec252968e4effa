"""What is not finite in the layer operators' inputs: results are those of the
formula in IEEE arithmetic where it meets them, and as ever elsewhere."""
import pytest
import torch

import layer_plain as plain
from test_gpu_layer_ops import BF16, F32, operands, rand

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module")
def ops():
    from gateddeltanet_b200 import build
    build.build()
    from gateddeltanet_b200 import ops
    return ops


@pytest.mark.parametrize("tokens", [1, 5, 16, 100, 700])
@pytest.mark.parametrize("outputs", [300, 301])
@pytest.mark.parametrize("activation", [None, "silu", "gelu", "swiglu"])
def test_linear_with_infinities(ops, tokens, outputs, activation):
    """In x, W, the bias and the residual; a product of infinity and 0, and a sum of two infinities, are NaN."""
    rows = outputs * (2 if activation == "swiglu" else 1)
    a = operands(tokens, 1032, rows, False)
    bias, residual = rand(rows, seed=3), rand(tokens, outputs, seed=4)
    a["x"][0, 17] = INF
    a["weight"][7, 500], a["weight"][9, 1031], a["weight"][11, 17] = INF, -INF, 0.0
    bias[20], bias[21], bias[22] = INF, -INF, NAN
    residual[tokens - 1, 30], residual[0, 31], residual[tokens // 2, 32] = INF, -INF, NAN
    want, off = plain.linear(**a, bias=bias, activation=activation, residual=residual)
    off = torch.nan_to_num(off, nan=0.0, posinf=0.0)  # counted where results are finite, whose operands are
    assert bool(want[0].isnan().any()) and bool(want.isinf().any()) and bool(want.isfinite().any() if tokens > 1 else True)
    for dtype in (F32, BF16):
        plain.check(ops.linear(**a, bias=bias, activation=activation, residual=residual, dtype=dtype), want, off, str(dtype))


@pytest.mark.parametrize("tokens", [1, 16, 100, 700])
@pytest.mark.parametrize("activation", [None, "gelu", "swiglu"])
def test_linear_of_8_bits_with_scales_that_are_not_finite(ops, tokens, activation):
    rows = 300 * (2 if activation == "swiglu" else 1)
    a = operands(tokens, 1040, rows, True)
    a["x_scales"][tokens // 2], a["weight_scales"][5], a["weight_scales"][6] = INF, NAN, INF
    # the product of the scales meets the sum, not its terms, whose infinities would be NaN together
    finite = {**a, "x_scales": a["x_scales"].nan_to_num(posinf=1.0), "weight_scales": a["weight_scales"].nan_to_num(nan=1.0, posinf=1.0)}
    _, off = plain.linear(**finite, activation=activation)
    y = (a["x"].cpu().double() @ a["weight"].cpu().double().T) * (a["x_scales"].cpu().double()[:, None] * a["weight_scales"].cpu().double())
    if activation == "swiglu":
        y, up = y.chunk(2, 1)
        y = plain.silu(y) * up
    elif activation == "gelu":
        y = 0.5 * y * (1 + torch.erf(y * 0.5 ** 0.5))
    assert bool(y.isinf().any()) and bool(y.isnan().any()) and bool(y.isfinite().any() if tokens > 1 else True)
    plain.check(ops.linear(**a, activation=activation, dtype=F32), y, off)


@pytest.mark.parametrize("channels", [64, 61])
@pytest.mark.parametrize("x_type,tail_type", [(BF16, F32), (BF16, BF16), (F32, F32)], ids=str)
@pytest.mark.parametrize("width", [2, 4])
@pytest.mark.parametrize("activation", [None, "silu"])
def test_conv(ops, channels, x_type, tail_type, width, activation):
    """A channel's values reach as many tokens as it has taps, in its own sequence, and its slot; a fresh sequence does not see
    its slot's old content."""
    starts = torch.tensor([0, 5, 6, 90, 90, 200], dtype=torch.int32, device="cuda")
    x, weight = rand(200, channels, dtype=x_type), rand(channels, width, seed=2)
    tails = rand(7, width - 1, channels, seed=3).to(tail_type)
    x[4, 3], x[5, 4], x[40, 5], x[41, 6], x[89, 7], x[199, 8], x[100, 60] = NAN, INF, -INF, NAN, INF, -INF, INF
    tails[0, -1, 10], tails[1, 0, 11], tails[2, -1, 12], tails[3, 0, 13], tails[6] = INF, NAN, -INF, NAN, NAN
    weight[5, 0], weight[20, -1] = 0.0, INF
    slots = torch.tensor([0, 1, 2, 3, 6], dtype=torch.int32, device="cuda")
    fresh = torch.tensor([False, False, False, False, True], device="cuda")
    args = dict(activation=activation, starts=starts, slots=slots, fresh=fresh)
    want, after, off = plain.conv(x, weight, tails, **args)
    off = torch.nan_to_num(off, nan=0.0, posinf=0.0)
    got = ops.short_conv(x, weight, tails, **args)
    plain.check(got, want, off, "out")
    assert torch.equal(tails.cpu().double().nan_to_num(nan=7e99), after.nan_to_num(nan=7e99))
    # one token more of each
    x = rand(5, channels, seed=6, dtype=x_type)
    x[2, 30] = NAN
    args = dict(activation=activation, slots=slots)
    want, after, off = plain.conv(x, weight, tails, **args)
    plain.check(ops.short_conv(x, weight, tails, **args), want, torch.nan_to_num(off, nan=0.0, posinf=0.0), "one more")
    assert torch.equal(tails.cpu().double().nan_to_num(nan=7e99), after.nan_to_num(nan=7e99))


@pytest.mark.parametrize("dim", [256, 77])
def test_norm(ops, dim):
    """In the weight, the gate and the residual: a weight's column, a gate's value, a row."""
    x, gate, weight, residual = rand(9, dim), rand(9, dim, seed=2), rand(dim, seed=3), rand(9, dim, seed=4)
    weight[3], weight[4], gate[2, 5], gate[3, 6], residual[7, 8] = NAN, INF, NAN, -INF, INF
    want, h = plain.norm(x, weight, residual, gate)
    got = ops.rms_norm(x, weight, residual=residual, gate=gate)
    plain.check(residual, h, plain.U * h.abs(), "residual")
    keep = [i for i in range(9) if i != 7]
    plain.check(got[keep], want[keep], torch.nan_to_num(plain.norm_error(gate) * want[keep].abs(), nan=0.0, posinf=0.0))
    assert bool(got[7].isnan().all())
