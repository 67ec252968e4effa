"""Calls of the layer operators that once went wrong."""
import importlib.util
import os

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


SILU_RANGES = [(-87, -40), (-40, -15), (-15, -6), (-6, -3), (-3, 0), (0, 3), (3, 40)]


def silu_is(x, got):
    """FP32 results: 2^t by ex2.approx 4 U, its correction 2 U, the sum and the product U each, 1 / x by rcp.approx 2 U less what
    the sum's own slope takes from the errors of 2^t, in all 9 U at most; and ln 2, rounded to 2.8e-9, counts by |x|."""
    x = x.cpu().double()
    want = plain.silu(x)
    off = (got.cpu().double() - want).abs()
    assert bool((off <= (9 + x.abs() / 20) * plain.U * want.abs()).all())


@pytest.mark.parametrize("low,high", SILU_RANGES)
def test_silu_of_far_values(ops, low, high):
    """To the last bits at both ends, in every operator that has it."""
    x = (torch.rand(1 << 12, 64, generator=torch.Generator().manual_seed(3)) * (high - low) + low).cuda()
    itself = torch.tensor([[0.0, 1.0]], device="cuda").repeat(64, 1)
    silu_is(x, ops.short_conv(x, itself, torch.zeros(len(x), 1, 64, device="cuda")))
    silu_is(x, ops.short_conv(x, itself, torch.zeros(1, 1, 64, device="cuda"), starts=torch.tensor([0, len(x)], dtype=torch.int32, device="cuda")))
    short = x.to(BF16)
    diagonal = torch.eye(64, device="cuda", dtype=BF16)
    for tokens in (5, 4000):  # either kernel: sums with one term
        silu_is(short[:tokens], ops.linear(short[:tokens], diagonal, activation="silu", dtype=F32))
        twice = torch.cat([diagonal, torch.zeros_like(diagonal)])
        silu_is(short[:tokens], ops.linear(short[:tokens], twice, bias=torch.cat([torch.zeros(64), torch.ones(64)]).cuda(), activation="swiglu", dtype=F32))
    ones = torch.ones_like(x)
    assert bool((ops.rms_norm(ones, eps=0.0) == 1).all())
    silu_is(x, ops.rms_norm(ones, gate=x, eps=0.0))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_silu_past_its_range(ops, dtype):
    """Where e^-x is no FP32 number any more: the value itself above, nothing below, and what is not finite as the formula has it."""
    x = torch.tensor([87.5, 88, 89, 128, 1e4, 1e30, 2.3e38, 3e38, float("inf"), -87.5, -88, -89, -104, -128, -1e4, -1e30, -2.3e38, -3e38,
                      float("-inf"), float("nan"), 0.0, -0.0]).to(dtype).cuda()[None].repeat(8, 1).contiguous()
    n = x.shape[1]
    itself, index = torch.tensor([[0.0, 1.0]], device="cuda").repeat(n, 1), torch.tensor([0, 8], dtype=torch.int32, device="cuda")
    rows = [ops.short_conv(x, itself, torch.zeros(8, 1, n, device="cuda")), ops.short_conv(x, itself, torch.zeros(1, 1, n, device="cuda"), starts=index),
            ops.rms_norm(torch.ones_like(x), gate=x, eps=0.0)]
    zero, bias = torch.zeros(20, 64, device="cuda", dtype=BF16), x[0].contiguous()
    for tokens in (3, 20):
        rows.append(ops.linear(zero[:tokens], torch.zeros(n, 64, device="cuda", dtype=BF16), bias=bias, activation="silu", dtype=dtype))
    # in a sequence the infinity of the token before meets the weight 0, which is NaN
    assert bool(rows[1][1:, 8].isnan().all())
    rows[1][1:, 8] = float("inf")
    for y in rows:
        for row in y:
            assert torch.equal(row[:9], x[0, :9])
            assert bool((row[9:18].abs() <= 1e-35).all()) and bool(row[18:20].isnan().all()) and bool((row[20:] == 0).all())


def test_silu_of_16_bits(ops):
    """Half a step of BF16 and what comes before it; one token at a time gives the bits of many."""
    x = ((torch.rand(1 << 12, 64, generator=torch.Generator().manual_seed(3)) - 0.7) * 120).cuda().to(BF16)
    itself = torch.tensor([[0.0, 1.0]], device="cuda").repeat(64, 1)
    got = ops.short_conv(x, itself, torch.zeros(1, 1, 64, device="cuda"), starts=torch.tensor([0, len(x)], dtype=torch.int32, device="cuda"))
    want = plain.silu(x.cpu().double())
    assert bool(((got.cpu().double() - want).abs() <= (2.0 ** -8 + 2.0 ** -17) * want.abs()).all())
    assert torch.equal(ops.short_conv(x, itself, torch.zeros(len(x), 1, 64, device="cuda")), got)


def gelu_is(x, got):
    """Results of gelu(x), x exact: FP32 (20 + x^2 / 40) U, as gdn_linear.h counts; 16 bits half a step more."""
    x, dtype = x.cpu().double(), got.dtype
    want = 0.5 * x * torch.special.erfc(-x * 0.5 ** 0.5)
    off = (20 + x * x / 40) * plain.U + (plain.half_step(dtype) if dtype != F32 else 0)
    assert bool(((got.cpu().double() - want).abs() <= off * want.abs()).all())


@pytest.mark.parametrize("low,high", [(-13, -8), (-8, -5), (-5, -3), (-3, -1), (-1, 0), (0, 1), (1, 8)])
@pytest.mark.parametrize("outputs", [512, 511])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_gelu_keeps_its_bits_below_zero(ops, low, high, outputs, dtype):
    """Of biases alone, in each kernel: a few tokens, tiles, two CTAs a tile; results in pieces and value by value."""
    x = ((torch.rand(outputs, generator=torch.Generator().manual_seed(3))) * (high - low) + low).cuda()
    weight = torch.zeros(outputs, 64, device="cuda", dtype=BF16)
    for tokens in (1, 16, 20, 300, 3000):
        y = ops.linear(torch.zeros(tokens, 64, device="cuda", dtype=BF16), weight, bias=x, activation="gelu", dtype=dtype)
        gelu_is(x.expand(tokens, -1), y)


def test_gelu_past_its_range(ops):
    x = torch.tensor([13.5, 20, 1e5, 1e30, 3e38, float("inf"), -13.5, -20, -1e5, -1e30, -3e38, float("-inf"), float("nan"), 0.0, -0.0, 1e-40]).cuda()
    weight = torch.zeros(16, 64, device="cuda", dtype=BF16)
    for tokens in (3, 40):
        for row in ops.linear(torch.zeros(tokens, 64, device="cuda", dtype=BF16), weight, bias=x, activation="gelu", dtype=F32):
            assert torch.equal(row[:6], x[:6]) and bool((row[6:11].abs() <= 1e-35).all())
            assert bool(row[11:13].isnan().all()) and bool((row[13:15] == 0).all()) and 0 <= float(row[15]) <= 6e-41


@pytest.mark.parametrize("tokens", [40, 300, 2000])
@pytest.mark.parametrize("inputs", [256, 768, 1024, 2048, 2600, 4096, 5632])
@pytest.mark.parametrize("activation", [None, "silu", "swiglu"])
def test_linear_keeps_its_bits(ops, tokens, inputs, activation):
    """FP32 results of BF16 in the 2-norm, as the header has it: under 2^-21 up to 2560 inputs and under 2^-20 beyond. (What
    FP32 sums one after the other of n products lose, half steps of U / sqrt 3 of partial sums that grow like a root, is
    U sqrt(n / 6): 2^-20 for 1536.)"""
    x, w = rand(tokens, inputs, dtype=BF16), (rand(1000 * (2 if activation == "swiglu" else 1), inputs, seed=2) * inputs ** -0.5).bfloat16()
    want, _ = plain.linear(x, w, activation=activation)
    got = ops.linear(x, w, activation=activation, dtype=F32).cpu().double()
    assert float((got - want).norm() / want.norm()) <= (2.0 ** -21 if inputs <= 2560 else 2.0 ** -20)


def test_norm_of_heads_side_by_side(ops):
    """x, gate, out and the residual of each head next to one another: results between the inputs, and in their place."""
    big = rand(30, 4, 4, 128, dtype=BF16)
    x, gate, out, residual = big.unbind(2)
    want, h = plain.norm(x, None, residual, gate)
    kept = x.clone(), gate.clone()
    assert ops.rms_norm(x, residual=residual, gate=gate, out=out) is out
    plain.check(out, want, plain.norm_error(gate) * want.abs(), "out")
    plain.check(residual, h, plain.U * h.abs(), "residual")
    assert torch.equal(x, kept[0]) and torch.equal(gate, kept[1])
    want, _ = plain.norm(x, None, None, gate)
    ops.rms_norm(x, gate=gate, out=x)
    plain.check(x, want, plain.norm_error(gate) * want.abs(), "in place")
    assert torch.equal(gate, kept[1])


def test_what_the_kernel_before_wrote(ops):
    """Calls whose launches overlap read weights, bounds and slots that were written just before, again and again in the same
    buffers, by a copy or by an operator: as with a wait after every call."""
    x, xs = rand(200, 512, dtype=BF16), [rand(n, 512, seed=2, dtype=BF16) for n in (3, 12)]
    bounds = [torch.tensor(b, dtype=torch.int32, device="cuda") for b in ([0, 50, 200], [0, 0, 10], [3, 150, 170])]
    places = [torch.tensor(b, dtype=torch.int32, device="cuda") for b in ([0, 1], [2, 0], [1, -1])]
    taps, flags = [rand(512, 4, seed=3 + i) for i in range(3)], [torch.tensor(b, device="cuda") for b in ([True, False], [False, False], [True, True])]
    left = rand(1000, 512, seed=9, dtype=BF16) * 0.05

    def chain(wait):
        starts, slots, fresh, weight, w = (torch.zeros_like(t) for t in (bounds[0], places[0], flags[0], taps[0], left))
        tails, results = torch.zeros(3, 3, 512, device="cuda"), []

        def after(y=None):
            if y is not None:
                results.append(y)
            if wait:
                torch.cuda.synchronize()
        for i in range(30):
            after(ops.rms_norm(x))
            for to, by in ((starts, bounds), (slots, places), (fresh, flags), (weight, taps)):
                to.copy_(by[i % 3])
                after()
            after(ops.short_conv(x, weight, tails, starts=starts, slots=slots, fresh=fresh))
            ops.linear(left, left[i:i + 512], activation="silu" if i % 2 else None, out=w)  # the next products' weight
            after()
            for a in xs:
                after(ops.linear(a, w, dtype=F32))
            after(ops.linear(x, w))
        return results + [tails]
    want = chain(True)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(chain(False), want))


@pytest.mark.parametrize("eight_bits", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("hidden,intermediate", [(100, None), (77, 71), (4, None)])
def test_server_of_any_width(ops, hidden, intermediate, eight_bits):
    """Hidden sizes whose rows are no multiples of 16 bytes: as they ran before the layers were made of operators."""
    spec = importlib.util.spec_from_file_location("serve", os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "serve.py"))
    serve = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(serve)
    model = serve.Model(vocab=103, hidden=hidden, layers=2, heads=2, head_dim=64, seed=3, intermediate=intermediate, eight_bits=eight_bits)
    prompts = [[5], list(range(70)), [1, 2, 3]]
    table, lens, states = serve.generate(model, prompts, 4)
    assert lens.tolist() == [5, 74, 7] and all(bool(s.isfinite().all()) for s in states)
    assert all(table[i, :len(p)].tolist() == p for i, p in enumerate(prompts))


def test_conv_by_pieces_of_fp32(ops):
    """A prompt at once, in pieces and token by token: the same bits, also where silu is far from 0."""
    x = (torch.rand(300, 512, generator=torch.Generator().manual_seed(1)) * 120 - 90).cuda()
    weight = torch.tensor([0.0, 0.3, 0.0, 1.0], device="cuda").repeat(512, 1)
    index = lambda *s: torch.tensor(s, dtype=torch.int32, device="cuda")  # noqa: E731
    whole, tails = torch.zeros(1, 3, 512, device="cuda"), torch.zeros(1, 3, 512, device="cuda")
    want = ops.short_conv(x, weight, whole, starts=index(0, 300))
    parts, at = [], 0
    for n in (1, 2, 100, 3, 100):
        parts.append(ops.short_conv(x[at:at + n], weight, tails, starts=index(0, n)))
        at += n
    parts += [ops.short_conv(x[t:t + 1], weight, tails) for t in range(at, 300)]
    assert torch.equal(torch.cat(parts), want) and torch.equal(tails, whole)


@pytest.mark.parametrize("activation", ["silu", "gelu", "swiglu"])
def test_activations_have_the_same_bits_in_every_kernel(ops, activation):
    """Of biases alone: a few tokens (one value at a time), tiles and divided sums (pairs of values)."""
    outputs = 500
    rows = outputs * (2 if activation == "swiglu" else 1)
    bias = ((torch.rand(rows, generator=torch.Generator().manual_seed(1)) - 0.6) * 60).cuda()
    weight = torch.zeros(rows, 2048, device="cuda", dtype=BF16)
    want = None
    for tokens in (1, 16, 20, 100, 600):
        y = ops.linear(torch.zeros(tokens, 2048, device="cuda", dtype=BF16), weight, bias=bias, activation=activation, dtype=F32)
        want = y[:1] if want is None else want
        assert torch.equal(y, want.expand(tokens, -1))
