"""The layer operators of gateddeltanet_b200/ops.py (rms_norm, linear,
short_conv) against their 64-bit forms (layer_plain.py), which also say how far
roundings may take them."""
import pytest
import torch

import layer_plain as plain

pytestmark = pytest.mark.gpu
F32, BF16, E4M3 = torch.float32, torch.bfloat16, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops():
    from gateddeltanet_b200 import build
    build.build()
    from gateddeltanet_b200 import ops
    return ops


def rand(*shape, seed=1, dtype=F32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def padded(x, *extra, value=7.0):
    """x as a view into a larger tensor (extra elements behind each dimension's end), and that tensor."""
    big = torch.full([n + e for n, e in zip(x.shape, extra)], value, device=x.device).to(x.dtype)
    view = big[tuple(slice(0, n) for n in x.shape)]
    view.copy_(x)
    return view, big


def around(big, view, value=7.0):
    """Whether what is outside the view is as padded() left it."""
    rest = big.float().clone()
    rest[tuple(slice(0, n) for n in view.shape)] = value
    return bool((rest == value).all())


# ---- rms_norm

NORM_SHAPES = [(1, 2048), (3, 1), (5, 7), (2, 8), (7, 64), (130, 100), (9, 1999), (4, 2040), (3, 8192), (2, 8200), (2, 16384),
               (1, 16383), (300, 256), (5, 8, 256), (3, 4, 128), (2, 3, 50), (2, 64, 256), (6, 2, 1000), (1, 12, 7)]


@pytest.mark.parametrize("shape", NORM_SHAPES, ids=str)
@pytest.mark.parametrize("x_type,res_type,out_type", [(BF16, None, BF16), (BF16, F32, BF16), (BF16, BF16, E4M3), (F32, F32, F32),
                                                      (F32, None, E4M3), (F32, BF16, BF16), (BF16, None, F32)], ids=str)
def test_norm(ops, shape, x_type, res_type, out_type):
    gated, weighted = len(shape) == 3, shape[-1] != 64
    x = rand(*shape, seed=2, dtype=x_type) * 3
    weight = rand(shape[-1], seed=3, dtype=BF16 if shape[-1] % 3 else F32) if weighted else None
    residual = None if res_type is None else rand(*shape, seed=4, dtype=res_type)
    gate = rand(*shape, seed=5, dtype=x_type) * 2 if gated else None
    want, h = plain.norm(x, weight, residual, gate, eps=1e-5)
    got = ops.rms_norm(x, weight, residual=residual, gate=gate, eps=1e-5, dtype=out_type)
    off = plain.norm_error(gate) * want.abs()
    if residual is not None:
        plain.check(residual, h, plain.U * h.abs(), "residual")
    if out_type != E4M3:
        assert got.dtype == out_type
        plain.check(got, want, off, "out")
        return
    check_eight(got, want, off)


def check_eight(got, want, off):
    got, scales = got
    assert got.dtype == E4M3 and scales.dtype == F32
    top = want.flatten(1).abs().amax(1) / 448
    assert bool(((scales.cpu().double() - top).abs() <= top * (plain.norm_error(1) + 4 * plain.U)).all())
    s = scales.cpu().double().view(-1, *[1] * (want.dim() - 1))
    # half a step of E4M3 is 2^-4 of the value, and 2^-10 below its smallest normal value
    room = (want.abs() + off) / s * 2.0 ** -4
    assert bool(((got.cpu().double() - want / s).abs() <= torch.maximum(room, torch.full_like(room, 2.0 ** -10)) + off / s + 4 * plain.U * want.abs() / s).all())
    assert bool((got.cpu().float().abs().flatten(1).amax(1) == 448).all())


@pytest.mark.parametrize("out_type", [BF16, E4M3], ids=str)
@pytest.mark.parametrize("extra", [(0, 0, 8), (1, 2, 16), (3, 1, 3), (0, 5, 1)], ids=str)
def test_norm_strides(ops, extra, out_type):
    x, _ = padded(rand(6, 4, 128, dtype=BF16), *extra)
    gate, _ = padded(rand(6, 4, 128, seed=2, dtype=BF16), *extra[::-1])
    residual, big = padded(rand(6, 4, 128, seed=3), *extra)
    out, far = padded(torch.zeros(6, 4, 128, device="cuda").to(out_type), *extra)
    scales = torch.full((8,), 7.0, device="cuda")
    want, h = plain.norm(x, None, residual, gate)
    got = ops.rms_norm(x, residual=residual, gate=gate, out=out, dtype=out_type, scales=scales[1:7] if out_type == E4M3 else None)
    assert around(big, residual) and around(far, out)
    plain.check(residual, h, plain.U * h.abs(), "residual")
    off = plain.norm_error(gate) * want.abs()
    if out_type == E4M3:
        assert got[0] is out and bool((scales[[0, 7]] == 7).all())
        check_eight(got, want, off)
    else:
        assert got is out
        plain.check(out, want, off, "out")


@pytest.mark.parametrize("dim", [4, 12, 2044, 4100, 8188, 8204, 16380])
@pytest.mark.parametrize("x_type,res_type,out_type", [(BF16, BF16, BF16), (BF16, F32, E4M3), (F32, BF16, F32), (BF16, None, F32)], ids=str)
@pytest.mark.parametrize("shift", [0, 4, 2])
def test_norm_rows_of_fours(ops, dim, x_type, res_type, out_type, shift):
    """Lengths that are multiples of four alone, on 8-byte boundaries of BF16 rows and off them."""
    x = rand(5 * dim + shift, seed=2, dtype=x_type)[shift:].view(5, dim)
    weight = rand(dim, seed=3, dtype=BF16)
    residual = None if res_type is None else rand(5, dim + 4, seed=4, dtype=res_type)[:, :dim]
    kept = None if res_type is None else residual._base[:, dim:].clone()
    far = torch.full((5, dim + 4), 7.0, device="cuda").to(out_type)
    want, h = plain.norm(x, weight, residual)
    got = ops.rms_norm(x, weight, residual=residual, dtype=out_type, out=far[:, :dim])
    off = plain.norm_error(None) * want.abs()
    if residual is not None:
        plain.check(residual, h, plain.U * h.abs(), "residual")
        assert torch.equal(residual._base[:, dim:], kept)
    assert bool((far[:, dim:].float() == 7).all())
    if out_type == E4M3:
        check_eight(got, want, off)
    else:
        plain.check(got, want, off, "out")


def test_norm_heads_before_tokens(ops):
    x = rand(4, 6, 128, dtype=BF16).transpose(0, 1)
    want, _ = plain.norm(x)
    out = torch.empty(4, 6, 128, device="cuda", dtype=BF16).transpose(0, 1)
    plain.check(ops.rms_norm(x, out=out), want, plain.norm_error(None) * want.abs())


@pytest.mark.parametrize("shape", [(5, 2048), (3, 777), (40, 100)], ids=str)
def test_norm_in_place(ops, shape):
    x = rand(*shape)
    want, _ = plain.norm(x)
    assert ops.rms_norm(x, out=x) is x
    plain.check(x, want, plain.norm_error(None) * want.abs())


@pytest.mark.parametrize("dim", [2048, 100, 77])
def test_norm_what_is_not_finite_stays_in_its_row(ops, dim):
    x = rand(9, dim, dtype=BF16)
    x[2, 5], x[4, 0], x[6] = float("nan"), float("inf"), 0.0
    want, _ = plain.norm(x)
    keep = [0, 1, 3, 5, 6, 7, 8]
    got = ops.rms_norm(x)
    plain.check(got[keep], want[keep], plain.norm_error(None) * want[keep].abs())
    assert bool(got[2].isnan().all()) and bool(got[4, 0].isnan())
    y, scales = ops.rms_norm(x, dtype=E4M3)
    assert bool(scales[[2, 4]].isnan().all()) and bool(y.float()[[2, 4]].isnan().all())
    assert bool((y.float()[6] == 0).all()) and float(scales[6]) == 2.0 ** -126
    keep.remove(6)
    check_eight((y[keep], scales[keep]), want[keep], plain.norm_error(None) * want[keep].abs())


def test_norm_nothing_to_do(ops):
    assert ops.rms_norm(torch.empty(0, 64, device="cuda")).shape == (0, 64)
    y, s = ops.rms_norm(torch.empty(0, 4, 64, device="cuda"), dtype=E4M3)
    assert y.shape == (0, 4, 64) and s.shape == (0,)


# ---- linear

def eight_bits(x):
    scale = x.abs().amax(-1).clamp_min(1e-30) / 448
    return (x / scale[:, None]).to(E4M3), scale


def operands(tokens, inputs, rows, eight, seed=1):
    x, w = rand(tokens, inputs, seed=seed), rand(rows, inputs, seed=seed + 1) * inputs ** -0.5
    if not eight:
        return dict(x=x.bfloat16(), weight=w.bfloat16())
    (x, xs), (w, ws) = eight_bits(x), eight_bits(w)
    return dict(x=x, weight=w, x_scales=xs, weight_scales=ws)


TOKENS = [1, 2, 7, 8, 9, 16, 17, 31, 64, 65, 127, 128, 129, 200, 256, 257, 640, 1025]


@pytest.mark.parametrize("tokens", TOKENS)
@pytest.mark.parametrize("eight", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("inputs,outputs,activation,extras", [
    (256, 512, None, ""), (2048, 1003, "silu", "b"), (1008, 64, "gelu", "br"), (528, 333, "swiglu", "br"), (64, 2000, "swiglu", ""),
    (16, 1, None, "r"), (4096, 40, None, "b")])
def test_linear(ops, tokens, eight, inputs, outputs, activation, extras):
    rows = outputs * (2 if activation == "swiglu" else 1)
    a = operands(tokens, inputs, rows, eight)
    even = tokens % 2 == 0
    bias = rand(rows, seed=3, dtype=BF16 if even else F32) if "b" in extras else None
    residual = rand(tokens, outputs, seed=4, dtype=F32 if even else BF16) if "r" in extras else None
    want, off = plain.linear(**a, bias=bias, activation=activation, residual=residual)
    for dtype in (F32, BF16):
        got = ops.linear(**a, bias=bias, activation=activation, residual=residual, dtype=dtype)
        assert got.dtype == dtype
        plain.check(got, want, off, str(dtype))


@pytest.mark.parametrize("tokens", [8, 9, 13, 16, 17])
@pytest.mark.parametrize("eight", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("inputs,outputs,activation", [(2048, 8208, None), (2000, 3700, "swiglu"), (5632, 2486, "gelu"), (5632, 2485, None)])
def test_linear_few_tokens_and_many_weights(ops, tokens, eight, inputs, outputs, activation):
    """Around the number of weights and of tokens where the other kernel takes over."""
    rows = outputs * (2 if activation == "swiglu" else 1)
    x, w = rand(tokens, inputs), rand(rows, inputs, seed=2) * inputs ** -0.5
    s = {}
    if eight:
        (x, s["x_scales"]), (w, s["weight_scales"]) = eight_bits(x), eight_bits(w)
    else:
        x, w = x.to(BF16), w.to(BF16)
    residual = rand(tokens, outputs, seed=3)
    want, off = plain.linear(x, w, activation=activation, residual=residual, **s)
    plain.check(ops.linear(x, w, activation=activation, residual=residual, dtype=F32, **s), want, off)


@pytest.mark.parametrize("tokens", [3, 16, 40, 300])
@pytest.mark.parametrize("eight", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("activation", [None, "silu", "gelu", "swiglu"])
@pytest.mark.parametrize("inputs", [768, 5632])
def test_linear_keeps_twenty_bits(ops, tokens, eight, activation, inputs):
    """FP32 results to 2^-20 in the 2-norm: sums that the tensor cores cut are kept short. Sums of 64 bits of what they see."""
    rows = 1000 * (2 if activation == "swiglu" else 1)
    x, w = rand(tokens, inputs), rand(rows, inputs, seed=2) * inputs ** -0.5
    s = {}
    if eight:
        (x, s["x_scales"]), (w, s["weight_scales"]) = eight_bits(x), eight_bits(w)
    else:
        x, w = x.to(BF16), w.to(BF16)
    want, _ = plain.linear(x, w, activation=activation, **s)
    got = ops.linear(x, w, activation=activation, dtype=F32, **s).cpu().double()
    assert float((got - want).norm() / want.norm()) <= 2.0 ** -20


@pytest.mark.parametrize("tokens", [3, 40, 300])
@pytest.mark.parametrize("eight", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("inputs", [1, 5, 63, 65, 130, 1001])
def test_linear_any_inputs(ops, tokens, eight, inputs):
    """Rows of any length, a multiple of 16 bytes apart; what lies between them is not read into the sums."""
    a = operands(tokens, inputs, 100, eight)
    extra = -inputs % 16 + 16
    want, off = plain.linear(**a)
    for n in ("x", "weight"):
        a[n], _ = padded(a[n], 2, extra, value=float("nan"))
    plain.check(ops.linear(**a, dtype=F32), want, off)


@pytest.mark.parametrize("tokens", [1, 12, 50, 200, 600])
@pytest.mark.parametrize("outputs", [96, 101])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
@pytest.mark.parametrize("extra", [8, 3])
def test_linear_strides_and_place(ops, tokens, outputs, dtype, extra):
    """Into a part of a larger tensor, which is also the residual."""
    a = operands(tokens, 320, outputs, False)
    out, big = padded(rand(tokens, outputs, seed=9, dtype=dtype), 3, extra)
    want, off = plain.linear(**a, residual=out)
    assert ops.linear(**a, residual=out, out=out) is out
    plain.check(out, want, off)
    assert around(big, out)
    other, far = padded(torch.zeros(tokens, outputs, device="cuda", dtype=dtype), 1, extra)
    want, off = plain.linear(**a, residual=out[:, :1].expand(tokens, outputs))
    ops.linear(**a, residual=out[:1].expand(tokens, outputs), out=other)
    want, off = plain.linear(**a, residual=out[:1].expand(tokens, outputs))
    plain.check(other, want, off)
    assert around(far, other)


@pytest.mark.parametrize("tokens", [5, 100, 700])
@pytest.mark.parametrize("eight", [False, True], ids=["bf16", "fp8"])
def test_linear_what_is_not_finite_stays_in_its_row(ops, tokens, eight):
    a = operands(tokens, 512, 300, eight)
    a["x"][3, 17] = float("nan")
    a["weight"][131, 500] = float("nan")
    got = ops.linear(**a, dtype=F32).isnan()
    want = torch.zeros_like(got)
    want[3], want[:, 131] = True, True
    assert torch.equal(got, want)


@pytest.mark.parametrize("outputs", [100, 132, 260, 98, 97, 104])
@pytest.mark.parametrize("shift", [0, 1, 2, 4])
@pytest.mark.parametrize("tokens", [7, 64, 300])
def test_linear_rows_of_results_at_any_alignment(ops, outputs, shift, tokens):
    """Rows that are multiples of 2, 4, 8 and 16 bytes apart and start there."""
    a = operands(tokens, 128, outputs, False)
    for dtype in (BF16, F32):
        for residual in (None, BF16, F32):
            flat = torch.full((tokens * outputs + shift + 8,), 7.0, device="cuda", dtype=dtype)
            out = flat[shift:shift + tokens * outputs].view(tokens, outputs)
            r = None if residual is None else rand(tokens * outputs + shift, seed=6, dtype=residual)[shift:].view(tokens, outputs)
            want, off = plain.linear(**a, residual=r)
            plain.check(ops.linear(**a, residual=r, out=out), want, off)
            assert bool((flat[:shift] == 7).all()) and bool((flat[shift + tokens * outputs:] == 7).all())


def test_linear_the_same_bits_each_time(ops):
    for tokens, outputs in ((1, 2048), (64, 2048), (130, 5632), (2000, 2048)):
        a = operands(tokens, 2048, outputs, False)
        first = ops.linear(**a, dtype=F32)
        for _ in range(5):
            assert torch.equal(ops.linear(**a, dtype=F32), first)


def test_linear_nothing_to_do(ops):
    w = rand(10, 64, dtype=BF16)
    assert ops.linear(torch.empty(0, 64, device="cuda", dtype=BF16), w).shape == (0, 10)
    assert ops.linear(rand(3, 64, dtype=BF16), w[:0]).shape == (3, 0)


# ---- short_conv

CONV_STARTS = [None, [0, 1], [0, 5], [0, 0, 3, 3, 4, 70, 71, 73, 200], [2, 6, 9, 40], [0, 3, 3, 3], [0, 33, 66, 99, 132, 133, 134, 135, 300]]


@pytest.mark.parametrize("starts", CONV_STARTS, ids=str)
@pytest.mark.parametrize("width", [2, 3, 4])
@pytest.mark.parametrize("channels", [64, 1, 1100, 1024])
@pytest.mark.parametrize("x_type,tail_type", [(BF16, F32), (BF16, BF16), (F32, F32)], ids=str)
def test_conv(ops, starts, width, channels, x_type, tail_type):
    tokens = 37 if starts is None else starts[-1] + 3
    n = tokens if starts is None else len(starts) - 1
    x = rand(tokens, channels, dtype=x_type)
    weight = rand(channels, width, seed=2, dtype=BF16 if width == 3 else F32)
    bias = rand(channels, seed=3, dtype=weight.dtype) if width != 4 else None
    tails = rand(n + 2, width - 1, channels, seed=4, dtype=BF16).to(tail_type)
    slots = torch.randperm(n + 2, generator=torch.Generator().manual_seed(5))[:n].int()
    if n > 2:
        slots[1] = -1 if n % 2 else n + 2
    fresh = torch.arange(n) % 3 == 0
    activation = None if channels == 64 else "silu"
    want, after, off = plain.conv(x, weight, tails, bias, activation, None if starts is None else torch.tensor(starts), slots, fresh)
    got = ops.short_conv(x, weight, tails, bias=bias, activation=activation,
                         starts=None if starts is None else torch.tensor(starts, dtype=torch.int32, device="cuda"),
                         slots=slots.cuda(), fresh=fresh.cuda())
    plain.check(got, want, off, "out")
    assert torch.equal(tails.cpu().double(), after)


def test_conv_many_sequences_without_tokens(ops):
    """Between two tokens, before and after them, with a slot for some."""
    lengths = [0] * 3000 + [2] + [0] * 5000 + [1, 0, 0, 70] + [0] * 40000
    starts = torch.tensor([0] + lengths).cumsum(0).int()
    slots = torch.full((len(lengths),), -1).int()
    used = [i for i, n in enumerate(lengths) if n] + [0, 4000, 47000]
    slots[used] = torch.arange(len(used)).int()
    fresh = torch.zeros(len(lengths), dtype=torch.bool)
    fresh[4000] = True
    x, weight, tails = rand(73, 64, dtype=BF16), rand(64, 4, seed=2), rand(len(used), 3, 64, seed=3)
    want, after, off = plain.conv(x, weight, tails, starts=starts, slots=slots, fresh=fresh)
    plain.check(ops.short_conv(x, weight, tails, starts=starts.cuda(), slots=slots.cuda(), fresh=fresh.cuda()), want, off)
    assert torch.equal(tails.cpu().double(), after)


@pytest.mark.parametrize("extra", [8, 3])
@pytest.mark.parametrize("starts", [None, [0, 20, 21, 50]], ids=str)
def test_conv_strides(ops, extra, starts):
    tokens = 50
    n = tokens if starts is None else len(starts) - 1
    x, _ = padded(rand(tokens, 96, dtype=BF16), 0, extra)
    tails, pool = padded(rand(n, 3, 96, seed=2), 2, 1, extra)
    out, big = padded(torch.zeros(tokens, 96, device="cuda", dtype=BF16), 1, extra)
    weight = rand(96, 4, seed=3)
    index = None if starts is None else torch.tensor(starts, dtype=torch.int32, device="cuda")
    want, after, off = plain.conv(x, weight, tails, starts=index)
    assert ops.short_conv(x, weight, tails, starts=index, out=out) is out
    plain.check(out, want, off)
    assert torch.equal(tails.cpu().double(), after) and around(pool, tails) and around(big, out)


@pytest.mark.parametrize("channels,starts,x_type", [(8, [0, 150001, 150003, 330001], BF16), (4, [0, 100, 101, 100001], F32),
                                                    (1001, [0, 20011, 20012, 40000], BF16), (6144, [0, 3000, 4096], BF16)], ids=str)
def test_conv_long_sequences(ops, channels, starts, x_type):
    """Tiles of every length the choice has, and more of them than run at once; sequence by sequence in 64 bits."""
    T, N = starts[-1], len(starts) - 1
    x, w = rand(T, channels, dtype=x_type), rand(channels, 4, seed=2)
    tails, b = rand(N, 3, channels, seed=3), rand(channels, seed=4)
    old = tails.double()
    y = ops.short_conv(x, w, tails, bias=b, starts=torch.tensor(starts, dtype=torch.int32, device="cuda"))
    for n in range(N):
        line = torch.cat([old[n], x[starts[n]:starts[n + 1]].double()])
        taps = [line[j:len(line) - 3 + j] * w[:, j].double() for j in range(4)]
        s, size = sum(taps) + b.double(), sum(t.abs() for t in taps) + b.double().abs()
        want = plain.silu(s)
        off = 1.1 * 5 * plain.U * size + 24 * plain.U * want.abs()  # as in plain.conv
        plain.check(y[starts[n]:starts[n + 1]], want.cpu(), off.cpu(), f"sequence {n}")
        assert torch.equal(tails[n].double(), line[len(line) - 3:])


def test_conv_by_pieces(ops):
    """A prompt in pieces, then token by token, as in one call: the same bits."""
    x, weight = rand(300, 512, dtype=BF16), rand(512, 4, seed=2)
    index = lambda *s: torch.tensor(s, dtype=torch.int32, device="cuda")  # noqa: E731
    whole, tails = torch.zeros(1, 3, 512, device="cuda"), torch.zeros(1, 3, 512, device="cuda")
    want = ops.short_conv(x, weight, whole, starts=index(0, 300))
    at, parts = 0, []
    for n in (1, 2, 100, 3, 190):
        parts.append(ops.short_conv(x[at:at + n], weight, tails, starts=index(0, n)))
        at += n
    for t in range(at, 300):
        parts.append(ops.short_conv(x[t:t + 1], weight, tails))
    assert torch.equal(torch.cat(parts), want) and torch.equal(tails, whole)


@pytest.mark.parametrize("starts", [[10, 3, 5], [4, 8, 0, 0], [5, 8, 3, 2], [0, 5, 9, 0, 0], [70, 0], [-5, 90, 200]], ids=str)
def test_conv_decreasing_starts_end(ops, starts):
    x, weight = rand(70, 64, dtype=BF16), rand(64, 4, seed=2)
    out, big = padded(torch.zeros(70, 64, device="cuda", dtype=BF16), 5, 0)
    tails, pool = padded(rand(len(starts) - 1, 3, 64), 2, 0, 0)
    ops.short_conv(x, weight, tails, starts=torch.tensor(starts, dtype=torch.int32, device="cuda"), out=out)
    torch.cuda.synchronize()
    assert around(big, out) and around(pool, tails)


def test_conv_nothing_to_do(ops):
    tails = rand(2, 3, 64)
    before = tails.clone()
    weight = rand(64, 4)
    none = torch.empty(0, 64, device="cuda")
    assert ops.short_conv(none, weight, tails).shape == (0, 64)
    assert torch.equal(tails, before)
    ops.short_conv(none, weight, tails, starts=torch.zeros(3, dtype=torch.int32, device="cuda"),
                   fresh=torch.tensor([False, True], device="cuda"))
    assert torch.equal(tails[0], before[0]) and bool((tails[1] == 0).all())
