"""Constraints on logits and the greedy pick (gateddeltanet_b200/ops.py
constrain_logits) against the row-by-row form in 64 bits.

Tolerances: a value goes through at most six FP32 operations (quotient,
product and two differences of the penalties, the biases' sum and their
addition; more biases of one token add one each), 2^-24 of the intermediate
values each, which are no more than 8 times the row's 2-norm mean here:
6 * 8 * 2^-24 = 2.9e-6 in the 2-norm. BF16 results are rounded once more, at
most 2^-8 of each value. Picks are whole numbers: they have to be those of
the written values, exactly."""
import math

import pytest
import torch

import ops_plain as plain

pytestmark = pytest.mark.gpu

TOL = {torch.float32: 2.9e-6, torch.bfloat16: 2 ** -8 + 2.9e-6}
INF = math.inf


@pytest.fixture(scope="module")
def ops():
    from gateddeltanet_b200 import build
    build.build()
    from gateddeltanet_b200 import ops
    return ops


def inputs(rows, vocab, history, biases, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    ri = lambda lo, hi, *s: torch.randint(lo, hi, s, generator=gen, dtype=torch.int32)  # noqa: E731
    tokens = ri(-2, vocab + 2, rows, history)  # a few ids outside the vocabulary
    common = ri(0, min(vocab, 7), rows, history)
    tokens = torch.where(torch.rand(rows, history, generator=gen) < 0.5, common, tokens)
    lens = ri(0, history + 1, rows)
    a = dict(logits=(torch.randn(rows, vocab, generator=gen) * 3).to(dtype), tokens=tokens, lens=lens,
             prompt_lens=(lens * torch.rand(rows, generator=gen)).int(), repetition=1 + torch.rand(rows, generator=gen),
             presence=torch.rand(rows, generator=gen), frequency=0.2 * torch.rand(rows, generator=gen),
             bias_ids=ri(-1, vocab + 1, rows, biases), bias=torch.randn(rows, biases, generator=gen),
             mask=ri(-2 ** 31, 2 ** 31 - 1, rows, (vocab + 31) // 32))
    return {n: x.cuda() for n, x in a.items()}


def compare(ops, a, **more):
    ref = plain.constrain(**a)
    before = {n: x.clone() for n, x in a.items()}
    out, picks = ops.constrain_logits(**a, **more)
    torch.cuda.synchronize()
    got = out.cpu().double()
    special = ~ref.isfinite()
    assert torch.equal(got[special].nan_to_num(nan=123.0, posinf=INF, neginf=-INF),
                       ref[special].nan_to_num(nan=123.0, posinf=INF, neginf=-INF))
    assert plain.rel(got[~special], ref[~special]) <= TOL[out.dtype]
    assert picks.tolist() == plain.greedy(out)
    if more.get("out") is not a["logits"]:
        for n, x in before.items():
            assert torch.equal(a[n].nan_to_num(nan=7e30) if a[n].is_floating_point() else a[n],
                               x.nan_to_num(nan=7e30) if x.is_floating_point() else x), f"{n} was written"
    return out, picks


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("rows,vocab,history,biases", [
    (1, 1, 1, 1), (1, 31, 5, 2), (3, 33, 1, 1), (2, 1000, 64, 3), (5, 4099, 700, 17), (1, 32000, 2000, 9),
    (70, 1003, 40, 4), (3, 70001, 300, 30), (300, 257, 9, 2)])
def test_all_constraints(ops, rows, vocab, history, biases, dtype):
    compare(ops, inputs(rows, vocab, history, biases, dtype, seed=vocab))


@pytest.mark.parametrize("left_out", [("mask",), ("bias", "bias_ids"), ("repetition",), ("presence", "frequency"),
                                      ("lens",), ("prompt_lens",), ("lens", "prompt_lens", "repetition", "bias", "bias_ids"),
                                      ("tokens", "lens", "prompt_lens", "repetition", "presence", "frequency"),
                                      ("tokens", "lens", "prompt_lens", "repetition", "presence", "frequency", "bias",
                                       "bias_ids", "mask")], ids=str)
def test_any_part_may_be_missing(ops, left_out):
    a = inputs(3, 2003, 100, 5, torch.float32, seed=1)
    compare(ops, {n: x for n, x in a.items() if n not in left_out})


def test_empty_history_and_no_entries(ops):
    a = inputs(2, 100, 3, 2, torch.float32, seed=2)
    a.update(tokens=a["tokens"][:, :0], bias=a["bias"][:, :0], bias_ids=a["bias_ids"][:, :0], lens=a["lens"] * 0)
    compare(ops, a)
    b = inputs(2, 100, 3, 2, torch.float32, seed=3)
    b["lens"][0] = -5           # nothing in use
    b["lens"][1] = 2 ** 30      # more than there is
    b["prompt_lens"][1] = -1
    compare(ops, b)


def test_masks_that_leave_one_or_nothing(ops):
    a = inputs(4, 5000, 50, 4, torch.bfloat16, seed=4)
    a["mask"].zero_()
    a["mask"][1, 4999 // 32] = 1 << (4999 % 32)
    a["mask"][2, 0] = 1
    out, picks = compare(ops, a)
    assert picks.tolist() == [-1, 4999, 0, -1]


def test_special_values(ops):
    """NaN, infinities and the lowest finite value, in masked places and outside them."""
    a = inputs(6, 300, 20, 3, torch.float32, seed=5)
    lowest = torch.finfo(torch.float32).min
    a["logits"][0] = float("nan")
    a["logits"][1, :150] = float("nan")
    a["logits"][2] = -INF
    a["logits"][3] = lowest
    a["logits"][4, 7] = INF
    a["logits"][4, 9] = INF
    a["mask"][4] = -1
    a["mask"][5] = 0
    a["logits"][5] = float("nan")
    a["repetition"].fill_(1.0)
    a["presence"].zero_()
    a["frequency"].zero_()
    a["bias"].zero_()
    out, picks = compare(ops, a)
    assert picks[0] == -1 and picks[2] == -1 and picks[4] == 7 and picks[5] == -1 and picks[3] >= 0
    assert bool((out[5] == -INF).all())


def test_ties_go_to_the_lowest_token(ops):
    for vocab in (64, 4096, 40000):
        logits = torch.zeros(3, vocab, device="cuda")
        logits[1, vocab // 2:] = 1
        logits[2, -1] = 1
        logits[0, 0] = -0.0
        _, picks = ops.constrain_logits(logits)
        assert picks.tolist() == [0, vocab // 2, vocab - 1]


def test_repeated_bias_entries_add_in_order(ops):
    """Entries of one token add up in list order: with 2^24 first, the ones after it are lost; after -2^24 they count."""
    logits = torch.zeros(1, 100, device="cuda")
    ids = torch.tensor([[5, 9, 5, 5, 5, 9]], dtype=torch.int32, device="cuda")
    bias = torch.tensor([[2.0 ** 24, 1, 1, -2.0 ** 24, 1, 2]], device="cuda")
    for _ in range(3):
        out, picks = ops.constrain_logits(logits, bias_ids=ids, bias=bias)
        assert out[0, 5] == 1 and out[0, 9] == 3 and picks.item() == 9
    many = torch.full((1, 2047), 3, dtype=torch.int32, device="cuda")
    out, picks = ops.constrain_logits(logits, bias_ids=many, bias=torch.full((1, 2047), 0.5, device="cuda"))
    assert out[0, 3] == 2047 * 0.5 and picks.item() == 3


def test_long_history(ops):
    """A count beyond 16 bits, and a token that only the prompt holds."""
    n = 70000
    tokens = torch.full((1, n), 11, dtype=torch.int32, device="cuda")
    tokens[0, 0] = 12
    logits = torch.ones(1, 50, device="cuda")
    one = torch.ones(1, device="cuda")
    out, picks = ops.constrain_logits(logits, tokens=tokens, prompt_lens=torch.ones(1, dtype=torch.int32, device="cuda"),
                                      frequency=one, repetition=2 * one)
    assert out[0, 11] == 0.5 - (n - 1) and out[0, 12] == 0.5 and picks.item() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_strides_and_alignment(ops, dtype):
    a = inputs(5, 777, 30, 4, dtype, seed=6)
    for shift_in, shift_out in ((0, 0), (1, 1), (3, 0), (0, 5)):
        wide = torch.empty(5, 800, device="cuda", dtype=dtype)
        wide[:, shift_in:shift_in + 777] = a["logits"]
        out = torch.full((5, 801), 7.0, device="cuda", dtype=dtype)
        tokens = torch.empty(5, 41, device="cuda", dtype=torch.int32)
        tokens[:, 2:32] = a["tokens"]
        b = dict(a, logits=wide[:, shift_in:shift_in + 777], tokens=tokens[:, 2:32])
        compare(ops, b, out=out[:, shift_out:shift_out + 777])
        assert bool((out[:, :shift_out] == 7).all()) and bool((out[:, shift_out + 777:] == 7).all())


def test_in_place_and_same_bits(ops):
    a = inputs(40, 9001, 500, 20, torch.float32, seed=7)
    out, picks = ops.constrain_logits(**a)
    again = dict(a, logits=a["logits"].clone())
    out2, picks2 = ops.constrain_logits(**again, out=again["logits"])
    assert out2.data_ptr() == again["logits"].data_ptr()
    assert torch.equal(out, out2) and torch.equal(picks, picks2)


def test_refusals(ops):
    a = inputs(2, 100, 5, 2, torch.float32)
    bad = [dict(logits=a["logits"].half()), dict(logits=a["logits"].t()), dict(logits=a["logits"].cpu()),
           dict(logits=a["logits"][0]), dict(tokens=a["tokens"].long()), dict(tokens=a["tokens"][:1]),
           dict(lens=a["lens"].float()), dict(mask=a["mask"][:, :2]), dict(bias=a["bias"][:, :1]), dict(bias=None),
           dict(tokens=None), dict(repetition=a["repetition"].double()), dict(out=torch.empty(2, 100, device="cuda").half()),
           dict(out=torch.empty(1, 100, device="cuda").expand(2, 100)), dict(presence=a["presence"][:1])]
    for change in bad:
        with pytest.raises(ValueError):
            ops.constrain_logits(**{**a, **change})
    with pytest.raises(RuntimeError, match="vocab"):
        ops.constrain_logits(torch.zeros(1, 2 ** 18 + 1, device="cuda"))
    with pytest.raises(RuntimeError, match="biases"):
        ops.constrain_logits(a["logits"], bias_ids=torch.zeros(2, 2048, device="cuda", dtype=torch.int32),
                             bias=torch.zeros(2, 2048, device="cuda"))
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.constrain_logits(a["logits"].clone().requires_grad_())
