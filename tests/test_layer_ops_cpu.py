"""The C entries of the layer operators refuse what they cannot do before any
device is touched, and the torch binding what does not fit (no GPU needed);
the plain forms agree with a second way of writing the formulas."""
import ctypes
import struct

import pytest
import torch

import gateddeltanet_b200 as gdn
import layer_plain as plain
from test_ops_cpu import FAKE, lib  # noqa: F401

NORM = struct.Struct("@7Q8q3I5ifI")   # GdnB200NormArgs
LINEAR = struct.Struct("@8Q4q3I6iI")  # GdnB200LinearArgs
CONV = struct.Struct("@9Q4q5I5i")     # GdnB200ConvArgs
FAR = FAKE + (1 << 30)  # well apart from FAKE


def pack(layout, fields, change):
    assert set(change) <= set(fields)
    return layout.pack(*{**fields, **change}.values())


def norm_args(**change):
    return pack(NORM, dict(
        x=FAKE, gate=0, weight=FAR, residual=0, out=FAKE + (1 << 26), scales=0, stream=0, x_token=256, x_head=64, gate_token=256,
        gate_head=64, residual_token=256, residual_head=64, out_token=256, out_head=64, tokens=5, heads=4, dim=64, dtype=1,
        weight_dtype=0, residual_dtype=0, out_dtype=1, device=77, eps=1e-6, reserved=0), change)


def linear_args(**change):
    return pack(LINEAR, dict(
        x=FAKE, weight=FAR, bias=0, residual=0, x_scales=0, weight_scales=0, out=FAKE + (1 << 26), stream=0, x_row=64, weight_row=64,
        residual_row=100, out_row=100, tokens=5, inputs=64, outputs=100, dtype=1, bias_dtype=0, residual_dtype=0, out_dtype=1,
        activation=0, device=77, reserved=0), change)


def conv_args(**change):
    return pack(CONV, dict(
        x=FAKE, weight=FAR, bias=0, tails=FAR + (1 << 26), out=FAKE + (1 << 26), starts=FAKE, slots=FAKE, fresh=0, stream=0,
        x_token=64, out_token=64, tails_slot=192, tails_row=64, sequences=2, tokens=5, channels=64, width=4, tail_slots=2, dtype=1,
        weight_dtype=0, tail_dtype=0, activation=1, device=77), change)


@pytest.mark.parametrize("change,reason", [
    (dict(dtype=2), "dtype"), (dict(weight_dtype=2), "weight_dtype"), (dict(residual=FAR, residual_dtype=2), "residual_dtype"),
    (dict(out_dtype=3), "out_dtype"), (dict(dim=0), "no values"), (dict(tokens=2 ** 30), "too many"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(x=0), "missing"), (dict(out=0), "missing"), (dict(out_dtype=2), "scales"),
    (dict(x_token=-1), "stride"), (dict(x=FAKE + 1), "misaligned"), (dict(residual=FAR + 2), "misaligned"),
    (dict(heads=1, dim=16385), "more than one CTA"), (dict(out_dtype=2, scales=FAR, heads=257, dim=64), "more than one CTA"),
    (dict(out=FAKE + 2), "out overlaps"), (dict(out=FAKE, out_dtype=0), "out overlaps"), (dict(gate=FAKE + (1 << 26)), "out overlaps"),
    (dict(residual=FAKE, residual_dtype=1), "residual overlaps"), (dict(residual=FAR, gate=FAR), "residual overlaps"),
    (dict(out_dtype=2, scales=FAKE), "scales overlaps"), (dict(out=FAKE, out_token=512), "out overlaps"),
    (dict(out=FAKE, x_token=0, out_token=0), "rows of out"), (dict(out_head=63), "rows of out"), (dict(out_token=255), "rows of out"),
    (dict(out_token=64, out_head=319), "rows of out"), (dict(residual=FAR + (1 << 26), residual_head=0), "rows of the residual")])
def test_norm_refusals(lib, change, reason):  # noqa: F811
    assert lib.gdn_b200_rms_norm(norm_args(**change)) == -1
    assert reason in gdn.last_error()


@pytest.mark.parametrize("change", [
    dict(), dict(out=FAKE), dict(weight=0), dict(residual=FAR + (1 << 26)), dict(gate=FAKE), dict(out_dtype=2, scales=FAR + 4096),
    dict(heads=1, dim=16384, x_token=16384, out_token=16384), dict(x=FAKE + 2), dict(tokens=1, heads=1, x_token=0, out_token=0),
    dict(out_token=64, out_head=320), dict(x_token=0), dict(x_token=512, gate=FAKE + 512, gate_token=512, out=FAKE, out_token=512)], ids=str)
def test_norm_is_taken(lib, change):  # noqa: F811
    assert lib.gdn_b200_rms_norm(norm_args(**change)) == -1
    assert "device" in gdn.last_error()  # refused for the device alone


@pytest.mark.parametrize("change,reason", [
    (dict(dtype=0), "dtype"), (dict(bias=FAR, bias_dtype=2), "bias_dtype"), (dict(residual=FAR, residual_dtype=3), "residual_dtype"),
    (dict(out_dtype=2), "out_dtype"), (dict(activation=4), "activation"), (dict(inputs=0), "no inputs"),
    (dict(tokens=2 ** 24 + 1), "too large"), (dict(tokens=2 ** 20, outputs=2 ** 20, out_row=2 ** 20), "too large"),
    (dict(x=0), "missing"), (dict(weight=0), "missing"), (dict(out=0), "missing"), (dict(dtype=2), "scales"),
    (dict(x=FAKE + 8), "16-byte"), (dict(x_row=68), "16-byte"), (dict(weight_row=71), "16-byte"), (dict(x_row=56), "overlap"),
    (dict(weight_row=0), "overlap"), (dict(out_row=99), "rows of out"), (dict(residual=FAR, residual_row=-1), "stride"),
    (dict(x_row=1 << 40), "far apart"), (dict(out=FAKE + (1 << 26) + 1), "misaligned"), (dict(out=FAKE), "overlaps"),
    (dict(out=FAR + 64), "overlaps"), (dict(residual=FAKE + (1 << 26), residual_dtype=0), "overlaps"),
    (dict(residual=FAKE + (1 << 26) + 2, residual_dtype=1), "overlaps"), (dict(bias=FAKE + (1 << 26)), "overlaps")])
def test_linear_refusals(lib, change, reason):  # noqa: F811
    assert lib.gdn_b200_linear(linear_args(**change)) == -1
    assert reason in gdn.last_error()


@pytest.mark.parametrize("change", [
    dict(), dict(residual=FAKE + (1 << 26), residual_dtype=1), dict(inputs=57), dict(dtype=2, x_scales=FAKE, weight_scales=FAR),
    dict(tokens=1, x_row=0), dict(activation=3), dict(x_row=128, out=FAKE + 128, out_row=128, outputs=32),
    dict(residual=FAR + 200, residual_row=0)], ids=str)
def test_linear_is_taken(lib, change):  # noqa: F811
    assert lib.gdn_b200_linear(linear_args(**change)) == -1
    assert "device" in gdn.last_error()


@pytest.mark.parametrize("change,reason", [
    (dict(dtype=2), "dtype"), (dict(weight_dtype=2), "weight_dtype"), (dict(dtype=0, tail_dtype=1), "tail_dtype"),
    (dict(activation=2), "activation"), (dict(width=1), "width"), (dict(width=5), "width"), (dict(tokens=2 ** 30), "too many"),
    (dict(channels=2 ** 23), "too many"), (dict(starts=0), "without starts"), (dict(sequences=0), "no sequence"),
    (dict(slots=0, tail_slots=1), "slots"), (dict(weight=0), "missing"), (dict(tails=0), "missing"), (dict(x=0), "missing"),
    (dict(x_token=-64), "stride"), (dict(out_token=63), "rows of out"), (dict(tails_row=63), "tails overlap"),
    (dict(tails_slot=191), "tails overlap"), (dict(tails=FAR + 2), "misaligned"), (dict(out=FAKE + 2), "out overlaps"),
    (dict(out=FAKE), "out overlaps"), (dict(tails=FAKE), "tails overlaps"), (dict(tails=FAR), "tails overlaps")])
def test_conv_refusals(lib, change, reason):  # noqa: F811
    assert lib.gdn_b200_short_conv(conv_args(**change)) == -1
    assert reason in gdn.last_error()


@pytest.mark.parametrize("change", [dict(), dict(width=2, tails_row=0), dict(tail_dtype=1), dict(x_token=0), dict(tokens=0, x=0, out=0),
                                    dict(x_token=128, out=FAKE + 128, out_token=128)], ids=str)
def test_conv_is_taken(lib, change):  # noqa: F811
    assert lib.gdn_b200_short_conv(conv_args(**change)) == -1
    assert "device" in gdn.last_error()


def test_nothing_to_do(lib):  # noqa: F811
    assert lib.gdn_b200_rms_norm(norm_args(tokens=0)) == 0 and lib.gdn_b200_rms_norm(norm_args(heads=0)) == 0
    assert lib.gdn_b200_linear(linear_args(tokens=0)) == 0 and lib.gdn_b200_linear(linear_args(outputs=0)) == 0
    assert lib.gdn_b200_short_conv(conv_args(sequences=0, tokens=0)) == 0 and lib.gdn_b200_short_conv(conv_args(channels=0)) == 0
    for entry in ("rms_norm", "linear", "short_conv"):
        assert getattr(lib, "gdn_b200_" + entry)(None) == -1


def test_argument_layouts():
    assert NORM.size == 7 * 8 + 8 * 8 + 10 * 4 and LINEAR.size == 8 * 8 + 4 * 8 + 10 * 4 and CONV.size == 9 * 8 + 4 * 8 + 10 * 4
    assert ctypes.sizeof(ctypes.c_void_p) == 8


@pytest.fixture(scope="module")
def ops():
    from gateddeltanet_b200 import build
    build.build()
    from gateddeltanet_b200 import ops
    return ops


def bf16(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


@pytest.mark.parametrize("call,reason", [
    (lambda o: o.rms_norm(bf16(2, 8)), "CUDA device"), (lambda o: o.rms_norm(bf16(8)), "dimensions"),
    (lambda o: o.rms_norm(bf16(2, 8).half()), "neither float nor bfloat16"),
    (lambda o: o.rms_norm([1.0]), "not a tensor"), (lambda o: o.rms_norm(None), "missing"),
    (lambda o: o.linear(bf16(2, 8), bf16(4, 8)), "CUDA device"), (lambda o: o.linear(bf16(2, 8).float(), bf16(4, 8)), "neither bfloat16"),
    (lambda o: o.linear(bf16(2, 8), bf16(4, 9)), "shape"), (lambda o: o.linear(bf16(2, 8), bf16(3, 8), activation="swiglu"), "halves"),
    (lambda o: o.linear(bf16(2, 8), bf16(4, 8), activation="relu"), "activation"), (lambda o: o.linear(bf16(2, 8), bf16(4, 8), activation=3), "activation"),
    (lambda o: o.short_conv(bf16(2, 8), bf16(8, 4), bf16(2, 3, 8)), "CUDA device"),
    (lambda o: o.short_conv(bf16(2, 8), bf16(8, 4), bf16(2, 4, 8)), "shape"),
    (lambda o: o.short_conv(bf16(2, 8), bf16(8, 4), bf16(2, 3, 8), activation="gelu"), "activation")])
def test_binding_refusals(ops, call, reason):
    with pytest.raises(ValueError, match=reason):
        call(ops)


def test_gradients_are_refused(ops):
    x = bf16(2, 8).requires_grad_()
    for call in (lambda: ops.rms_norm(x), lambda: ops.linear(x, bf16(4, 8)), lambda: ops.linear(bf16(2, 8), bf16(4, 8), residual=x),
                 lambda: ops.short_conv(x, bf16(8, 4), bf16(2, 3, 8)), lambda: ops.short_conv(bf16(2, 8), bf16(8, 4), x)):
        with pytest.raises(RuntimeError, match="gradient"):
            call()


def test_plain_forms_by_torch():
    gen = torch.Generator().manual_seed(1)
    rn = lambda *s: torch.randn(s, generator=gen, dtype=torch.float64)  # noqa: E731
    x, w, g, r = rn(5, 3, 16), rn(16), rn(5, 3, 16), rn(5, 3, 16)
    y, h = plain.norm(x, w, r, g, eps=1e-5)
    assert torch.allclose(y, torch.nn.functional.rms_norm(x + r, (16,), w, 1e-5) * torch.nn.functional.silu(g)) and torch.equal(h, x + r)
    x, w, b, r = rn(4, 16), rn(6, 16), rn(6), rn(4, 3)
    F = torch.nn.functional
    a, u = F.linear(x, w, b).chunk(2, 1)
    assert torch.allclose(plain.linear(x, w, b, "swiglu", r)[0], F.silu(a) * u + r)
    assert torch.allclose(plain.linear(x, w, b, "gelu")[0], F.gelu(F.linear(x, w, b)))
    x, w, tails = rn(7, 6), rn(6, 4), rn(2, 3, 6)
    y, after, _ = plain.conv(x, w, tails, activation=None, starts=torch.tensor([0, 7]), slots=torch.tensor([1]))
    line = torch.cat([tails[1], x]).T[None]
    assert torch.allclose(y, F.conv1d(line, w[:, None], groups=6)[0].T) and torch.equal(after[1], x[-3:]) and torch.equal(after[0], tails[0])


@pytest.mark.parametrize("entry,args,reason", [
    ("gdn_b200_linear", lambda: linear_args(dtype=2, x_scales=FAKE + 2, weight_scales=FAR), "misaligned"),
    ("gdn_b200_linear", lambda: linear_args(dtype=2, x_scales=FAKE, weight_scales=FAR + 1), "misaligned"),
    ("gdn_b200_short_conv", lambda: conv_args(starts=FAKE + 2), "misaligned"),
    ("gdn_b200_short_conv", lambda: conv_args(slots=FAKE + 1), "misaligned"),
    ("gdn_b200_rms_norm", lambda: norm_args(heads=0, out_dtype=2, scales=FAR), "no values")])
def test_vectors_off_their_boundaries_and_scales_of_nothing(lib, entry, args, reason):  # noqa: F811
    assert getattr(lib, entry)(args()) == -1
    assert reason in gdn.last_error()


def test_norm_of_no_heads(lib):  # noqa: F811
    assert lib.gdn_b200_rms_norm(norm_args(heads=0)) == 0
