"""Plain 64-bit forms of the layer operators (rms_norm, linear and short_conv of
gateddeltanet_b200/ops.py) on the CPU, from the formulas of include/gdn_b200.h,
and how far FP32 arithmetic may be from them, element by element.

A rounding is off by at most half a step, U = 2^-24 relative for FP32."""
import torch

U = 2.0 ** -24


def half_step(dtype):
    """Of a value rounded to dtype, relative to the value."""
    return torch.finfo(dtype).eps / 2


def silu(x):
    return x * torch.sigmoid(x)


def norm(x, weight=None, residual=None, gate=None, eps=1e-6):
    """(y, h) in float64."""
    h = x.detach().cpu().double()
    if residual is not None:
        h = h + residual.detach().cpu().double()
    y = h / (h.square().mean(-1, keepdim=True) + eps).sqrt()
    if weight is not None:
        y = y * weight.detach().cpu().double()
    if gate is not None:
        y = y * silu(gate.detach().cpu().double())
    return y, h


def norm_error(gate):
    """Relative error of y before its rounding. The sum of squares: sixteen terms in a row and at most twelve joins, each term
    with its h's rounding twice, halved by the root (16 U); rsqrtf 4 U; h and three products 4 U. silu: the exponential
    2 + 1.2 |x| steps of 2 U, which count by |x| sigmoid(-x) < 0.3 at most and so 5 U, its sum, and a quotient of 4 U."""
    return 24 * U if gate is None else 40 * U


def linear(x, weight, bias=None, activation=None, residual=None, x_scales=None, weight_scales=None):
    """(y, its error before the rounding) in float64.

    The tensor cores add 16 products (or more) at a time to an FP32 sum, each time with an error of at most two steps (4 U) of the
    sum of magnitudes; a split of k adds up to 16 more. Then the scales (2 U each), the bias, the activation (slope at most
    1.13, and 24 U of its own result) and the residual."""
    x, w = x.detach().cpu().double(), weight.detach().cpu().double()
    if x_scales is not None:
        x, w = x * x_scales.detach().cpu().double()[:, None], w * weight_scales.detach().cpu().double()[:, None]
    y, size = x @ w.T, x.abs() @ w.abs().T
    off = ((x.shape[1] + 15) // 16 + 20) * 4 * U * size
    if bias is not None:
        y = y + bias.detach().cpu().double()
        off = off + U * y.abs()
    if activation == "swiglu":
        (a, b), (da, db) = y.chunk(2, 1), off.chunk(2, 1)
        y = silu(a) * b
        off = 1.1 * da * (b.abs() + db) + silu(a).abs() * db + 26 * U * y.abs()
    elif activation is not None:
        y = silu(y) if activation == "silu" else 0.5 * y * (1 + torch.erf(y * 0.5 ** 0.5))
        # gelu: the distribution function's formula is off by 7.5e-8, 2.2e-7 at most times |v|, and the roundings of its sum near
        # 0.5 come to 2.5 U |v| where |v| < 1.5 and are relative to the small result beyond: under 7 U in all
        off = 1.13 * off + 24 * U * y.abs() + (7 * U if activation == "gelu" else 0)
    if residual is not None:
        y = y + residual.detach().cpu().double()
        off = off + U * y.abs()
    return y, off


def conv(x, weight, tails, bias=None, activation="silu", starts=None, slots=None, fresh=None):
    """(y, tails, error of y before its rounding) in float64; tails keeps its values where the call leaves them."""
    x, w, tails = x.detach().cpu().double(), weight.detach().cpu().double(), tails.detach().cpu().double().clone()
    T, W = x.shape[0], w.shape[1]
    starts = list(range(T + 1)) if starts is None else [max(0, min(int(s), T)) for s in starts.tolist()]
    y, off = torch.zeros_like(x), torch.zeros_like(x)
    for n in range(len(starts) - 1):
        slot = n if slots is None else int(slots[n])
        if not 0 <= slot < tails.shape[0]:
            continue
        old = torch.zeros_like(tails[slot]) if fresh is not None and bool(fresh[n]) else tails[slot].clone()
        line = torch.cat([old, x[starts[n]:starts[n + 1]]])
        for t in range(starts[n], starts[n + 1]):
            window = line[t - starts[n]:t - starts[n] + W].T * w
            s, size = window.sum(1), window.abs().sum(1)
            if bias is not None:
                s, size = s + bias.detach().cpu().double(), size + bias.detach().cpu().double().abs()
            off[t] = (W + 1) * U * size
            if activation == "silu":
                off[t] = 1.1 * off[t] + 24 * U * silu(s).abs()
                s = silu(s)
            y[t] = s
        tails[slot] = line[len(line) - (W - 1):]
    return y, tails, off


def check(got, want, off, what=""):
    """got is want, off by at most `off` before its rounding to its own type. What is not finite has to be the same."""
    got, dtype = got.detach().cpu().double(), got.dtype
    assert got.shape == want.shape, what
    odd = ~want.isfinite()
    assert bool((got[odd].isnan() == want[odd].isnan()).all()) and bool((got[odd & ~want.isnan()] == want[odd & ~want.isnan()]).all()), what
    room = off + (want.abs() + off) * half_step(dtype) + torch.finfo(dtype).tiny
    far = ((got - want).abs() / room)[~odd]
    assert far.numel() == 0 or float(far.max()) <= 1, f"{what}: {float(far.max()):.3g} times what rounding allows"
