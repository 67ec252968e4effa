"""The rest of a gated-delta-rule layer on device tensors: what is measured, in plain torch and through the framework.

  norm    root-mean-square norm, with the addition to the residual before it, a swish gate after it, and outputs
          in 16 or 32 bits or in 8 bits with a scale for each token
  linear  x W^T with 16-bit operands or 8-bit ones with scales, then bias, activation and residual
  conv    the short causal convolution over packed sequences, last inputs kept in a pool of slots, for new tokens and prompts

norm:    h = residual + x;  y = h / sqrt(mean(h^2) + eps) * weight * silu(gate);  8 bits: y / s with s = max(|y|) / 448 of the token
linear:  y = act(sx sw x W^T + bias) + residual;  swiglu: silu of the first half of the outputs times the second half
conv:    y[t] = silu(sum_j w[j] x[t - (width - 1) + j]), where what lies before the sequence comes from its slot
"""
import random

import torch

own = False

LARGEST = 448.0  # of the 8-bit type
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32, "fp8": torch.float8_e4m3fn}


def listed():
    norm = dict(op="norm", heads=1, dim=2048, x="bf16", residual="none", gate=False, to="bf16")
    linear = dict(op="linear", operands="bf16", bias=False, activation="none", residual="none", to="bf16")
    conv = dict(op="conv", streams=64, longest=1, spread=0, channels=6144, width=4, dtype="bf16", tail="fp32")
    return [
        # one conversation, one new token: between two layers of GDN-1.3B
        dict(norm, name="norm, 1 token", tokens=1, residual="bf16"),
        # the benchmark's prompt between two layers, into the 8-bit projection that follows
        dict(norm, name="norm, 4096 tokens to 8 bits", tokens=4096, residual="fp32", to="fp8"),
        # the output norm of the delta rule's heads with its gate
        dict(norm, name="norm, 4096 x 8 gated heads", tokens=4096, heads=8, dim=256, gate=True),
        # odd rows that start at any alignment
        dict(norm, name="norm, 515 odd rows", tokens=515, dim=1999, x="fp32", residual="fp32", to="fp32"),
        # one conversation: q, k, v, gate and the two small projections of a layer in one product
        dict(linear, name="linear, 1 token", tokens=1, inputs=2048, outputs=8208),
        # the usual number of streams a GPU: gate and up projections of the MLP
        dict(linear, name="linear, 64 tokens swiglu", tokens=64, inputs=2048, outputs=5632, activation="swiglu"),
        # the same streams' logits
        dict(linear, name="linear, 64 rows of logits", tokens=64, inputs=2048, outputs=32000, to="fp32"),
        # ragged sizes: bias and activation of any model
        dict(linear, name="linear, 333 odd", tokens=333, inputs=1000, outputs=1003, bias=True, activation="gelu"),
        # the benchmark's prompt: down projection onto the residual
        dict(linear, name="linear, 4096 tokens down", tokens=4096, inputs=5632, outputs=2048, residual="fp32", to="fp32"),
        # the same prompt in 8 bits: gate and up projections, the most work of a layer
        dict(linear, name="linear, 4096 tokens swiglu 8 bits", tokens=4096, inputs=2048, outputs=5632, operands="fp8",
             activation="swiglu"),
        # q, k and v of the new token of every stream
        dict(conv, name="conv, 64 streams"),
        # prompts of very different lengths
        dict(conv, name="conv, 24 ragged", streams=24, longest=2047, spread=5),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    op = rng.choice(("norm", "linear", "linear", "conv"))
    if op == "norm":
        heads = rng.choice((1, 1, 2, 4, 8, 12))
        dim = rng.choice((64, 128, 256)) if heads > 1 else rng.choice((1, 8)) * _log_int(rng, 50, 1000)
        return dict(op=op, tokens=_log_int(rng, 1, 4096), heads=heads, dim=dim, x=rng.choice(("bf16", "bf16", "fp32")),
                    residual=rng.choice(("none", "bf16", "fp32")) if heads == 1 else "none", gate=heads > 1,
                    to=rng.choice(("bf16", "fp32", "fp8")))
    if op == "linear":
        operands = rng.choice(("bf16", "bf16", "fp8"))
        tokens, inputs = _log_int(rng, 1, 4096), 16 * _log_int(rng, 4, 352)
        most = min(32000, 4096 * 2048 * 5632 // (tokens * inputs))
        return dict(op=op, tokens=tokens, inputs=inputs, outputs=_log_int(rng, 16, most), operands=operands,
                    bias=rng.random() < 0.3, activation=rng.choice(("none", "none", "silu", "gelu", "swiglu")),
                    residual=rng.choice(("none", "bf16", "fp32")), to=rng.choice(("bf16", "fp32")))
    dtype = rng.choice(("bf16", "fp32"))
    longest = rng.choice((1, _log_int(rng, 1, 4096)))
    streams = _log_int(rng, 1, max(1, min(256, (24000 if dtype == "bf16" else 12000) // longest)))
    return dict(op=op, streams=streams, longest=longest, spread=rng.randrange(1, 1000) if longest > 1 and streams > 1 else 0,
                channels=rng.choice((1, 8)) * _log_int(rng, 16, 768), width=rng.choice((2, 3, 4, 4)), dtype=dtype,
                tail=rng.choice(("bf16", "fp32")) if dtype == "bf16" else "fp32")


def _lengths(case):
    """Tokens of every stream: all `longest`, or, with a spread, from none to `longest`."""
    n, longest = case["streams"], case["longest"]
    if not case["spread"]:
        return [longest] * n
    rng = random.Random(case["spread"])
    return [rng.randint(0, longest) for _ in range(n - 1)] + [longest]


def _eight_bits(x):
    """Rows of x in 8 bits, and their scales."""
    scale = (x.abs().amax(-1) / LARGEST).clamp_min(2.0 ** -126)
    return (x / scale[..., None]).to(torch.float8_e4m3fn), scale


def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(dev).manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=dev)

    def maybe(name, *shape):
        return None if case[name] == "none" else normal(*shape).to(TYPES[case[name]])

    if case["op"] == "norm":
        T, H, D, dt = case["tokens"], case["heads"], case["dim"], TYPES[case["x"]]
        shape = (T, D) if H == 1 else (T, H, D)
        some = torch.where(torch.rand(D, generator=gen, device=dev) < 0.005, 20.0, 1.0)  # channels of large values
        x = (normal(*shape) * some).to(dt)
        # the gate is a part of the projection that made it
        gate = normal(T, 4 * H * D + 2 * H).to(dt)[:, 3 * H * D:4 * H * D].view(shape) if case["gate"] else None
        return dict(case=case, x=x, weight=1 + 0.1 * normal(D), residual=maybe("residual", *shape), gate=gate)

    if case["op"] == "linear":
        T, K = case["tokens"], case["inputs"]
        N = case["outputs"] * (2 if case["activation"] == "swiglu" else 1)
        x, w = normal(T, K), normal(N, K) * K ** -0.5
        s = dict(case=case, bias=normal(N) if case["bias"] else None, residual=maybe("residual", T, case["outputs"]),
                 x_scales=None, w_scales=None)
        if case["operands"] == "fp8":
            (s["x"], s["x_scales"]), (s["w"], s["w_scales"]) = _eight_bits(x), _eight_bits(w)
        else:
            s["x"], s["w"] = x.bfloat16(), w.bfloat16()
        return s

    C, W, dt = case["channels"], case["width"], TYPES[case["dtype"]]
    lengths = _lengths(case)
    N, T = len(lengths), sum(lengths)
    # q, k and v are a part of the projection that made them
    x = normal(T, C + C // 3 + 16).to(dt)[:, :C]
    starts = torch.tensor([0] + lengths, device=dev).cumsum(0).to(torch.int32)
    slots = torch.randperm(N + 3, generator=gen, device=dev)[:N].to(torch.int32)
    fresh = torch.zeros(N, device=dev, dtype=torch.bool)
    if case["longest"] > 1:
        fresh[::2] = True  # new conversations; the others go on from their last inputs
    # what a slot holds was an input once
    tails = normal(N + 3, W - 1, C).to(dt).to(TYPES[case["tail"]])
    return dict(case=case, x=x, weight=(torch.rand((C, W), generator=gen, device=dev) - 0.5) * 2 * W ** -0.5, tails=tails,
                starts=starts, slots=slots, fresh=fresh, one_each=max(lengths) == min(lengths) == 1)


def run(s):
    case = s["case"]
    if own:
        from gateddeltanet_b200 import ops
        if case["op"] == "norm":
            y = ops.rms_norm(s["x"], s["weight"], residual=s["residual"], gate=s["gate"], eps=1e-6, dtype=TYPES[case["to"]])
            return _norm_outputs(s, *(y if case["to"] == "fp8" else (y, None)))
        if case["op"] == "linear":
            activation = None if case["activation"] == "none" else case["activation"]
            return {"y": ops.linear(s["x"], s["w"], bias=s["bias"], activation=activation, residual=s["residual"],
                                    x_scales=s["x_scales"], weight_scales=s["w_scales"], dtype=TYPES[case["to"]])}
        y = ops.short_conv(s["x"], s["weight"], s["tails"], activation="silu", starts=None if s["one_each"] else s["starts"],
                           slots=s["slots"], fresh=s["fresh"])
        return {"y": y, "tails": s["tails"]}
    return {"norm": _plain_norm, "linear": _plain_linear, "conv": _plain_conv}[case["op"]](s)


def _norm_outputs(s, y, scales):
    """What the call gives; 8-bit values stand for themselves, beside their scales."""
    out = {"y": y}
    if scales is not None:
        out["scales"] = scales
    if s["residual"] is not None:
        out["residual"] = s["residual"]
    return out


def _silu(x):
    return x / (1 + (-x).exp())


def _plain_norm(s):
    h = s["x"].float()
    if s["residual"] is not None:
        h = h + s["residual"].float()
        s["residual"].copy_(h)
    y = h / (h.square().mean(-1, keepdim=True) + 1e-6).sqrt() * s["weight"]
    if s["gate"] is not None:
        y = y * _silu(s["gate"].float())
    if s["case"]["to"] != "fp8":
        return _norm_outputs(s, y.to(TYPES[s["case"]["to"]]), None)
    y8, scales = _eight_bits(y.flatten(1))
    return _norm_outputs(s, y8.view(y.shape), scales)


def _plain_linear(s):
    case = s["case"]
    y = s["x"].float() @ s["w"].float().T
    if s["x_scales"] is not None:
        y = y * s["x_scales"][:, None] * s["w_scales"]
    if s["bias"] is not None:
        y = y + s["bias"]
    if case["activation"] == "swiglu":
        gate, up = y.chunk(2, 1)
        y = _silu(gate) * up
    elif case["activation"] == "silu":
        y = _silu(y)
    elif case["activation"] == "gelu":
        y = 0.5 * y * (1 + (y * 0.5 ** 0.5).erf())
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return {"y": y.to(TYPES[case["to"]])}


def _plain_conv(s):
    x, W, tails, slots = s["x"].float(), s["case"]["width"], s["tails"], s["slots"].long()
    T, N = x.shape[0], slots.shape[0]
    begin, length = s["starts"][:-1].long(), (s["starts"][1:] - s["starts"][:-1]).long()
    t = torch.arange(T, device="cuda")
    stream = torch.searchsorted(s["starts"][1:].long(), t, right=True)
    at = t - begin[stream]
    past = torch.where(s["fresh"][:, None, None], 0.0, tails[slots].float())  # [streams, W - 1, channels]
    y = torch.zeros_like(x)
    for j in range(W):
        back = W - 1 - j
        before = past[stream, (at + j).clamp_max(W - 2)]
        y = y + s["weight"][:, j] * torch.where((at >= back)[:, None], x[(t - back).clamp_min(0)], before)
    last = length[:, None] - (W - 1) + torch.arange(W - 1, device="cuda")  # the positions that a slot keeps
    inside = x[(begin[:, None] + last).clamp(0, T - 1)]
    older = past[torch.arange(N, device="cuda")[:, None], (last + W - 1).clamp_max(W - 2)]
    tails[slots] = torch.where((last >= 0)[..., None], inside, older).to(tails.dtype)
    return {"y": _silu(y).to(s["x"].dtype), "tails": tails}


def work(case):
    size = {"none": 0, "fp8": 1, "bf16": 2, "fp32": 4}
    if case["op"] == "norm":
        n = case["tokens"] * case["heads"] * case["dim"]
        each = size[case["x"]] * (2 if case["gate"] else 1) + 2 * size[case["residual"]] + size[case["to"]]
        return {"bytes": n * each + 4 * case["dim"] + (4 * case["tokens"] if case["to"] == "fp8" else 0), "flops": 8 * n}
    if case["op"] == "linear":
        T, K, M = case["tokens"], case["inputs"], case["outputs"]
        N = M * (2 if case["activation"] == "swiglu" else 1)
        scales = 4 * (T + N) if case["operands"] == "fp8" else 0
        return {"bytes": (T + N) * K * size[case["operands"]] + T * M * (size[case["to"]] + size[case["residual"]]) +
                (4 * N if case["bias"] else 0) + scales, "flops": 2 * T * N * K}
    C, W, T, N = case["channels"], case["width"], sum(_lengths(case)), case["streams"]
    # a new conversation's last inputs are written only
    kept = (2 * N - (len(range(0, N, 2)) if case["longest"] > 1 else 0)) * (W - 1) * C * size[case["tail"]]
    return {"bytes": 2 * T * C * size[case["dtype"]] + 4 * C * W + kept, "flops": 2 * T * C * W}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        h = s["x"].double()
        if s["residual"] is not None:
            h += s["residual"].double()
        y = torch.einsum("...d,...,d->...d", h, (h.pow(2).sum(-1) / case["dim"] + 1e-6).rsqrt(), s["weight"].double())
        if s["gate"] is not None:
            y = y * s["gate"].double() * torch.sigmoid(s["gate"].double())
        out = {"y": y}
        if case["to"] == "fp8":
            out["scales"] = torch.linalg.vector_norm(y.flatten(1), float("inf"), dim=1) / LARGEST
            out["y"] = torch.einsum("t...,t->t...", y, 1 / out["scales"])
        if s["residual"] is not None:
            out["residual"] = h
        return out
    if case["op"] == "linear":
        x, w = s["x"].double(), s["w"].double()
        if s["x_scales"] is not None:
            x, w = (torch.einsum("rk,r->rk", a, b.double()) for a, b in ((x, s["x_scales"]), (w, s["w_scales"])))
        y = torch.einsum("tk,nk->tn", x, w)
        if s["bias"] is not None:
            y += s["bias"].double()
        half = case["outputs"]
        if case["activation"] == "swiglu":
            y = y[:, :half] * torch.sigmoid(y[:, :half]) * y[:, half:]
        elif case["activation"] == "silu":
            y = y * torch.sigmoid(y)
        elif case["activation"] == "gelu":
            y = y * torch.special.ndtr(y)
        return {"y": y if s["residual"] is None else y + s["residual"].double()}
    W, tails = case["width"], s["tails"].double()
    y, bounds = [], s["starts"].tolist()
    for n, slot in enumerate(s["slots"].tolist()):
        old = torch.zeros_like(tails[slot]) if bool(s["fresh"][n]) else tails[slot].clone()
        line = torch.cat([old, s["x"][bounds[n]:bounds[n + 1]].double()])
        y.append(torch.einsum("tcj,cj->tc", line.unfold(0, W, 1), s["weight"].double()))
        tails[slot] = line[len(line) - (W - 1):]
    y = torch.cat(y)
    return {"y": y * torch.sigmoid(y), "tails": tails}
