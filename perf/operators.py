"""Operators of a serving step on device tensors: what is measured, in plain torch and through the framework.

  step    the gated delta rule for the new token (or the few tokens) of every decode stream, states in a pool of slots
  chunk   the gated delta rule over the prompts of a ragged batch, states in the same pool
  logits  penalties for repeated tokens, biases and a grammar mask on the logits of every stream, and the greedy pick

Per value head, with the state S [V][K] in FP32:  S' = e^g S,  d = beta (v - S' k),  S = S' + d k^T,  o = scale S q.
"""
import random

import torch

own = False

CHUNK = 64  # tokens the plain prompt form takes at once


def listed():
    model = dict(heads=8, v_heads=8, key_dim=256, value_dim=256)  # the head layout of GDN-1.3B
    return [
        # one conversation, one new token: latency of the smallest call
        dict(name="step, 1 stream", op="step", streams=1, longest=1, spread=0, dtype="bf16", normalize=True, **model),
        # the framework's usual number of streams a GPU
        dict(name="step, 64 streams", op="step", streams=64, longest=1, spread=0, dtype="bf16", normalize=True, **model),
        # a full server
        dict(name="step, 256 streams", op="step", streams=256, longest=1, spread=0, dtype="fp32", normalize=True, **model),
        # drafted tokens checked: 0 to 6 a stream, more value heads than key heads
        dict(name="step, drafts of 27", op="step", streams=27, longest=6, spread=11, dtype="fp32", normalize=False,
             heads=4, v_heads=12, key_dim=128, value_dim=128),
        # a short prompt, one token over a chunk
        dict(name="chunk, 65 tokens", op="chunk", streams=1, longest=65, spread=0, dtype="bf16", normalize=True, **model),
        # the benchmark's prompt
        dict(name="chunk, 4096 tokens", op="chunk", streams=1, longest=4096, spread=0, dtype="bf16", normalize=True, **model),
        # prompts of very different lengths, some slots without any token
        dict(name="chunk, 24 ragged", op="chunk", streams=24, longest=2047, spread=5, dtype="bf16", normalize=True, **model),
        # smaller heads, grouped, q and k normalised by the caller
        dict(name="chunk, 8 x 1000 grouped", op="chunk", streams=8, longest=1000, spread=0, dtype="bf16", normalize=False,
             heads=4, v_heads=8, key_dim=128, value_dim=128),
        # one conversation's logits
        dict(name="logits, 1 row", op="logits", rows=1, vocab=32000, history=300, biases=16, dtype="fp32"),
        # the usual number of streams, long conversations
        dict(name="logits, 64 rows", op="logits", rows=64, vocab=32000, history=4096, biases=32, dtype="fp32"),
        # a full server with a large vocabulary
        dict(name="logits, 256 large rows", op="logits", rows=256, vocab=131072, history=8192, biases=64, dtype="bf16"),
        # odd sizes: rows that start at any alignment
        dict(name="logits, 19 odd rows", op="logits", rows=19, vocab=32003, history=777, biases=5, dtype="fp32"),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    op = rng.choice(("step", "chunk", "logits"))
    if op == "logits":
        rows = _log_int(rng, 1, 256)
        vocab = _log_int(rng, 1000, 131072)
        return dict(op=op, rows=rows, vocab=vocab, history=_log_int(rng, 1, 8192), biases=_log_int(rng, 1, 64),
                    dtype=rng.choice(("fp32", "bf16")))
    heads = rng.choice((1, 2, 3, 4, 8))
    group = rng.choice((1, 1, 2, 3)) if heads <= 4 else 1
    case = dict(op=op, heads=heads, v_heads=heads * group, key_dim=rng.choice((64, 128, 256)),
                value_dim=rng.choice((64, 128, 256)), normalize=rng.random() < 0.5)
    if op == "step":
        longest = rng.choice((1, 1, 2, 3, 6))
        return dict(case, streams=_log_int(rng, 1, 256), longest=longest, spread=rng.randrange(1, 1000) if longest > 1 else 0,
                    dtype=rng.choice(("fp32", "bf16")))
    longest = _log_int(rng, 1, 4096)
    streams = _log_int(rng, 1, max(1, min(48, 24000 // longest)))
    return dict(case, streams=streams, longest=longest, spread=rng.randrange(1, 1000) if streams > 1 else 0, dtype="bf16")


def _lengths(case):
    """Tokens of every stream: all `longest`, or, with a spread, from none to `longest`."""
    n, longest = case["streams"], case["longest"]
    if not case["spread"]:
        return [longest] * n
    rng = random.Random(case["spread"])
    return [rng.randint(0, longest) for _ in range(n - 1)] + [longest]


def _dtype(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(dev).manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=gen, device=dev)

    if case["op"] == "logits":
        B, V, L, M = case["rows"], case["vocab"], case["history"], case["biases"]
        logits = (normal(B, V) * 3).to(_dtype(case))
        tokens = torch.randint(0, V, (B, L), generator=gen, device=dev, dtype=torch.int32)
        recent = torch.randint(0, min(V, 50), (B, L), generator=gen, device=dev, dtype=torch.int32)  # texts repeat words
        tokens = torch.where(torch.rand((B, L), generator=gen, device=dev) < 0.5, recent, tokens)
        lens = torch.randint(0, L + 1, (B,), generator=gen, device=dev, dtype=torch.int32)
        prompt = (lens * torch.rand((B,), generator=gen, device=dev)).to(torch.int32)
        uniform = torch.rand((B, 3), generator=gen, device=dev)
        first = torch.randint(0, V, (B, 1), generator=gen, device=dev)
        bias_ids = ((first + torch.arange(M, device=dev) * max(1, V // M)) % V).to(torch.int32)
        bias_ids[:, M // 2 + 1:] = -1  # entries a row does not use
        mask = torch.randint(-2 ** 31, 2 ** 31, (B, (V + 31) // 32), generator=gen, device=dev).to(torch.int32)
        mask[::3] = -1  # rows without a grammar
        if B > 4:
            mask[4] = 0  # a grammar that allows nothing
        return dict(case=case, logits=logits, out=torch.empty_like(logits), tokens=tokens, lens=lens, prompt=prompt,
                    repetition=1 + uniform[:, 0].contiguous(), presence=uniform[:, 1].contiguous(),
                    frequency=0.3 * uniform[:, 2].contiguous(), bias_ids=bias_ids, bias=normal(B, M) * 2, mask=mask)

    H, HV, K, V, dt = case["heads"], case["v_heads"], case["key_dim"], case["value_dim"], _dtype(case)
    lengths = _lengths(case)
    N, T = len(lengths), sum(lengths)
    pool = N + 3
    q, k = normal(T, H, K), normal(T, H, K)
    if not case["normalize"]:
        q, k = (x / x.norm(dim=-1, keepdim=True) for x in (q, k))
    v = normal(T, HV, V)
    g = -torch.nn.functional.softplus(normal(T, HV) - 4)  # log decay
    beta = torch.sigmoid(normal(T, HV))
    starts = torch.tensor([0] + lengths, device=dev).cumsum(0).to(torch.int32)
    slots = torch.randperm(pool, generator=gen, device=dev)[:N].to(torch.int32)
    fresh = torch.zeros(N, device=dev, dtype=torch.bool)
    if case["op"] == "chunk":
        fresh[::2] = True  # new conversations; the others go on from their state
    state = normal(pool, HV, V, K) * 0.1
    return dict(case=case, q=q.to(dt), k=k.to(dt), v=v.to(dt), g=g, beta=beta, state=state, starts=starts, slots=slots,
                fresh=fresh, longest=max(lengths), one_each=max(lengths) == min(lengths) == 1)


def run(s):
    case = s["case"]
    if own:
        from gateddeltanet_b200 import ops
        if case["op"] == "logits":
            out, picks = ops.constrain_logits(
                s["logits"], tokens=s["tokens"], lens=s["lens"], prompt_lens=s["prompt"], repetition=s["repetition"],
                presence=s["presence"], frequency=s["frequency"], bias_ids=s["bias_ids"], bias=s["bias"],
                mask=s["mask"], out=s["out"])
            return {"logits": out, "picks": picks}
        rule = ops.delta_step if case["op"] == "step" else ops.delta_chunk
        o = rule(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"], starts=None if s["one_each"] else s["starts"],
                 slots=s["slots"], fresh=s["fresh"], normalize=case["normalize"])
        return {"o": o, "state": s["state"]}
    if case["op"] == "logits":
        return _plain_logits(s)
    return _plain_step(s) if case["op"] == "step" else _plain_chunk(s)


def _unit(x, on):
    x = x.float()
    return x / (x.square().sum(-1, keepdim=True) + 1e-6).sqrt() if on else x


def _padded(s, length):
    """Row of every (stream, position) in the packed tensors, and whether there is one."""
    at = s["starts"][:-1, None] + torch.arange(length, device="cuda")
    have = at < s["starts"][1:, None]
    return torch.where(have, at, 0).long(), have


def _inputs(s, length):
    """q, k, v [N, HV, length, .], g and beta [N, HV, length] in 32 bits: zeros where a stream has no token."""
    case = s["case"]
    at, have = _padded(s, length)
    group = case["v_heads"] // case["heads"]
    q = _unit(s["q"], case["normalize"]).repeat_interleave(group, 1) * case["key_dim"] ** -0.5
    k = _unit(s["k"], case["normalize"]).repeat_interleave(group, 1)
    q, k, v = (torch.where(have[..., None, None], x[at], 0.0).transpose(1, 2) for x in (q, k, s["v"].float()))
    g, beta = (torch.where(have[..., None], x[at], 0.0).transpose(1, 2) for x in (s["g"], s["beta"]))
    S = torch.where(s["fresh"][:, None, None, None], 0.0, s["state"][s["slots"].long()])
    return at, have, q, k, v, g, beta, S


def _outputs(s, have, o, S):
    """o [N, HV, length, V] back to packed rows, and the states to their slots."""
    s["state"][s["slots"].long()] = S
    return {"o": o.transpose(1, 2)[have].to(s["v"].dtype), "state": s["state"]}


def _plain_step(s):
    at, have, q, k, v, g, beta, S = _inputs(s, s["longest"])
    o = torch.empty_like(v)
    for t in range(s["longest"]):
        S = S * g[:, :, t, None, None].exp()
        d = beta[:, :, t, None] * (v[:, :, t] - (S @ k[:, :, t, :, None]).squeeze(-1))
        S = S + d[..., None] * k[:, :, t, None, :]
        o[:, :, t] = (S @ q[:, :, t, :, None]).squeeze(-1)
    return _outputs(s, have, o, S)


def _plain_chunk(s):
    length = -(-s["longest"] // CHUNK) * CHUNK
    at, have, q, k, v, g, beta, S = _inputs(s, length)
    N, HV = g.shape[:2]
    q, k, v, g, beta = (x.unflatten(2, (-1, CHUNK)) for x in (q, k, v, g, beta))
    G = g.cumsum(-1)
    lower = torch.ones(CHUNK, CHUNK, device="cuda", dtype=torch.bool).tril()
    decay = torch.where(lower, G[..., :, None] - G[..., None, :], float("-inf")).exp()
    A = (beta[..., None] * decay * (k @ k.transpose(-1, -2))).tril(-1)
    eye = torch.eye(CHUNK, device="cuda")
    inverse, power = eye - A, A
    for _ in range(5):  # (I + A)^-1 = (I - A)(I + A^2)(I + A^4)...: A^64 = 0
        power = power @ power
        inverse = inverse + inverse @ power
    P = decay * (q @ k.transpose(-1, -2))
    o = torch.empty_like(v)
    for c in range(length // CHUNK):
        at0 = G[:, :, c, :, None].exp()
        d = inverse[:, :, c] @ (beta[:, :, c, :, None] * (v[:, :, c] - at0 * (k[:, :, c] @ S.transpose(-1, -2))))
        o[:, :, c] = at0 * (q[:, :, c] @ S.transpose(-1, -2)) + P[:, :, c] @ d
        to_end = (G[:, :, c, -1:] - G[:, :, c]).exp()[..., None]
        S = S * at0[:, :, -1:] + (to_end * d).transpose(-1, -2) @ k[:, :, c]
    return _outputs(s, have, o.flatten(2, 3), S)


def _plain_logits(s):
    x = s["logits"].float()
    B, V = x.shape
    ids, at = s["tokens"].long(), torch.arange(s["tokens"].shape[1], device="cuda")
    there = (at < s["lens"][:, None]) & (ids >= 0) & (ids < V)
    ids = torch.where(there, ids, V)
    seen = torch.zeros(B, V + 1, device="cuda", dtype=torch.int32).scatter_add(1, ids, there.int())[:, :V] > 0
    made = (there & (at >= s["prompt"][:, None])).int()
    n = torch.zeros(B, V + 1, device="cuda", dtype=torch.int32).scatter_add(1, ids, made)[:, :V]
    r, f, p = (s[name][:, None] for name in ("repetition", "frequency", "presence"))
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = torch.where(n > 0, x - f * n - p, x)
    used = (s["bias_ids"] >= 0) & (s["bias_ids"] < V)
    x = x + torch.zeros(B, V + 1, device="cuda").scatter_add(1, torch.where(used, s["bias_ids"], V).long(),
                                                             torch.where(used, s["bias"], 0.0))[:, :V]
    v = torch.arange(V, device="cuda")
    allowed = (s["mask"][:, v // 32] >> (v % 32)) & 1
    x = torch.where(allowed > 0, x, float("-inf")).to(s["logits"].dtype)
    y = torch.where(x.isnan(), float("-inf"), x.float())
    top = y.amax(1, keepdim=True)
    pick = torch.where((y == top) & (top > float("-inf")), v, V).amin(1)
    return {"logits": x, "picks": torch.where(pick == V, -1, pick).int()}


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "logits":
        B, V, L, M = case["rows"], case["vocab"], case["history"], case["biases"]
        # a history is half full on average
        return {"bytes": B * (2 * V * size + V / 8 + 4 * L / 2 + 8 * M + 24), "flops": 2 * B * V}
    H, HV, K, V = case["heads"], case["v_heads"], case["key_dim"], case["value_dim"]
    lengths = _lengths(case)
    T = sum(lengths)
    fresh = 0 if case["op"] == "step" else len(lengths[::2])  # a new conversation's state is written only
    states = (2 * len(lengths) - fresh) * HV * V * K * 4
    return {"bytes": T * ((2 * H * K + 2 * HV * V) * size + 8 * HV) + states, "flops": T * HV * (6 * K * V + 4 * V)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logits":
        return _exact_logits(s)
    group = case["v_heads"] // case["heads"]
    q, k, v, g, beta, state = (s[name].double() for name in ("q", "k", "v", "g", "beta", "state"))
    if case["normalize"]:
        q, k = (x * (x.pow(2).sum(-1, keepdim=True) + 1e-6).rsqrt() for x in (q, k))
    o = torch.zeros_like(v)
    starts, slots = s["starts"].tolist(), s["slots"].tolist()
    for n, fresh in enumerate(s["fresh"].tolist()):
        if fresh:
            state[slots[n]] = 0
    for t in range(s["longest"]):  # the t-th token of every stream that has one
        at = [starts[n] + t for n in range(len(slots)) if starts[n] + t < starts[n + 1]]
        to = [slots[n] for n in range(len(slots)) if starts[n] + t < starts[n + 1]]
        qt, kt = (x[at].repeat_interleave(group, 1) for x in (q, k))
        S = g[at].exp()[..., None, None] * state[to]
        error = v[at] - torch.einsum("nhvk,nhk->nhv", S, kt)
        S = S + torch.einsum("nhv,nhk->nhvk", beta[at][..., None] * error, kt)
        o[at] = torch.einsum("nhvk,nhk->nhv", S, qt) / case["key_dim"] ** 0.5
        state[to] = S
    return {"o": o, "state": state}


def _exact_logits(s):
    x = s["logits"].double().cpu()
    B, V = x.shape
    tokens, lens, prompt, ids, bias = (s[name].cpu() for name in ("tokens", "lens", "prompt", "bias_ids", "bias"))
    word = torch.arange(V) // 32
    for b in range(B):
        n, m = int(lens[b]), int(prompt[b])
        past = torch.bincount(tokens[b, :n].long(), minlength=V)
        made = torch.bincount(tokens[b, m:n].long(), minlength=V)
        r, p, f = (float(s[name][b]) for name in ("repetition", "presence", "frequency"))
        row = x[b]
        row[past > 0] *= torch.where(row > 0, 1 / r, r)[past > 0]
        row -= f * made.double() + p * (made > 0).double()
        use = ids[b] >= 0
        row.index_add_(0, ids[b][use].long(), bias[b][use].double())
        row[((s["mask"][b].cpu()[word] >> (torch.arange(V) % 32)) & 1) == 0] = float("-inf")
    return {"logits": x, "picks": None}
