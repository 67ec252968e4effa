"""Plain 64-bit forms of the serving operators (gateddeltanet_b200/ops.py),
token by token and row by row from the formulas of include/gdn_b200.h."""
import math

import torch


def delta_rule(q, k, v, g, beta, state, starts=None, slots=None, fresh=None, scale=None, normalize=False):
    """(o, state) in float64 on the CPU; the inputs stay as they are."""
    q, k, v, g, beta, state = (x.detach().cpu().double() for x in (q, k, v, g, beta, state.clone()))
    tokens, heads, key_dim = q.shape
    group = v.shape[1] // heads
    starts = list(range(tokens + 1)) if starts is None else starts.tolist()
    n = len(starts) - 1
    slots = list(range(n)) if slots is None else slots.tolist()
    fresh = [False] * n if fresh is None else [bool(x) for x in fresh.tolist()]
    scale = key_dim ** -0.5 if scale is None else scale
    if normalize:
        q, k = (x / (x.square().sum(-1, keepdim=True) + 1e-6).sqrt() for x in (q, k))
    q, k = (x.repeat_interleave(group, 1) for x in (q, k))
    o = torch.zeros_like(v)
    for i in range(n):
        if not 0 <= slots[i] < state.shape[0]:
            continue
        S = torch.zeros_like(state[0]) if fresh[i] else state[slots[i]].clone()
        for t in range(max(0, min(starts[i], tokens)), max(0, min(starts[i + 1], tokens))):
            S = S * g[t].exp()[:, None, None]
            d = beta[t][:, None] * (v[t] - (S * k[t][:, None, :]).sum(-1))
            S = S + d[:, :, None] * k[t][:, None, :]
            o[t] = scale * (S * q[t][:, None, :]).sum(-1)
        state[slots[i]] = S
    return o, state


def constrain(logits, tokens=None, lens=None, prompt_lens=None, repetition=None, presence=None, frequency=None,
              bias_ids=None, bias=None, mask=None):
    """(values in float64 before the rounding to the logits' type) on the CPU."""
    x = logits.detach().cpu().double().clone()
    rows, vocab = x.shape
    for b in range(rows):
        if tokens is not None:
            n = tokens.shape[1] if lens is None else max(0, min(int(lens[b]), tokens.shape[1]))
            m = 0 if prompt_lens is None else int(prompt_lens[b])
            history = tokens[b, :n].tolist()
            made = {}
            for i, v in enumerate(history):
                if i >= m:
                    made[v] = made.get(v, 0) + 1
            for v in set(history):
                if not 0 <= v < vocab:
                    continue
                if repetition is not None:
                    r = float(repetition[b])
                    x[b, v] = x[b, v] / r if x[b, v] > 0 else x[b, v] * r
                if made.get(v):
                    if frequency is not None:
                        x[b, v] -= float(frequency[b]) * made[v]
                    if presence is not None:
                        x[b, v] -= float(presence[b])
        if bias is not None:
            for v, w in zip(bias_ids[b].tolist(), bias[b].tolist()):
                if 0 <= v < vocab:
                    x[b, v] += w
        if mask is not None:
            word = mask[b].tolist()
            gone = [v for v in range(vocab) if not (word[v // 32] >> (v % 32)) & 1]
            x[b, gone] = -math.inf
    return x


def greedy(values):
    """Lowest index of each row's largest value; NaN never, -1 if none is above -inf."""
    picks = []
    for row in values.detach().cpu().double().tolist():
        best, at = -math.inf, -1
        for v, y in enumerate(row):
            if y > best:
                best, at = y, v
        picks.append(at)
    return picks


def rel(x, y):
    """2-norm of the difference over the 2-norm of y; all values have to be finite."""
    x, y = x.detach().cpu().double(), y.double()
    assert x.shape == y.shape and bool(x.isfinite().all())
    norm = float(y.norm())
    off = float((x - y).norm())
    return off / norm if norm else off
