"""A small server on the serving operators (gateddeltanet_b200/ops.py).

Gated-delta-rule layers with random weights: the prompts of a ragged batch go
through delta_chunk, every new token through delta_step on the same pooled
states, and the logits of each step through constrain_logits, which also picks
the next token. Token table, states and logits stay on the device.

    python examples/serve.py [--streams 8] [--layers 4] [--new 64]
"""
from __future__ import annotations

import argparse
import os
import sys
from typing import List, Optional

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from gateddeltanet_b200 import ops  # noqa: E402


class Model:
    """Embedding, `layers` gated-delta-rule mixers, tied LM head."""

    def __init__(self, vocab: int = 32000, hidden: int = 2048, layers: int = 4, heads: int = 8, head_dim: int = 256, seed: int = 1):
        gen = torch.Generator("cuda").manual_seed(seed)

        def weight(*shape):
            return (torch.randn(shape, generator=gen, device="cuda") * shape[-1] ** -0.5).bfloat16()

        self.vocab, self.heads, self.head_dim = vocab, heads, head_dim
        width = heads * head_dim
        self.embedding = weight(vocab, hidden)
        self.layers = [dict(qkvg=weight(4 * width, hidden), ab=weight(2 * heads, hidden), o=weight(hidden, width),
                            a_log=torch.rand(heads, generator=gen, device="cuda") * 2) for _ in range(layers)]

    def states(self, slots: int) -> List[torch.Tensor]:
        """A pool of states for each layer."""
        return [torch.zeros(slots, self.heads, self.head_dim, self.head_dim, device="cuda") for _ in self.layers]

    def forward(self, tokens: torch.Tensor, states, slots, starts: Optional[torch.Tensor] = None,
                fresh: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Hidden vectors of packed tokens: prompts (starts given) or one new token of each stream."""
        x = self.embedding[tokens.long()]
        rule = ops.delta_step if starts is None else ops.delta_chunk
        for layer, state in zip(self.layers, states):
            h = F.rms_norm(x, x.shape[-1:])
            q, k, v, gate = (h @ layer["qkvg"].T).unflatten(1, (4, self.heads, self.head_dim)).unbind(1)
            a, b = (h @ layer["ab"].T).float().chunk(2, dim=1)
            o = rule(q, k, v, -layer["a_log"].exp() * F.softplus(a - 4), torch.sigmoid(b), state, starts=starts, slots=slots,
                     fresh=fresh, normalize=True)
            x = x + (F.rms_norm(o, o.shape[-1:]) * F.silu(gate)).flatten(1) @ layer["o"].T
        return F.rms_norm(x, x.shape[-1:])

    def logits(self, hidden: torch.Tensor) -> torch.Tensor:
        return hidden @ self.embedding.T


@torch.no_grad()
def generate(model: Model, prompts: List[List[int]], new: int, masks: Optional[torch.Tensor] = None, repetition: float = 1.2,
             frequency: float = 0.1, presence: float = 0.1, bias: Optional[dict] = None):
    """Greedy continuation of each prompt by `new` tokens under penalties,
    biases {token: value} and masks (int32 [streams, ceil(vocab / 32)], bit set
    = allowed). A stream whose constraints leave no token ends there. Returns
    (table of all tokens, lengths, states)."""
    n = len(prompts)
    lengths = [len(p) for p in prompts]
    if not lengths or min(lengths) == 0:
        raise ValueError("a prompt of at least one token is needed for each stream")
    device = "cuda"
    table = torch.zeros(n, max(lengths) + new, dtype=torch.int32, device=device)
    for i, p in enumerate(prompts):
        table[i, :len(p)] = torch.tensor(p, dtype=torch.int32)
    prompt_lens = torch.tensor(lengths, dtype=torch.int32, device=device)
    lens = prompt_lens.clone()
    starts = F.pad(prompt_lens.cumsum(0), (1, 0)).int()
    slots = torch.randperm(n, device=device).int()
    each = lambda value: torch.full((n,), value, device=device)  # noqa: E731
    penalties = dict(repetition=each(repetition), frequency=each(frequency), presence=each(presence))
    if bias:
        penalties["bias_ids"] = torch.tensor([list(bias)] * n, dtype=torch.int32, device=device)
        penalties["bias"] = torch.tensor([list(bias.values())] * n, dtype=torch.float32, device=device)
    states = model.states(n)
    packed = torch.cat([table[i, :m] for i, m in enumerate(lengths)])
    hidden = model.forward(packed, states, slots, starts=starts, fresh=torch.ones(n, dtype=torch.bool, device=device))
    hidden = hidden[starts[1:].long() - 1]
    rows = torch.arange(n, device=device)
    going = torch.ones(n, dtype=torch.bool, device=device)
    for step in range(new):
        logits = model.logits(hidden)
        _, picks = ops.constrain_logits(logits, tokens=table, lens=lens, prompt_lens=prompt_lens, mask=masks, out=logits,
                                        **penalties)
        going &= picks >= 0
        picks = torch.where(going, picks, 0)
        table[rows, lens.long()] = picks
        lens += going
        if step + 1 < new:
            # slot -1: a stream that has ended stays in the batch, but its states do not change
            hidden = model.forward(picks, states, torch.where(going, slots, -1))
    return table, lens, [s[slots.long()] for s in states]


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--streams", type=int, default=8)
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--new", type=int, default=64)
    args = ap.parse_args()
    model = Model(layers=args.layers)
    gen = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, model.vocab, (int(torch.randint(1, 500, (1,), generator=gen)),), generator=gen).tolist()
               for _ in range(args.streams)]
    generate(model, prompts, 2)
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    begin.record()
    table, lens, _ = generate(model, prompts, args.new)
    end.record()
    torch.cuda.synchronize()
    for i in range(min(3, args.streams)):
        print(f"stream {i}: {len(prompts[i])} prompt tokens, then {table[i, len(prompts[i]):int(lens[i])].tolist()[:12]} ...")
    print(f"{args.streams} streams, {sum(map(len, prompts))} prompt tokens and {args.new} new ones each: "
          f"{begin.elapsed_time(end):.1f} ms")


if __name__ == "__main__":
    main()
