"""A small server on the serving operators (gateddeltanet_b200/ops.py).

Gated-delta-rule layers with random weights, each made of the operators: norm,
projection, short convolution, delta rule, gated norm and projection onto the
residual, norm, gate and up projection, projection onto the residual. The
prompts of a ragged batch go through delta_chunk, every new token through
delta_step on the same pooled states and last inputs, and the logits of each
step through constrain_logits, which also picks the next token. Token table,
states and logits stay on the device. With 8-bit weights the norms give 8-bit
activations with a scale for each token.

    python examples/serve.py [--streams 8] [--layers 4] [--new 64] [--eight-bits]
"""
from __future__ import annotations

import argparse
import os
import sys
from typing import List, Optional, Tuple

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from gateddeltanet_b200 import ops  # noqa: E402


E4M3 = torch.float8_e4m3fn


def aligned(n: int, columns: int, dtype: torch.dtype) -> torch.Tensor:
    """[n, columns] whose rows start on 16-byte boundaries, as ops.linear takes them."""
    return torch.empty(n, -(-columns // 16) * 16, dtype=dtype, device="cuda")[:, :columns]


def room(n: int, columns: int, dtype: torch.dtype) -> Optional[torch.Tensor]:
    """Such rows for a result that ops.linear reads; None where it has them by itself."""
    return None if columns % 16 == 0 else aligned(n, columns, dtype)


class Model:
    """Embedding, `layers` gated-delta-rule layers with their MLPs, tied LM head."""

    def __init__(self, vocab: int = 32000, hidden: int = 2048, layers: int = 4, heads: int = 8, head_dim: int = 256, seed: int = 1,
                 intermediate: Optional[int] = None, eight_bits: bool = False):
        gen = torch.Generator("cuda").manual_seed(seed)

        def weight(*shape):
            return aligned(*shape, torch.bfloat16).copy_(torch.randn(shape, generator=gen, device="cuda") * shape[-1] ** -0.5)

        def projection(rows, columns):
            """Arguments of ops.linear: a weight, in 8 bits with the scales of its rows."""
            w = weight(rows, columns)
            if not eight_bits:
                return dict(weight=w)
            scales = w.float().abs().amax(1) / 448
            return dict(weight=aligned(*w.shape, E4M3).copy_(w.float() / scales[:, None]), weight_scales=scales)

        self.vocab, self.heads, self.head_dim, self.eight_bits = vocab, heads, head_dim, eight_bits
        width = heads * head_dim
        inner = intermediate or max(16, hidden * 11 // 64 * 16)  # 5632 of 2048
        ones = lambda n: torch.ones(n, device="cuda")  # noqa: E731
        self.embedding = weight(vocab, hidden)
        self.layers = [dict(
            attn_norm=ones(hidden), o_norm=ones(head_dim), mlp_norm=ones(hidden),
            # q, k, v, gate and the two gates' rows; whole 16-byte rows of the result
            qkvgab=projection(-(-(4 * width + 2 * heads) // 8) * 8, hidden),
            conv=(torch.rand(3 * width, 4, generator=gen, device="cuda") - 0.5), o=projection(hidden, width),
            gate_up=projection(2 * inner, hidden), down=dict(weight=weight(hidden, inner)),
            a_log=torch.rand(heads, generator=gen, device="cuda") * 2) for _ in range(layers)]
        self.norm = ones(hidden)

    def states(self, slots: int) -> List[Tuple[torch.Tensor, torch.Tensor]]:
        """For each layer a pool of states and one of the convolution's last inputs."""
        return [(torch.zeros(slots, self.heads, self.head_dim, self.head_dim, device="cuda"),
                 torch.zeros(slots, 3, 3 * self.heads * self.head_dim, device="cuda")) for _ in self.layers]

    def normed(self, x: torch.Tensor, weight: torch.Tensor, gate: Optional[torch.Tensor] = None) -> dict:
        """Arguments of ops.linear: the norm of x, in 8 bits for 8-bit weights."""
        dtype = E4M3 if self.eight_bits else torch.bfloat16
        y = ops.rms_norm(x, weight, gate=gate, dtype=dtype, out=room(*x.shape[-2:], dtype))
        return dict(x=y[0].flatten(1), x_scales=y[1]) if self.eight_bits else dict(x=y.flatten(1))

    def forward(self, tokens: torch.Tensor, states, slots, starts: Optional[torch.Tensor] = None,
                fresh: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Hidden vectors of packed tokens: prompts (starts given) or one new token of each stream."""
        residual = self.embedding[tokens.long()].float()
        rule = ops.delta_step if starts is None else ops.delta_chunk
        width = self.heads * self.head_dim
        sequences = dict(starts=starts, slots=slots, fresh=fresh)
        for layer, (state, tails) in zip(self.layers, states):
            qkvgab = ops.linear(**self.normed(residual, layer["attn_norm"]), **layer["qkvgab"])
            qkv = ops.short_conv(qkvgab[:, :3 * width], layer["conv"], tails, **sequences)
            q, k, v = qkv.unflatten(1, (3, self.heads, self.head_dim)).unbind(1)
            gate = qkvgab[:, 3 * width:4 * width].unflatten(1, (self.heads, self.head_dim))
            a, b = qkvgab[:, 4 * width:4 * width + 2 * self.heads].float().chunk(2, dim=1)
            o = rule(q, k, v, -layer["a_log"].exp() * F.softplus(a - 4), torch.sigmoid(b), state, normalize=True, **sequences)
            ops.linear(**self.normed(o, layer["o_norm"], gate), **layer["o"], residual=residual, out=residual)
            inner = ops.linear(**self.normed(residual, layer["mlp_norm"]), **layer["gate_up"], activation="swiglu",
                               out=room(len(residual), layer["down"]["weight"].shape[1], torch.bfloat16))
            ops.linear(inner, **layer["down"], residual=residual, out=residual)
        return ops.rms_norm(residual, self.norm, dtype=torch.bfloat16)

    def logits(self, hidden: torch.Tensor) -> torch.Tensor:
        if hidden.shape[1] % 16:
            hidden = aligned(*hidden.shape, hidden.dtype).copy_(hidden)
        return ops.linear(hidden, self.embedding, dtype=torch.float32)


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
    return table, lens, [state[slots.long()] for state, _ in states]


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--streams", type=int, default=8)
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--new", type=int, default=64)
    ap.add_argument("--eight-bits", action="store_true")
    args = ap.parse_args()
    model = Model(layers=args.layers, eight_bits=args.eight_bits)
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
