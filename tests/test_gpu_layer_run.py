"""The layer operators together, as a layer uses them: each link is held
against its 64-bit form on the values that the link before gave, for ragged
prompts and for single tokens; and the example server on them."""
import importlib.util
import os

import pytest
import torch

import layer_plain as plain
import ops_plain
from test_gpu_layer_ops import E4M3, check_eight, eight_bits, rand
from test_gpu_ops_delta import STATE_TOL

pytestmark = pytest.mark.gpu
REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIDDEN, HEADS, DIM, INNER = 256, 2, 64, 704
WIDTH = HEADS * DIM


@pytest.fixture(scope="module")
def ops():
    from gateddeltanet_b200 import build
    build.build()
    from gateddeltanet_b200 import ops
    return ops


class Layer:
    def __init__(self, eight):
        def projection(rows, columns, seed):
            w = rand(rows, columns, seed=seed) * columns ** -0.5
            if not eight:
                return dict(weight=w.bfloat16())
            w, s = eight_bits(w)
            return dict(weight=w, weight_scales=s)
        self.eight = eight
        self.norms = [1 + 0.1 * rand(n, seed=40 + i) for i, n in enumerate((HIDDEN, DIM, HIDDEN))]
        self.qkvgab, self.o = projection(4 * WIDTH + 8, HIDDEN, 1), projection(HIDDEN, WIDTH, 2)
        self.gate_up, self.down = projection(2 * INNER, HIDDEN, 3), dict(weight=(rand(HIDDEN, INNER, seed=4) * INNER ** -0.5).bfloat16())
        self.conv = rand(3 * WIDTH, 4, seed=5) * 0.5

    def run(self, ops, residual, state, tails, check, **sequences):
        """One layer on packed tokens; check(name, got, want, off) for each link."""
        def normed(x, weight, gate=None):
            if not self.eight:
                y = ops.rms_norm(x, weight, gate=gate, dtype=torch.bfloat16)
                if check:
                    want, _ = plain.norm(x, weight, None, gate)
                    check("norm", y, want, plain.norm_error(gate) * want.abs())
                return dict(x=y.flatten(1))
            y = ops.rms_norm(x, weight, gate=gate, dtype=E4M3)
            if check:
                want, _ = plain.norm(x, weight, None, gate)
                check_eight(y, want, plain.norm_error(gate) * want.abs())
            return dict(x=y[0].flatten(1), x_scales=y[1])

        def linear(out=None, residual=None, **a):
            want = plain.linear(**{n: v for n, v in a.items()}, residual=residual) if check else None
            y = ops.linear(**a, residual=residual, out=out)
            if check:
                check("linear", y, *want)
            return y

        qkvgab = linear(**normed(residual, self.norms[0]), **self.qkvgab)
        before = tails.clone()
        qkv = ops.short_conv(qkvgab[:, :3 * WIDTH], self.conv, tails, **sequences)
        if check:
            want, after, off = plain.conv(qkvgab[:, :3 * WIDTH], self.conv, before, **sequences)
            check("conv", qkv, want, off)
            assert torch.equal(tails.cpu().double(), after)
        q, k, v = qkv.unflatten(1, (3, HEADS, DIM)).unbind(1)
        a, b = qkvgab[:, 4 * WIDTH:4 * WIDTH + 2 * HEADS].float().chunk(2, 1)
        g, beta = -torch.nn.functional.softplus(a - 4), torch.sigmoid(b)
        old = state.clone()
        rule = ops.delta_step if sequences["starts"] is None else ops.delta_chunk
        o = rule(q, k, v, g, beta, state, normalize=True, **sequences)
        if check:
            _, want = ops_plain.delta_rule(q, k, v, g, beta, old, normalize=True, **sequences)
            assert ops_plain.rel(state, want) < STATE_TOL
        gate = qkvgab[:, 3 * WIDTH:4 * WIDTH].unflatten(1, (HEADS, DIM))
        linear(**normed(o, self.norms[1], gate), **self.o, residual=residual, out=residual)
        inner = linear(**normed(residual, self.norms[2]), **self.gate_up, activation="swiglu")
        linear(x=inner, **self.down, residual=residual, out=residual)
        return residual


@pytest.mark.parametrize("eight", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("lengths", [[70, 0, 1, 3, 150], [2, 1]], ids=str)
def test_a_layer(ops, eight, lengths):
    layer = Layer(eight)
    n = len(lengths)
    state, tails = torch.zeros(n + 1, HEADS, DIM, DIM, device="cuda"), rand(n + 1, 3, 3 * WIDTH, seed=7)
    slots = torch.randperm(n + 1, generator=torch.Generator().manual_seed(8))[:n].int().cuda()
    starts = torch.tensor([0] + lengths).cumsum(0).int().cuda()
    layer.run(ops, rand(sum(lengths), HIDDEN, seed=9), state, tails, plain_check, starts=starts, slots=slots,
              fresh=torch.ones(n, dtype=torch.bool, device="cuda"))
    for step in range(3):
        layer.run(ops, rand(n, HIDDEN, seed=10 + step), state, tails, plain_check, starts=None, slots=slots, fresh=None)


def plain_check(name, got, want, off):
    plain.check(got, want, off, name)


@pytest.mark.parametrize("eight", [False, True], ids=["bf16", "fp8"])
@pytest.mark.parametrize("streams", [3, 40])
def test_a_captured_layer(ops, eight, streams):
    """A graph of a step gives the bits of the calls, replay after replay, with new content in the same buffers."""
    layer = Layer(eight)
    inputs = [rand(streams, HIDDEN, seed=20 + i) for i in range(4)]
    slots = torch.arange(streams, device="cuda").int()

    def fresh_pools():
        return torch.zeros(streams, HEADS, DIM, DIM, device="cuda"), torch.zeros(streams, 3, 3 * WIDTH, device="cuda")
    state, tails = fresh_pools()
    want = [layer.run(ops, x.clone(), state, tails, None, starts=None, slots=slots, fresh=None) for x in inputs]
    pools = fresh_pools()
    buffer = inputs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer.run(ops, buffer, *pools, None, starts=None, slots=slots, fresh=None)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.run(ops, buffer, *pools, None, starts=None, slots=slots, fresh=None)
    for p in pools:
        p.zero_()
    for x, y in zip(inputs, want):
        buffer.copy_(x)
        graph.replay()
        assert torch.equal(buffer, y)
    assert torch.equal(pools[0], state) and torch.equal(pools[1], tails)


@pytest.fixture(scope="module")
def serve():
    spec = importlib.util.spec_from_file_location("serve", os.path.join(REPO, "examples", "serve.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_server_with_eight_bits(ops, serve):
    model = serve.Model(vocab=1003, hidden=256, layers=2, heads=2, head_dim=64, seed=3, eight_bits=True)
    gen = torch.Generator().manual_seed(4)
    prompts = [torch.randint(0, 1003, (n,), generator=gen).tolist() for n in (1, 70, 33)]
    table, lens, states = serve.generate(model, prompts, 5)
    assert lens.tolist() == [6, 75, 38] and all(bool(s.isfinite().all()) for s in states)
    assert all(table[i, :len(p)].tolist() == p for i, p in enumerate(prompts))


def test_command_with_eight_bits(ops, serve, capsys, monkeypatch):
    monkeypatch.setattr("sys.argv", ["serve.py", "--streams", "3", "--layers", "1", "--new", "3", "--eight-bits"])
    serve.main()
    assert "3 streams" in capsys.readouterr().out
