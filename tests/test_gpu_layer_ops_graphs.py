"""The layer operators in captured graphs of more than one branch, and in
several graphs at once: launches overlap within a branch, results do not."""
import pytest
import torch

from test_gpu_layer_ops import BF16, E4M3, F32, operands, rand

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from gateddeltanet_b200 import build
    build.build()
    from gateddeltanet_b200 import ops
    return ops


def captured(body):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        body()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        body()
    return graph


@pytest.mark.parametrize("tokens", [1, 40, 600])
def test_two_branches(ops, tokens):
    """A norm and a convolution on two streams, joined by a product of both, forked again: first and last in the graph, after a
    copy, after a fork and after a join."""
    x, source = torch.zeros(tokens, 512, device="cuda", dtype=BF16), rand(tokens, 512, dtype=BF16)
    w, taps, tails = operands(1, 1024, 512, False)["weight"], rand(512, 4, seed=3), torch.zeros(tokens, 3, 512, device="cuda")
    both, y, z = torch.zeros(tokens, 1024, device="cuda", dtype=BF16), torch.zeros(tokens, 512, device="cuda", dtype=BF16), torch.zeros(tokens, 512, device="cuda")
    y8, scales = torch.zeros(tokens, 512, device="cuda").to(E4M3), torch.zeros(tokens, device="cuda")
    other = torch.cuda.Stream()

    def body():
        x.copy_(source)
        other.wait_stream(torch.cuda.current_stream())
        ops.rms_norm(x, out=both[:, :512])
        with torch.cuda.stream(other):
            ops.short_conv(x, taps, tails, out=both[:, 512:])
        torch.cuda.current_stream().wait_stream(other)
        ops.linear(both, w, activation="gelu", out=y)
        other.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(other):
            ops.rms_norm(y, out=y8, scales=scales)
        ops.linear(y, w[:, :512], out=z, dtype=F32)
        torch.cuda.current_stream().wait_stream(other)
    results = (both, y, z, y8, scales, tails)
    graph = captured(body)
    for seed in range(4):
        source.copy_(rand(tokens, 512, seed=seed, dtype=BF16))
        tails.zero_()
        body()
        torch.cuda.synchronize()
        want = [t.clone() for t in results]
        for t in results:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a.float(), b.float()) for a, b in zip(results, want))


def test_graphs_at_once(ops):
    """Two graphs of the same calls on their own buffers, replayed on two streams at the same time."""
    def calls(seed):
        residual, x8 = rand(300, 2048, seed=seed), torch.zeros(300, 2048, device="cuda").to(E4M3)
        scales, a = torch.zeros(300, device="cuda"), operands(300, 2048, 1024, True, seed=seed + 1)
        mid, down = torch.zeros(300, 512, device="cuda", dtype=BF16), operands(1, 512, 2048, False, seed=seed + 2)["weight"]

        def body():
            ops.rms_norm(residual, out=x8, scales=scales)
            ops.linear(x8, a["weight"], activation="swiglu", x_scales=scales, weight_scales=a["weight_scales"], out=mid)
            ops.linear(mid, down, residual=residual, out=residual)
        return body, residual
    (one, r1), (two, r2) = calls(1), calls(11)
    before = r1.clone(), r2.clone()
    graphs = captured(one), captured(two)
    r1.copy_(before[0]), r2.copy_(before[1])
    for _ in range(6):
        one(), two()
    torch.cuda.synchronize()
    want = r1.clone(), r2.clone()
    streams = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        r1.copy_(before[0]), r2.copy_(before[1])
        torch.cuda.synchronize()
        for _ in range(6):
            for s, g in zip(streams, graphs):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        assert torch.equal(r1, want[0]) and torch.equal(r2, want[1])
