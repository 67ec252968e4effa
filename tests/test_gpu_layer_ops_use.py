"""The layer operators in the ways a program may call them: other streams,
several threads, parts of large buffers, waits that run out, what is refused."""
import threading

import pytest
import torch

import layer_plain as plain
from test_gpu_layer_ops import BF16, E4M3, F32, check_eight, operands, padded, rand

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from gateddeltanet_b200 import build
    build.build()
    from gateddeltanet_b200 import ops
    return ops


@pytest.mark.parametrize("tokens,outputs", [(64, 2048), (40, 33000), (3000, 1024)], ids=["a cluster", "many tiles", "two CTAs a tile"])
def test_a_wait_that_runs_out(ops, tokens, outputs):
    """One copy is left out: the call ends, says so, and leaves NaN where sums are missing and nothing wrong elsewhere."""
    import gateddeltanet_b200 as gdn
    a = operands(tokens, 2048, outputs, False)
    want = ops.linear(**a, dtype=F32)
    ops.linear_status()
    gdn.lib().gdn_b200_test_drop_copy(3)
    got = ops.linear(**a, dtype=F32)
    with pytest.raises(RuntimeError, match="ran out"):
        ops.linear_status()
    bad = got.isnan()
    assert bool(bad.any()) and torch.equal(got[~bad], want[~bad])
    ops.linear_status()
    assert torch.equal(ops.linear(**a, dtype=F32), want)


def calls(ops, seed):
    """One call of each, and their results."""
    x, w = rand(300, 512, seed=seed, dtype=BF16), rand(512, 4, seed=seed + 1)
    tails = rand(2, 3, 512, seed=seed + 2)
    starts = torch.tensor([0, 100, 300], dtype=torch.int32, device="cuda")
    proj = operands(300, 512, 1000, False, seed=seed + 3)
    few = operands(5, 512, 1000, True, seed=seed + 4)

    def run():
        t = tails.clone()
        y, s = ops.rms_norm(x, dtype=E4M3)
        return [y.float(), s, ops.linear(**proj), ops.linear(**few), ops.short_conv(x, w, t, starts=starts), t]
    return run


def test_several_streams(ops):
    runs = [calls(ops, 10 * i) for i in range(4)]
    want = [r() for r in runs]
    streams = [torch.cuda.Stream() for _ in runs]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        got = []
        for r, s in zip(runs, streams):
            with torch.cuda.stream(s):
                got.append(r())
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))


def test_several_threads(ops):
    runs = [calls(ops, 10 * i) for i in range(4)]
    want = [r() for r in runs]
    torch.cuda.synchronize()
    wrong = []

    def work(run, want):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                if not all(torch.equal(a, b) for a, b in zip(run(), want)):
                    wrong.append(1)
    threads = [threading.Thread(target=work, args=a) for a in zip(runs, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_results_of_the_call_before(ops):
    """A chain of calls in which each reads what the one before has written, over and over in the same buffers: launches
    overlap, results do not."""
    for tokens in (1, 40, 600):
        w = [operands(tokens, 1024, 1024, False, seed=i)["weight"] for i in range(3)]
        conv, tails = rand(1024, 4, seed=5), torch.zeros(tokens, 3, 1024, device="cuda")
        start = rand(tokens, 1024, seed=6)

        def chain(wait):
            residual = start.clone()
            x = torch.empty(tokens, 1024, device="cuda", dtype=BF16)
            y = torch.empty_like(x)
            t = tails.clone()
            for _ in range(4):
                for call in (lambda: ops.rms_norm(residual, out=x, dtype=BF16), lambda: ops.linear(x, w[0], out=y),
                             lambda: ops.short_conv(y, conv, t, out=x), lambda: ops.linear(x, w[1], activation="gelu", out=y),
                             lambda: ops.linear(y, w[2], residual=residual, out=residual)):
                    call()
                    if wait:
                        torch.cuda.synchronize()
            return residual, t
        want = chain(True)
        for _ in range(5):
            got = chain(False)
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_far_apart(ops):
    """Offsets past 32 bits: rows 2^27 elements apart, and more than 2^31 results."""
    step, tokens = 1 << 27, 20
    big = torch.empty(step * tokens, dtype=BF16, device="cuda")
    x = big.as_strided((tokens, 256), (step, 1))
    x.copy_(rand(tokens, 256))
    out = big.as_strided((tokens, 256), (step, 1), 1024)
    want, _ = plain.norm(x)
    plain.check(ops.rms_norm(x, out=out), want, plain.norm_error(None) * want.abs(), "norm")
    w = operands(1, 256, 256, False)["weight"]
    for n in (3, tokens):
        a = x[tokens - n:]
        want, off = plain.linear(a, w)
        plain.check(ops.linear(a, w, out=out[tokens - n:]), want, off, "linear")
    conv, tails = rand(256, 4, seed=3), torch.zeros(2, 3, 256, device="cuda")
    starts = torch.tensor([0, 11, 20], dtype=torch.int32, device="cuda")
    want, after, off = plain.conv(x, conv, tails, starts=starts)
    plain.check(ops.short_conv(x, conv, tails, starts=starts, out=out), want, off, "conv")
    assert torch.equal(tails.cpu().double(), after)
    pool = big.as_strided((tokens, 3, 256), (step, 256, 1), 4096)
    pool.copy_(rand(tokens, 3, 256, seed=4))
    want, after, off = plain.conv(x, conv, pool)
    plain.check(ops.short_conv(x, conv, pool, out=out), want, off, "conv, single tokens")
    assert torch.equal(pool.cpu().double(), after)
    del big, x, out, pool, a
    torch.cuda.empty_cache()
    x, w = rand(70000, 64, dtype=BF16), rand(32000, 64, seed=2, dtype=BF16)
    got = ops.linear(x, w)
    want, off = plain.linear(x[-3:], w)
    plain.check(got[-3:], want, off, "many results")


def test_written_tensors_get_a_version(ops):
    x, tails = rand(4, 64, dtype=BF16), torch.zeros(4, 3, 64, device="cuda")
    residual, out, scales = rand(4, 64), torch.empty(4, 64, device="cuda", dtype=E4M3), torch.empty(4, device="cuda")
    before = [t._version for t in (residual, out, scales, tails)]
    ops.rms_norm(x, residual=residual, out=out, scales=scales)
    ops.short_conv(x, rand(64, 4), tails)
    assert [t._version for t in (residual, out, scales, tails)] == [v + 1 for v in before]
    y = torch.empty(4, 64, device="cuda", dtype=BF16)
    ops.linear(x, rand(64, 64, dtype=BF16), out=y)
    assert y._version == 1
    with torch.inference_mode():
        ops.rms_norm(rand(4, 64), residual=rand(4, 64))


def test_refusals(ops):
    x, w = rand(8, 64, dtype=BF16), rand(64, 64, dtype=BF16)
    big = torch.zeros(8, 256, device="cuda", dtype=BF16)
    for call, error, reason in [
            (lambda: ops.rms_norm(x.T), ValueError, "not contiguous"),
            (lambda: ops.rms_norm(x, residual=x), RuntimeError, "overlaps"),
            (lambda: ops.rms_norm(x, residual=torch.zeros(1, 64, device="cuda").expand(8, 64)), ValueError, "overlap"),
            (lambda: ops.rms_norm(big[:, :64], out=big[:, 32:96]), RuntimeError, "overlaps"),
            (lambda: ops.rms_norm(x, dtype=torch.float16), ValueError, "not computed"),
            (lambda: ops.rms_norm(x, out=big[:, :64], dtype=F32), ValueError, "type"),
            (lambda: ops.rms_norm(x, scales=torch.zeros(8, device="cuda")), ValueError, "8-bit"),
            (lambda: ops.rms_norm(x, rand(64).cpu()), ValueError, "CUDA device"),
            (lambda: ops.rms_norm(rand(2, 16385)), RuntimeError, "more than one CTA"),
            (lambda: ops.linear(rand(8, 60, dtype=BF16), rand(64, 60, dtype=BF16)), RuntimeError, "16-byte"),
            (lambda: ops.linear(big[:, 1:65], w), RuntimeError, "16-byte"),
            (lambda: ops.linear(x[:1].expand(8, 64), w), RuntimeError, "overlap"),
            (lambda: ops.linear(x, w, out=x), RuntimeError, "overlaps"),
            (lambda: ops.linear(x, w, residual=big[:, :64], out=big[:, 8:72]), RuntimeError, "overlaps"),
            (lambda: ops.linear(x, w, x_scales=torch.ones(8, device="cuda")), ValueError, "8-bit"),
            (lambda: ops.linear(x.to(E4M3), w.to(E4M3)), ValueError, "need"),
            (lambda: ops.linear(x, w, dtype=E4M3), ValueError, "not computed"),
            (lambda: ops.linear(x, w, residual=rand(8, 32)), ValueError, "shape"),
            (lambda: ops.short_conv(x, rand(64, 5), torch.zeros(8, 4, 64, device="cuda")), RuntimeError, "width"),
            (lambda: ops.short_conv(x, rand(64, 4), torch.zeros(7, 3, 64, device="cuda")), RuntimeError, "slots"),
            (lambda: ops.short_conv(x, rand(4, 64).T, torch.zeros(8, 3, 64, device="cuda")), ValueError, "not contiguous"),
            (lambda: ops.short_conv(x.float(), rand(64, 4), torch.zeros(8, 3, 64, device="cuda", dtype=BF16)), RuntimeError, "tail_dtype"),
            (lambda: ops.short_conv(x, rand(64, 4), torch.zeros(1, 3, 64, device="cuda").expand(8, 3, 64)), RuntimeError, "tails overlap"),
            (lambda: ops.short_conv(x, rand(64, 4), torch.zeros(8, 3, 64, device="cuda"), out=x), RuntimeError, "overlaps"),
            (lambda: ops.short_conv(x, rand(64, 4), torch.zeros(8, 3, 64, device="cuda"), starts=torch.zeros(3, dtype=torch.int64, device="cuda")),
             ValueError, "type")]:
        with pytest.raises(error, match=reason):
            call()
    with pytest.raises(ValueError, match="CUDA device"):
        ops.linear_status("cpu")
    torch.zeros(3, device="cuda").add_(1).sum().item()  # no error is left behind


def test_interleaved_tensors_are_taken(ops):
    """Inputs, gate and results side by side in one buffer, row by row."""
    big = rand(30, 1024, dtype=BF16)
    x, gate, out = (big[:, i * 256:(i + 1) * 256] for i in range(3))
    want, _ = plain.norm(x, None, None, gate)
    plain.check(ops.rms_norm(x, gate=gate, out=out), want, plain.norm_error(gate) * want.abs())
    w = operands(1, 256, 256, False)["weight"]
    want, off = plain.linear(x, w)
    plain.check(ops.linear(x, w, out=big[:, 768:]), want, off)
    y, s = ops.rms_norm(x.unflatten(1, (4, 64)), gate=gate.unflatten(1, (4, 64)), dtype=E4M3)
    want, _ = plain.norm(x.unflatten(1, (4, 64)), None, None, gate.unflatten(1, (4, 64)))
    check_eight((y, s), want, plain.norm_error(gate) * want.abs())
    part, far = padded(torch.zeros(30, 256, device="cuda", dtype=BF16), 2, 8)
    ops.linear(x, w, out=part)
    assert bool((far[:, 256:] == 7).all()) and bool((far[30:] == 7).all())
