"""The serving operators (gateddeltanet_b200/ops.py) where they were once
wrong, unsafe or unseen; tolerances are those of test_gpu_ops_delta.py and
test_gpu_ops_logits.py unless a test derives its own."""
import pytest
import torch

import ops_plain as plain
from test_gpu_ops_delta import STATE_TOL, compare, inputs, out_tol

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from gateddeltanet_b200 import build
    build.build()
    from gateddeltanet_b200 import ops
    return ops


@pytest.mark.parametrize("rule", ["delta_step", "delta_chunk"])
@pytest.mark.parametrize("starts", [[10, 3, 5], [4, 8, 0, 0], [5, 8, 3, 2], [0, 5, 9, 0, 0], [70, 0]], ids=str)
@pytest.mark.parametrize("pad", [0, 200])
def test_decreasing_starts_end(ops, rule, starts, pad):
    """They give no particular values, but the call ends and touches nothing outside its tensors; with 200 empty
    sequences more, delta_step's pipeline has them."""
    starts = starts[:1] * pad + starts
    a, o = inputs([70] + [0] * (len(starts) - 2), 8, 8, 128, 128, torch.bfloat16, seed=40)
    o["starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    wide = torch.full((90, 8, 128), 7.0, device="cuda", dtype=torch.bfloat16)
    state = torch.full((a["state"].shape[0] + 2, 8, 128, 128), 7.0, device="cuda")
    state[1:-1] = a["state"]
    getattr(ops, rule)(**{**a, "state": state[1:-1]}, **o, out=wide[10:80])
    torch.cuda.synchronize()
    assert bool((wide[:10] == 7).all()) and bool((wide[80:] == 7).all())
    assert bool((state[0] == 7).all()) and bool((state[-1] == 7).all())


@pytest.mark.parametrize("shape", [(8, 8, 256, 256), (2, 8, 128, 128), (3, 3, 64, 32)], ids=str)
def test_chunk_same_bits_beside_other_work(ops, shape):
    """Warps that come late (the SMs are shared with a product on another stream) still read their own chunk's scalars."""
    a, o = inputs([1500, 700, 64], *shape, torch.bfloat16, seed=41)
    start = a.pop("state")
    first = None
    side = torch.cuda.Stream()
    x = torch.randn(2048, 2048, device="cuda", dtype=torch.bfloat16)
    for _ in range(20):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(4):
                y = x @ x
        state = start.clone()
        out = ops.delta_chunk(**a, state=state, **o)
        if first is None:
            first = (out, state)
        assert torch.equal(out, first[0]) and torch.equal(state, first[1])
    torch.cuda.synchronize()
    assert y.shape == x.shape


def test_threads_with_vocabularies_of_different_sizes(ops):
    """Calls of several host threads, each on its own stream, with tables of very different sizes."""
    import threading

    import gateddeltanet_b200 as gdn
    from test_ops_cpu import logits_args
    lib = gdn.lib()
    wrong, keep = [], []

    def work(vocab):
        with torch.cuda.stream(torch.cuda.Stream()):
            logits = torch.zeros(1, vocab, device="cuda")
            tokens = torch.zeros(1, 4, dtype=torch.int32, device="cuda")
            picks = torch.empty(1, dtype=torch.int32, device="cuda")
            keep.append((logits, tokens, picks))
            args = logits_args(logits=logits.data_ptr(), out=logits.data_ptr(), picks=picks.data_ptr(), tokens=tokens.data_ptr(),
                               lens=0, prompt_lens=0, repetition=0, presence=0, frequency=0, bias_ids=0, bias=0, mask=0,
                               stream=torch.cuda.current_stream().cuda_stream, logits_row=vocab, out_row=vocab, tokens_row=4,
                               rows=1, vocab=vocab, history=4, biases=0)
            for _ in range(4000):
                if lib.gdn_b200_constrain_logits(args) != 0:
                    wrong.append((vocab, gdn.last_error()))
                    return
    torch.zeros(1, device="cuda")
    threads = [threading.Thread(target=work, args=(v,)) for v in (200000, 1000, 262144, 50)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not wrong


def test_a_refused_call_leaves_no_error_behind(ops):
    import gateddeltanet_b200 as gdn
    a, o = inputs([1] * 40, 8, 8, 256, 256, torch.bfloat16, seed=42)
    few = {n: (x[:2] if n != "state" else x) for n, x in a.items()}
    for rule, args in ((ops.delta_step, a), (ops.delta_step, few), (ops.delta_chunk, few)):
        assert gdn.lib().gdn_b200_delta_status(99) == -1
        rule(**args, normalize=True)
        assert gdn.lib().gdn_b200_delta_status(99) == -1
        torch.zeros(3, device="cuda").add_(1).sum().item()
    assert gdn.lib().gdn_b200_delta_status(99) == -1
    ops.constrain_logits(torch.zeros(1, 40, device="cuda"))


def test_status_waits_for_every_stream(ops):
    import gateddeltanet_b200 as gdn
    x = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    side, done = torch.cuda.Stream(), torch.cuda.Event()
    with torch.cuda.stream(side):
        for _ in range(60):
            y = x @ x
        done.record()
    assert gdn.lib().gdn_b200_delta_status(0) == 0
    assert done.query()
    assert y.shape == x.shape
    ops.delta_status()
    ops.delta_status("cuda:0")
    with pytest.raises(RuntimeError, match="delta_status"):
        ops.delta_status(99)


def test_gradients_are_refused(ops):
    """Nothing that would lose a gradient is taken: no floating-point input, no output, no tangent."""
    from torch.autograd import forward_ad
    from test_gpu_ops_logits import inputs as logits_inputs
    a = logits_inputs(2, 100, 5, 2, torch.float32)
    a["out"] = torch.empty_like(a["logits"])
    d, o = inputs([3, 1], 2, 4, 64, 64, torch.bfloat16)
    d["out"] = torch.empty_like(d["v"])
    for call, args, more in ((ops.constrain_logits, a, {}), (ops.delta_step, d, o), (ops.delta_chunk, d, o)):
        for n, x in args.items():
            if not x.is_floating_point():
                continue
            with pytest.raises(RuntimeError, match="no gradient"):
                call(**{**args, n: x.clone().requires_grad_()}, **more)
            with torch.no_grad():
                call(**{**args, n: x.clone().requires_grad_()}, **more)
            with forward_ad.dual_level(), pytest.raises(RuntimeError, match="no gradient"):
                call(**{**args, n: forward_ad.make_dual(x.clone(), torch.ones_like(x))}, **more)


def test_written_tensors_get_a_new_version(ops):
    d, o = inputs([3, 1], 2, 4, 64, 64, torch.bfloat16)
    out, logits = torch.empty_like(d["v"]), torch.zeros(2, 50, device="cuda")
    for rule in (ops.delta_step, ops.delta_chunk):
        before = (d["state"]._version, out._version, d["v"]._version)
        rule(**d, **o, out=out)
        assert (d["state"]._version, out._version, d["v"]._version) == (before[0] + 1, before[1] + 1, before[2])
    before = logits._version
    ops.constrain_logits(logits, out=logits)
    assert logits._version == before + 1
    with torch.inference_mode():
        made = dict(d, state=d["state"] * 1)
    ops.delta_step(**made, **o)  # tensors without a version


def test_out_of_memory_is_torchs_own(ops):
    tokens = 2 ** 30
    wide = dict(q=torch.zeros(1, 1, 64, device="cuda", dtype=torch.bfloat16), k=torch.zeros(1, 1, 64, device="cuda", dtype=torch.bfloat16),
                v=torch.zeros(1, 1, 256, device="cuda", dtype=torch.bfloat16), g=torch.zeros(1, 1, device="cuda"),
                beta=torch.zeros(1, 1, device="cuda"))
    wide = {n: x.expand(tokens, *x.shape[1:]) for n, x in wide.items()}
    state = torch.zeros(1, 1, 256, 64, device="cuda")
    starts = torch.tensor([0, 0], dtype=torch.int32, device="cuda")
    for rule in (ops.delta_step, ops.delta_chunk):
        with pytest.raises(torch.OutOfMemoryError):
            rule(**wide, state=state, starts=starts)
    with pytest.raises(torch.OutOfMemoryError):
        ops.constrain_logits(torch.zeros(1, 2 ** 18, device="cuda").expand(2 ** 21, -1))


@pytest.mark.parametrize("rule", ["delta_step", "delta_chunk"])
def test_strides_of_a_single_entry_do_not_matter(ops, rule):
    """One token, one head or one slot: where the next one would be is not asked."""
    for lengths, heads in (([1], 2), ([70], 1)):
        a, o = inputs(lengths, heads, heads, 64, 32, torch.bfloat16, seed=43)
        o["slots"] = torch.zeros(1, dtype=torch.int32, device="cuda")
        for n in ("q", "k", "v", "state"):
            x = a[n][:1] if n == "state" else a[n]
            stride = [1003 if size == 1 else step for size, step in zip(x.shape, x.stride())]
            a[n] = x.contiguous().as_strided(x.shape, stride)
        compare(getattr(ops, rule), a, o, out_tol(rule, torch.bfloat16))


@pytest.mark.parametrize("rule", ["delta_step", "delta_chunk"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")], ids=str)
@pytest.mark.parametrize("what", ["q", "k", "v", "g", "beta", "state"])
@pytest.mark.parametrize("shape", [(2, 4, 64, 64), (2, 2, 256, 256), (5, 5, 256, 256), (8, 8, 128, 128)], ids=str)
def test_no_value_spreads_backwards(ops, rule, what, bad, shape):
    """A NaN or an infinity of one token reaches neither the tokens before it nor, where it is a value's, other value rows."""
    if what == "g" and bad < 0:
        bad = float("nan")  # log 0 is a decay like others
    lengths = [150, 97]
    for at in (0, 37, 64, 101, 148):
        a, o = inputs(lengths, *shape, torch.bfloat16, seed=44, normalize=at % 2 == 0)
        if what == "state":
            a["state"][int(o["slots"][0]), 1, 7, 5] = bad
        else:
            a[what][(at, 1, 7) if a[what].dim() == 3 else (at, 1)] = bad
        ref_o, ref_s = plain.delta_rule(**a, **o)
        out = getattr(ops, rule)(**a, **o).cpu().double()
        state = a["state"].cpu().double()
        assert torch.equal(out.isfinite(), ref_o.isfinite()) and torch.equal(state.isfinite(), ref_s.isfinite())
        fine = ref_o.isfinite()
        assert plain.rel(out[fine], ref_o[fine]) <= out_tol(rule, torch.bfloat16)
        fine = ref_s.isfinite()
        assert plain.rel(state[fine], ref_s[fine]) <= STATE_TOL


@pytest.mark.parametrize("shape", [(2, 2, 64, 64), (2, 2, 128, 128), (6, 6, 128, 128), (1, 1, 256, 256), (6, 6, 256, 256)], ids=str)
@pytest.mark.parametrize("length", [64, 700])
def test_chunk_outputs_are_fp32_before_their_rounding(ops, length, shape):
    """The output's rounding to BF16 hides an error e before it except where it
    falls the other way: for a value with spacing u between its neighbours that
    happens with probability |e| / u and then costs u. With u <= 2^-7 |o| the
    squares sum to sum |e| u <= 2^-7 ||e|| ||o||: sqrt(2^-7 E) off the rounded
    exact output for a relative error E. FP32 sums of 256 + 64 products have E =
    sqrt(320) 2^-24 / sqrt(3) (a rounding is spread evenly over its interval),
    so 7.0e-5. The count of these outputs varies: a tenth of it, where there
    are 100; n outputs have about n E 2^7."""
    E = 320 ** 0.5 * 2 ** -24 / 3 ** 0.5
    n = max(1, 2000 // length)
    a, o = inputs([length] * n, *shape, torch.bfloat16, seed=45)
    a["k"] = (a["k"].float() * 0.5 + 1).bfloat16()  # keys somewhat alike and large beta: outputs that the chunk's tokens make
    a["beta"] = 0.5 + 0.5 * a["beta"]
    o["fresh"] = torch.ones(n, dtype=torch.bool, device="cuda")
    ref_o, _ = plain.delta_rule(**a, **o)
    out = ops.delta_chunk(**a, **o)
    flips = ref_o.numel() * E * 2 ** 7
    assert plain.rel(out, ref_o.bfloat16().double()) <= (2 ** -7 * E) ** 0.5 * (1 + 2 * flips ** -0.5)


@pytest.mark.parametrize("shape", [(1, 1, 64, 64), (2, 2, 128, 128), (2, 2, 256, 256)], ids=str)
@pytest.mark.parametrize("alike", [0.3, 0.1, 0.0])
@pytest.mark.parametrize("weakest", [0.5, 0.95])
def test_chunk_of_like_keys_with_large_beta(ops, alike, weakest, shape):
    """Keys nearly or fully the same and beta near 1: (I + A)^-1 has entries
    of at most 1 that fall off by 1 - beta from one token to the next, so that
    no rounding grows: the states are FP32 sums as elsewhere, sqrt(320) 2^-24 /
    sqrt(3) (a rounding is spread evenly over its interval), for the products
    of the state and again for those of the inverse."""
    a, o = inputs([700, 65], *shape, torch.bfloat16, seed=46)
    a["k"] = (a["k"].float() * alike + 1).bfloat16()
    a["beta"] = weakest + (1 - weakest) * torch.rand_like(a["beta"])
    compare(ops.delta_chunk, a, o, out_tol("delta_chunk", torch.bfloat16), state_tol=(320 * 2 / 3) ** 0.5 * 2 ** -24)


@pytest.mark.parametrize("n", [4096, 4097, 9000])
def test_chunk_of_more_sequences_than_are_ordered(ops, n):
    gen = torch.Generator().manual_seed(n)
    lengths = torch.randint(0, 3, (n,), generator=gen).tolist()
    lengths[n // 2], lengths[-1] = 130, 70
    a, o = inputs(lengths, 1, 1, 64, 32, torch.bfloat16, seed=n)
    compare(ops.delta_chunk, a, o, out_tol("delta_chunk", torch.bfloat16))


def test_chunk_time_grows_with_the_sequences_not_their_square(ops):
    def ms(n):
        one = lambda width: torch.zeros(n, 1, width, device="cuda", dtype=torch.bfloat16)  # noqa: E731
        gates = torch.zeros(n, 1, device="cuda")
        state = torch.zeros(n, 1, 32, 64, device="cuda")
        starts = torch.arange(n + 1, dtype=torch.int32, device="cuda")
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        times = []
        for _ in range(4):
            q, k, v = one(64), one(64), one(32)
            begin.record()
            ops.delta_chunk(q, k, v, gates, gates, state, starts=starts)
            end.record()
            torch.cuda.synchronize()
            times.append(begin.elapsed_time(end))
        return min(times)
    assert ms(100000) <= 10 * ms(20000)  # five times the work; by squares 25 times


@pytest.mark.parametrize("shape", [(4, 8, 128, 128), (9, 9, 128, 64), (3, 6, 128, 96)], ids=str)
def test_chunk_many_heads_of_128(ops, shape):
    """More CTAs than SMs: 32 value rows each."""
    a, o = inputs([129, 0, 64, 1, 40, 200, 63], *shape, torch.bfloat16, seed=47)
    o["fresh"] = torch.tensor([True, True, False, False, True, False, False], device="cuda")
    compare(ops.delta_chunk, a, o, out_tol("delta_chunk", torch.bfloat16))


@pytest.mark.parametrize("history", [65535, 65536])
@pytest.mark.parametrize("shift", [0, 1, 4])
def test_long_history_of_bfloat16(ops, history, shift):
    """Counts on both sides of 16 bits, in neighbouring tokens, in rows of any alignment."""
    tokens = torch.full((2, history), 11, dtype=torch.int32, device="cuda")
    tokens[0, :7] = 12
    tokens[1] = 10
    tokens[1, 5:8] = 700
    wide = torch.ones(2, 1003 + 8, device="cuda", dtype=torch.bfloat16)
    logits = wide[:, shift:shift + 1003]
    each = lambda x: torch.full((2,), x, device="cuda")  # noqa: E731
    args = dict(tokens=tokens, frequency=each(1.0), repetition=each(2.0), presence=each(0.25),
                prompt_lens=torch.tensor([3, 0], dtype=torch.int32, device="cuda"))
    out, picks = ops.constrain_logits(logits, **args)
    ref = plain.constrain(logits, **args)
    assert torch.equal(out.cpu(), ref.bfloat16()) and picks.tolist() == [0, 0]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("many", [(60, 2, 10, 128, 128), (20, 8, 8, 256, 256), (67, 1, 6, 256, 96), (301, 2, 4, 128, 96)], ids=str)
def test_pipeline_of_sequences_with_and_without_tokens(ops, many, dtype):
    """No more tokens than sequences and eight row blocks for each SM: delta_step's pipeline, with groups of up to
    eight tokens, longer sequences, fresh ones and slots outside the pool, at its blocks' edges."""
    n, *shape = many
    gen = torch.Generator().manual_seed(n + 1)
    lengths = torch.zeros(n, dtype=torch.int64)
    for at, length in ((1, 1), (2, 7), (n // 3, 8), (n // 2, 1), (n - 2, 3)):
        lengths[at] = length
    lengths[n - 1] = n - int(lengths.sum())  # the last sequence has the rest, more than a group
    a, o = inputs(lengths.tolist(), *shape, dtype, seed=n)
    o["fresh"] = (torch.rand(n, generator=gen) < 0.4).cuda()
    o["fresh"][2], o["fresh"][n - 1] = True, False
    o["slots"][n // 3] = -1
    compare(ops.delta_step, a, o, out_tol("delta_step", dtype))


@pytest.mark.parametrize("rule,lengths,shape", [("delta_step", [1] * 40, (8, 8, 256, 256)), ("delta_chunk", [200, 70, 129], (2, 2, 256, 256)),
                                                ("delta_chunk", [200, 70, 129], (8, 8, 256, 256)),
                                                ("delta_chunk", [200, 70, 129], (2, 2, 64, 64))], ids=str)
def test_a_wait_that_runs_out_leaves_no_state_to_pass_for_one(ops, rule, lengths, shape):
    """A copy that is not made: the CTA that waits for it gives up after its limit, its states are NaN, the others right,
    the status says so once, and the next call is as if nothing had been."""
    import gateddeltanet_b200 as gdn
    ops.delta_status()
    a, o = inputs(lengths, *shape, torch.bfloat16, seed=49)
    start = a["state"].clone()
    ref_o, ref_s = plain.delta_rule(**a, **o)
    assert gdn.lib().gdn_b200_test_drop_copy(3) == 0
    getattr(ops, rule)(**a, **o)
    with pytest.raises(RuntimeError, match="ran out"):
        ops.delta_status()
    ops.delta_status()
    state, slots = a["state"].cpu().double(), o["slots"].cpu().long()
    bad = state.isnan()
    rows = bad.any(-1)
    assert torch.equal(rows, bad.all(-1)) and 0 < int(rows.sum()) < int(rows[slots].numel())
    assert not bool(rows[[i for i in range(rows.shape[0]) if i not in slots.tolist()]].any())
    assert plain.rel(state[~bad], ref_s[~bad]) <= STATE_TOL
    assert bool(rows[slots[0], 0].any())
    a["state"] = start
    compare(getattr(ops, rule), a, o, out_tol(rule, torch.bfloat16))
