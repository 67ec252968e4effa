"""The gated delta rule over pooled states (gateddeltanet_b200/ops.py
delta_step, delta_chunk) against the token-by-token form in 64 bits.

Tolerances, by what each result is made of: the state is FP32 throughout (or
products of BF16 terms that hold 24 bits) and sums of at most 256 + 64 terms,
whose rounding errors are independent: sqrt(320) 2^-24 = 1.1e-6 of a sum's
size, taken twice for the decayed errors of the tokens before. FP32 outputs
are one more such sum. A BF16 output (8 significant bits) is rounded once, at
most 2^-8 of each value and so in the 2-norm too; a chunk's output may also
take up to three factors rounded to BF16 (2^-8 / sqrt(3) each, independent):
2^-8 sqrt(1 + 1)."""
import pytest
import torch

import ops_plain as plain

pytestmark = pytest.mark.gpu

STATE_TOL = 2.2e-6
OUT_TOL = {torch.float32: 3.3e-6, torch.bfloat16: 2 ** -8}
CHUNK_OUT_TOL = 2 ** -8 * 2 ** 0.5


@pytest.fixture(scope="module")
def ops():
    from gateddeltanet_b200 import build
    build.build()
    from gateddeltanet_b200 import ops
    return ops


def inputs(lengths, heads, v_heads, key_dim, value_dim, dtype, seed=0, normalize=True, pool=None, decay=-4.0):
    gen = torch.Generator().manual_seed(seed)
    T, N = sum(lengths), len(lengths)
    rn = lambda *s: torch.randn(s, generator=gen)  # noqa: E731
    q, k = rn(T, heads, key_dim), rn(T, heads, key_dim)
    if not normalize:
        q, k = (x / (x.norm(dim=-1, keepdim=True) + 1e-9) for x in (q, k))
    pool = pool or N + 2
    a = dict(q=q.to(dtype), k=k.to(dtype), v=rn(T, v_heads, value_dim).to(dtype),
             g=-torch.nn.functional.softplus(rn(T, v_heads) + decay), beta=torch.sigmoid(rn(T, v_heads)),
             state=rn(pool, v_heads, value_dim, key_dim) * 0.1)
    o = dict(starts=torch.tensor([0] + lengths).cumsum(0).to(torch.int32),
             slots=torch.randperm(pool, generator=gen)[:N].to(torch.int32), normalize=normalize)
    return {n: x.cuda() for n, x in a.items()}, {n: x.cuda() if isinstance(x, torch.Tensor) else x for n, x in o.items()}


def compare(rule, a, o, out_tol, state_tol=STATE_TOL, **more):
    ref_o, ref_s = plain.delta_rule(**a, **o)
    before = {n: x.clone() for n, x in a.items() if n != "state"}
    out = rule(**a, **o, **more)
    torch.cuda.synchronize()
    assert plain.rel(out, ref_o) <= out_tol
    assert plain.rel(a["state"], ref_s) <= state_tol
    for n, x in before.items():
        assert torch.equal(a[n], x), f"{n} was written"
    return out


def out_tol(rule, dtype):
    return CHUNK_OUT_TOL if rule == "delta_chunk" else OUT_TOL[dtype]


SHAPES = [(1, 1, 64, 64), (2, 2, 128, 128), (3, 3, 256, 256), (2, 6, 128, 64), (1, 3, 64, 256), (4, 4, 256, 32),
          (1, 2, 256, 96)]
LENGTHS = [[1], [1, 1, 1], [0, 3, 0, 7, 1], [63], [64], [65], [129, 0, 64, 1, 40], [200, 17]]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("lengths", LENGTHS[:5], ids=str)
def test_step(ops, lengths, shape, dtype):
    a, o = inputs(lengths, *shape, dtype, seed=len(lengths))
    compare(ops.delta_step, a, o, OUT_TOL[dtype])


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
def test_chunk(ops, lengths, shape):
    a, o = inputs(lengths, *shape, torch.bfloat16, seed=7 + len(lengths), normalize=len(lengths) % 2 == 0)
    compare(ops.delta_chunk, a, o, CHUNK_OUT_TOL)


def test_long_prompt(ops):
    a, o = inputs([1500], 2, 2, 256, 256, torch.bfloat16, seed=3)
    compare(ops.delta_chunk, a, o, CHUNK_OUT_TOL)


def test_one_token_each_without_starts(ops):
    for dtype in (torch.float32, torch.bfloat16):
        a, o = inputs([1] * 5, 2, 2, 256, 256, dtype, seed=4)
        o["starts"] = None
        compare(ops.delta_step, a, o, OUT_TOL[dtype])
    a, o = inputs([1] * 3, 2, 2, 128, 128, torch.bfloat16, seed=4, pool=3)
    o["starts"] = o["slots"] = None
    compare(ops.delta_chunk, a, o, CHUNK_OUT_TOL)


@pytest.mark.parametrize("rule", ["delta_step", "delta_chunk"])
def test_fresh_states_hide_the_pool(ops, rule):
    """A fresh sequence does not read its slot, whatever it holds; one without tokens leaves zeros."""
    a, o = inputs([70, 0, 3, 0], 2, 2, 128, 64, torch.bfloat16, seed=5)
    o["fresh"] = torch.tensor([True, True, False, False], device="cuda")
    a["state"][o["slots"][:2].long()] = float("nan")
    clean = dict(a, state=torch.nan_to_num(a["state"], nan=0.0))
    ref_o, ref_s = plain.delta_rule(**clean, **o)
    out = getattr(ops, rule)(**a, **o)
    assert plain.rel(out, ref_o) <= out_tol(rule, torch.bfloat16)
    assert plain.rel(a["state"], ref_s) <= STATE_TOL


@pytest.mark.parametrize("rule", ["delta_step", "delta_chunk"])
def test_slots_outside_the_pool_and_uncovered_tokens(ops, rule):
    a, o = inputs([5, 66, 4], 2, 2, 64, 64, torch.bfloat16, seed=6)
    o["slots"][1], o["slots"][2] = -1, a["state"].shape[0]
    extra = {n: torch.cat([a[n], a[n][:70]]) for n in ("q", "k", "v", "g", "beta")}  # tokens after the last sequence
    a.update(extra)
    ref_o, ref_s = plain.delta_rule(**a, **o)
    out = torch.full_like(a["v"], float("nan"))
    getattr(ops, rule)(**a, **o, out=out)
    assert bool((out[5:] == 0).all())
    assert plain.rel(out, ref_o) <= out_tol(rule, torch.bfloat16)
    assert plain.rel(a["state"], ref_s) <= STATE_TOL


@pytest.mark.parametrize("rule", ["delta_step", "delta_chunk"])
def test_starts_are_clamped(ops, rule):
    """Bounds outside the packed tokens reach no memory outside them."""
    a, o = inputs([5, 6], 1, 1, 64, 64, torch.bfloat16, seed=8)
    o["starts"] = torch.tensor([-3, 5, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    compare(getattr(ops, rule), a, o, out_tol(rule, torch.bfloat16))


@pytest.mark.parametrize("rule", ["delta_step", "delta_chunk"])
def test_strided_inputs(ops, rule):
    """q, k, v as slices of one projection's rows, gates transposed, outputs head by head, a pool with gaps."""
    H, HV, K, V, lengths = 2, 4, 128, 64, [3, 70]
    a, o = inputs(lengths, H, HV, K, V, torch.bfloat16, seed=9)
    T = sum(lengths)
    packed = torch.full((T, 2 * H * K + HV * V + 24), float("nan"), device="cuda", dtype=torch.bfloat16)
    q, k, v = packed[:, 8:8 + H * K], packed[:, 8 + H * K:8 + 2 * H * K], packed[:, 16 + 2 * H * K:16 + 2 * H * K + HV * V]
    q, k, v = q.unflatten(1, (H, K)), k.unflatten(1, (H, K)), v.unflatten(1, (HV, V))
    for to, n in ((q, "q"), (k, "k"), (v, "v")):
        to.copy_(a[n])
    pool = torch.zeros(a["state"].shape[0], HV * V * K + 12, device="cuda")
    state = pool[:, 4:4 + HV * V * K].unflatten(1, (HV, V, K))
    state.copy_(a["state"])
    a.update(q=q, k=k, v=v, g=a["g"].t().contiguous().t(), beta=a["beta"].t().contiguous().t(), state=state)
    out = torch.empty(HV, T, V, device="cuda", dtype=torch.bfloat16).transpose(0, 1)
    compare(getattr(ops, rule), a, o, out_tol(rule, torch.bfloat16), out=out)
    assert bool((pool[:, :4] == 0).all()) and bool((pool[:, 4 + HV * V * K:] == 0).all())


def test_step_takes_any_alignment(ops):
    a, o = inputs([2, 1], 1, 1, 64, 32, torch.bfloat16, seed=10)
    for n in ("q", "k", "v"):
        wide = torch.empty(*a[n].shape[:2], a[n].shape[2] + 3, device="cuda", dtype=torch.bfloat16)
        wide[..., 3:] = a[n]
        a[n] = wide[..., 3:]
    compare(ops.delta_step, a, o, OUT_TOL[torch.bfloat16])


@pytest.mark.parametrize("rule", ["delta_step", "delta_chunk"])
@pytest.mark.parametrize("decay", [3.0, -9.0, "reset", "none"])
def test_decays(ops, rule, decay):
    """Strong and weak decay, decays to nothing (log 0 and far below the exponent range) amid weak ones, none at all."""
    a, o = inputs([150, 20], 2, 2, 128, 64, torch.bfloat16, seed=11, decay=-6.0 if isinstance(decay, str) else decay)
    if decay == "reset":
        a["g"][::7] = float("-inf")
        a["g"][3::11] = -300.0
    if decay == "none":
        a["g"].zero_()
    compare(getattr(ops, rule), a, o, out_tol(rule, torch.bfloat16))


@pytest.mark.parametrize("shape", [(1, 1, 64, 64), (2, 2, 256, 256)], ids=str)
@pytest.mark.parametrize("alike", [0.3, 0.0])
def test_chunk_of_like_keys(ops, alike, shape):
    """All keys of a sequence nearly or fully the same: the chunk's triangular
    system has a condition number of up to about 64 (its tokens), by which the
    rounding of an FP32 solution, 2^-24, may grow: 3.8e-6 more than elsewhere."""
    a, o = inputs([400, 65], *shape, torch.bfloat16, seed=31)
    a["k"] = (a["k"].float() * alike + 1).bfloat16()
    compare(ops.delta_chunk, a, o, CHUNK_OUT_TOL, state_tol=STATE_TOL + 64 * 2 ** -24)


@pytest.mark.parametrize("rule", ["delta_step", "delta_chunk"])
def test_zero_keys_and_queries(ops, rule):
    """Rows of zeros (padding) have no norm: they give zeros and only decay the state."""
    a, o = inputs([67], 1, 2, 64, 64, torch.bfloat16, seed=12)
    a["k"][10:20] = 0
    a["q"][15:30] = 0
    compare(getattr(ops, rule), a, o, out_tol(rule, torch.bfloat16))


@pytest.mark.parametrize("rule", ["delta_step", "delta_chunk"])
def test_one_sequence_cannot_spoil_another(ops, rule):
    """NaN and infinities of one sequence stay in it, next to it in memory or not."""
    a, o = inputs([5, 60, 70], 2, 2, 128, 64, torch.bfloat16, seed=13)
    clean_o, clean_s = plain.delta_rule(**a, **o)
    for n, bad in (("q", float("nan")), ("k", float("inf")), ("v", float("nan"))):
        a[n][5:65] = bad
    a["g"][5:65] = float("nan")
    out = getattr(ops, rule)(**a, **o)
    keep = [0, 1, 2, 3, 4] + list(range(65, 135))
    assert plain.rel(out[keep], clean_o[keep]) <= out_tol(rule, torch.bfloat16)
    slots = o["slots"][[0, 2]].tolist()
    assert plain.rel(a["state"][slots], clean_s[slots]) <= STATE_TOL
    assert bool(out[5:65].isnan().all()) and bool(a["state"][int(o["slots"][1])].isnan().any())


@pytest.mark.parametrize("rule", ["delta_step", "delta_chunk"])
def test_same_bits_again_and_on_another_stream(ops, rule):
    a, o = inputs([130, 1, 64], 2, 2, 256, 128, torch.bfloat16, seed=14)
    first = dict(a, state=a["state"].clone())
    out = getattr(ops, rule)(**first, **o)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = dict(a, state=a["state"].clone())
        out2 = getattr(ops, rule)(**again, **o)
    side.synchronize()
    torch.cuda.synchronize()
    assert torch.equal(out, out2) and torch.equal(first["state"], again["state"])


@pytest.mark.parametrize("rule", ["delta_step", "delta_chunk"])
def test_graph_capture(ops, rule):
    a, o = inputs([40, 1], 1, 1, 128, 64, torch.bfloat16, seed=15)
    ref_o, ref_s = plain.delta_rule(**a, **o)
    start = a["state"].clone()
    call = lambda: getattr(ops, rule)(**a, **o)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    a["state"].copy_(start)
    graph.replay()
    torch.cuda.synchronize()
    assert plain.rel(out, ref_o) <= out_tol(rule, torch.bfloat16)
    assert plain.rel(a["state"], ref_s) <= STATE_TOL


def test_state_pool_beyond_32_bit_offsets(ops):
    """The last slots of a pool of more than 2^32 bytes and 2^31 floats."""
    slots, HV, V, K = 4200, 8, 256, 256  # 2.2e9 floats
    state = torch.empty(slots, HV, V, K, device="cuda")
    a, o = inputs([66, 2], 8, 8, 256, 256, torch.bfloat16, seed=16)
    small = a.pop("state")[:2].clone()
    at = torch.tensor([slots - 1, slots - 700], device="cuda")
    for rule in ("delta_step", "delta_chunk"):
        state[at] = small
        ref_o, ref_s = plain.delta_rule(**a, state=small, starts=o["starts"], normalize=True)
        out = getattr(ops, rule)(**a, state=state, starts=o["starts"], slots=at.int(), normalize=True)
        assert plain.rel(out, ref_o) <= out_tol(rule, torch.bfloat16)
        assert plain.rel(state[at], ref_s) <= STATE_TOL


@pytest.mark.parametrize("n", [2047, 2049])
def test_chunk_of_very_many_sequences(ops, n):
    """Both ways of finding a record's sequence: by all threads at once, and by halving."""
    gen = torch.Generator().manual_seed(n)
    lengths = torch.randint(0, 3, (n,), generator=gen).tolist()
    lengths[n // 2] = 130
    a, o = inputs(lengths, 1, 1, 64, 32, torch.bfloat16, seed=n)
    compare(ops.delta_chunk, a, o, CHUNK_OUT_TOL)


def test_chunk_then_steps_is_one_sequence(ops):
    """A prompt through delta_chunk and its next tokens through delta_step."""
    a, o = inputs([140], 2, 2, 256, 256, torch.bfloat16, seed=17)
    ref_o, ref_s = plain.delta_rule(**a, **o)
    part = lambda x, y: {n: t[x:y] for n, t in a.items() if n != "state"}  # noqa: E731
    o1 = ops.delta_chunk(**part(0, 137), state=a["state"], starts=torch.tensor([0, 137], device="cuda", dtype=torch.int32),
                         slots=o["slots"], normalize=True)
    rest = [ops.delta_step(**part(t, t + 1), state=a["state"], slots=o["slots"], normalize=True) for t in range(137, 140)]
    assert plain.rel(torch.cat([o1] + rest), ref_o) <= CHUNK_OUT_TOL
    assert plain.rel(a["state"], ref_s) <= STATE_TOL


def test_nothing_to_do(ops):
    a, o = inputs([0, 0], 1, 1, 64, 64, torch.bfloat16)
    kept = a["state"].clone()
    for rule in (ops.delta_step, ops.delta_chunk):
        assert rule(**a, **o).shape == (0, 1, 64)
        none = dict(a, state=a["state"][:0])
        assert rule(**none).shape == (0, 1, 64)
    assert torch.equal(a["state"], kept)


def test_refusals(ops):
    a, o = inputs([3, 1], 2, 4, 64, 64, torch.bfloat16)
    for rule in (ops.delta_step, ops.delta_chunk):
        bad = [dict(k=a["k"][:3]), dict(k=a["k"].float()), dict(v=a["v"][:, :3]), dict(v=a["v"].transpose(1, 2)),
               dict(g=a["g"].double()), dict(beta=a["beta"][:, :2]), dict(state=a["state"].bfloat16()),
               dict(state=a["state"].transpose(2, 3)), dict(state=a["state"][..., :32]), dict(q=a["q"].cpu()),
               dict(slots=o["slots"].long()), dict(slots=o["slots"][:1]), dict(starts=o["starts"].float()),
               dict(fresh=o["slots"]), dict(out=torch.empty(4, 4, 64, device="cuda")),
               dict(out=torch.empty(1, 4, 64, device="cuda", dtype=torch.bfloat16).expand(4, 4, 64)),
               dict(q=a["q"].half(), k=a["k"].half(), v=a["v"].half())]
        for change in bad:
            with pytest.raises(ValueError):
                rule(**{**a, **o, **change})
        with pytest.raises(RuntimeError, match="key_dim"):
            rule(**{**a, **o, "q": a["q"][..., :32], "k": a["k"][..., :32], "state": a["state"][..., :32].contiguous()})
        with pytest.raises(RuntimeError, match="state slots"):
            rule(**{**a, "starts": o["starts"], "state": a["state"][:1]})
        with pytest.raises(RuntimeError, match="no gradient"):
            rule(**{**a, **o, "q": a["q"].clone().requires_grad_()})
    with pytest.raises(RuntimeError, match="BF16"):
        ops.delta_chunk(**{**a, **o, "q": a["q"].float(), "k": a["k"].float(), "v": a["v"].float()})
    wide = torch.empty(4, 2, 67, device="cuda", dtype=torch.bfloat16)[..., 3:]
    with pytest.raises(RuntimeError, match="16-byte"):
        ops.delta_chunk(**{**a, **o, "q": wide})


# enough states for the pipeline over row blocks (eight blocks of 32 KB or less for each of 148 SMs)
MANY = [(150, 8, 8, 64, 64), (60, 2, 10, 128, 128), (20, 8, 8, 256, 256), (19, 4, 8, 256, 256), (67, 1, 6, 256, 96),
        (301, 2, 4, 64, 96)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("longest", [1, 3, 4, 9])
@pytest.mark.parametrize("many", MANY, ids=str)
def test_many_states(ops, many, longest, dtype):
    n, *shape = many
    gen = torch.Generator().manual_seed(n + longest)
    lengths = [1] * n if longest == 1 else torch.randint(0, longest + 1, (n,), generator=gen).tolist()
    a, o = inputs(lengths, *shape, dtype, seed=n)
    if longest != 1:
        o["fresh"] = (torch.rand(n, generator=gen) < 0.3).cuda()
        a["state"][o["slots"][o["fresh"]].long()] = float("nan")  # not read
        o["slots"][::9] = -1
        keep = torch.isin(torch.arange(a["state"].shape[0], device="cuda"), o["slots"])
        a["state"][~keep] = 0.5
        clean = dict(a, state=a["state"].nan_to_num(nan=0.0))
    else:
        clean = dict(a, state=a["state"].clone())
    ref_o, ref_s = plain.delta_rule(**clean, **o)
    out = ops.delta_step(**a, **o)
    assert plain.rel(out, ref_o) <= OUT_TOL[dtype]
    assert plain.rel(a["state"], ref_s) <= STATE_TOL


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("many", MANY[1:5], ids=str)
def test_many_states_few_with_tokens(ops, many, dtype):
    """No more tokens than sequences, but up to 19 in one: some states untouched, some advanced several times."""
    n, *shape = many
    gen = torch.Generator().manual_seed(n)
    lengths = torch.where(torch.rand(n, generator=gen) < 0.1, 1 + torch.randint(0, 19, (n,), generator=gen), 0)
    lengths[3] = 8
    lengths[5] = 9
    lengths = lengths.tolist()
    while sum(lengths) > n:
        lengths[lengths.index(max(lengths))] //= 2
    a, o = inputs(lengths, *shape, dtype, seed=n)
    o["fresh"] = (torch.rand(n, generator=gen) < 0.3).cuda()
    o["slots"][::9] = a["state"].shape[0]
    ref_o, ref_s = plain.delta_rule(**a, **o)
    out = ops.delta_step(**a, **o)
    assert plain.rel(out, ref_o) <= OUT_TOL[dtype]
    assert plain.rel(a["state"], ref_s) <= STATE_TOL


def test_many_states_uncovered_tokens(ops):
    for lengths in ([2] * 160, [1] * 80 + [0] * 80):
        a, o = inputs(lengths, 8, 8, 128, 128, torch.bfloat16, seed=21)
        T = sum(lengths)
        a.update({n: torch.cat([a[n], a[n][:9]]) for n in ("q", "k", "v", "g", "beta")})
        ref_o, ref_s = plain.delta_rule(**a, **o)
        out = torch.full_like(a["v"], float("nan"))
        ops.delta_step(**a, **o, out=out)
        assert bool((out[T:] == 0).all()) and plain.rel(out, ref_o) <= OUT_TOL[torch.bfloat16]
        assert plain.rel(a["state"], ref_s) <= STATE_TOL


def test_no_wait_ran_out():
    import gateddeltanet_b200 as gdn
    assert gdn.lib().gdn_b200_delta_status(0) == 0, gdn.last_error()
