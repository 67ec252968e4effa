"""The serving operators' C entries refuse what they cannot do before any
device is touched (no GPU needed), and the plain forms the GPU tests compare
with agree with a second way of writing the formulas."""
import ctypes
import struct

import pytest
import torch

import gateddeltanet_b200 as gdn
import ops_plain as plain

FAKE = 1 << 20  # an aligned address that no check follows
DELTA = struct.Struct("@13Q13q7I3ifI")   # GdnB200DeltaArgs
LOGITS = struct.Struct("@13Q6q4I2i")     # GdnB200LogitsArgs


@pytest.fixture(scope="module")
def lib():
    from gateddeltanet_b200 import build
    build.build()
    return gdn.lib()


def delta_args(**change):
    f = dict(q=FAKE, k=FAKE, v=FAKE, g=FAKE, beta=FAKE, state=FAKE, out=FAKE, starts=FAKE, slots=FAKE, fresh=0, workspace=FAKE,
             workspace_bytes=1 << 40, stream=0, q_token=64, q_head=64, k_token=64, k_head=64, v_token=64, v_head=64, g_token=1,
             g_head=1, beta_token=1, beta_head=1, out_token=64, out_head=64, state_slot=4096, sequences=2, tokens=5, heads=1,
             v_heads=1, key_dim=64, value_dim=64, state_slots=2, dtype=1, normalize=0, device=0, scale=1.0, reserved=0)
    assert set(change) <= set(f)
    return DELTA.pack(*{**f, **change}.values())


@pytest.mark.parametrize("change,reason", [
    (dict(dtype=2), "dtype"), (dict(key_dim=96), "key_dim"), (dict(value_dim=48), "value_dim"), (dict(value_dim=288), "value_dim"),
    (dict(heads=0), "heads"), (dict(heads=2, v_heads=3), "heads"), (dict(starts=0), "without starts"),
    (dict(sequences=0), "no sequence"), (dict(slots=0, state_slots=1), "slots"), (dict(state=FAKE + 4), "16-byte"),
    (dict(state=0), "state"), (dict(state_slot=4098), "state slots"), (dict(state_slot=64), "state slots"), (dict(q=0), "missing"),
    (dict(beta=0), "missing"), (dict(tokens=2 ** 32 - 1), "too many"),
    (dict(sequences=2 ** 22), "too many"), (dict(sequences=2 ** 21, v_heads=1024), "too many")])
@pytest.mark.parametrize("entry", ["gdn_b200_delta_step", "gdn_b200_delta_chunk"])
def test_delta_refusals(lib, entry, change, reason):
    assert getattr(lib, entry)(delta_args(**change)) == -1
    assert reason in gdn.last_error()


@pytest.mark.parametrize("change,reason", [
    (dict(dtype=0), "BF16"), (dict(q=FAKE + 2), "16-byte"), (dict(k_token=65), "16-byte"), (dict(v_head=66), "16-byte")])
def test_delta_chunk_refusals(lib, change, reason):
    assert lib.gdn_b200_delta_chunk(delta_args(**change)) == -1
    assert reason in gdn.last_error()


def test_delta_nothing_to_do(lib):
    assert lib.gdn_b200_delta_step(delta_args(sequences=0, tokens=0)) == 0
    assert lib.gdn_b200_delta_chunk(delta_args(sequences=0, tokens=0)) == 0
    assert lib.gdn_b200_delta_step(None) == -1


def logits_args(**change):
    f = dict(logits=FAKE, out=FAKE, picks=FAKE, tokens=FAKE, lens=FAKE, prompt_lens=FAKE, repetition=FAKE, presence=FAKE,
             frequency=FAKE, bias_ids=FAKE, bias=FAKE, mask=FAKE, stream=0, logits_row=100, out_row=100, tokens_row=5,
             bias_ids_row=2, bias_row=2, mask_row=4, rows=2, vocab=100, history=5, biases=2, dtype=0, device=0)
    assert set(change) <= set(f)
    return LOGITS.pack(*{**f, **change}.values())


@pytest.mark.parametrize("change,reason", [
    (dict(dtype=3), "dtype"), (dict(vocab=0), "vocab"), (dict(vocab=2 ** 18 + 1), "vocab"), (dict(history=2 ** 20), "history"),
    (dict(biases=2048), "biases"), (dict(logits=0), "missing"), (dict(picks=0), "missing"), (dict(tokens=0), "tokens"),
    (dict(bias=0), "go together"), (dict(logits=FAKE + 2), "misaligned"), (dict(out_row=99), "overlap"),
    (dict(logits_row=-1), "stride"), (dict(rows=2 ** 24), "rows")])
def test_logits_refusals(lib, change, reason):
    assert lib.gdn_b200_constrain_logits(logits_args(**change)) == -1
    assert reason in gdn.last_error()


def test_logits_nothing_to_do(lib):
    assert lib.gdn_b200_constrain_logits(logits_args(rows=0)) == 0


def test_plain_delta_rule_by_its_chunk_form():
    """The token-by-token form equals the triangular system of a whole sequence."""
    gen = torch.Generator().manual_seed(1)
    T, K, V = 23, 16, 8
    q, k, v = (torch.randn(T, 1, d, generator=gen, dtype=torch.float64) for d in (K, K, V))
    g, beta = -torch.rand(T, 1, generator=gen, dtype=torch.float64), torch.rand(T, 1, generator=gen, dtype=torch.float64)
    S0 = torch.randn(1, 1, V, K, generator=gen, dtype=torch.float64)
    o, S = plain.delta_rule(q, k, v, g, beta, S0, starts=torch.tensor([0, T]), normalize=True)
    qn, kn = (x[:, 0] / (x[:, 0].square().sum(-1, keepdim=True) + 1e-6).sqrt() for x in (q, k))
    G = g[:, 0].cumsum(0)
    D = (G[:, None] - G[None, :]).exp()
    A = (beta * D * (kn @ kn.T)).tril(-1)
    d = torch.linalg.solve(torch.eye(T, dtype=torch.float64) + A, beta * (v[:, 0] - G.exp()[:, None] * (kn @ S0[0, 0].T)))
    o2 = K ** -0.5 * (G.exp()[:, None] * (qn @ S0[0, 0].T) + (D * (qn @ kn.T)).tril() @ d)
    S2 = G[-1].exp() * S0[0, 0] + ((G[-1] - G).exp()[:, None] * d).T @ kn
    assert plain.rel(o[:, 0], o2) < 1e-12 and plain.rel(S[0, 0], S2) < 1e-12


def test_plain_constraints_by_hand():
    x = plain.constrain(torch.tensor([[1.0, -1.0, 2.0, 3.0, 0.5]]), tokens=torch.tensor([[0, 1, 1, 9, -1, 2]]),
                        lens=torch.tensor([5]), prompt_lens=torch.tensor([1]), repetition=torch.tensor([2.0]),
                        presence=torch.tensor([0.25]), frequency=torch.tensor([0.5]), bias_ids=torch.tensor([[4, 4, -1]]),
                        bias=torch.tensor([[1.0, 2.0, 9.0]]), mask=torch.tensor([[0b10111]]))
    assert x.tolist() == [[0.5, -2.0 - 1.0 - 0.25, 2.0, -float("inf"), 3.5]]
    assert plain.greedy(x) == [4] and plain.greedy(torch.full((1, 3), float("nan"))) == [-1]


def test_argument_layouts():
    assert DELTA.size == 13 * 8 + 13 * 8 + 12 * 4 and LOGITS.size == 13 * 8 + 6 * 8 + 6 * 4
    assert ctypes.sizeof(ctypes.c_size_t) == 8
