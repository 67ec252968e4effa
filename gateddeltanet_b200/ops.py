"""Serving operators on torch CUDA tensors: the gated delta rule over pooled
states (delta_step for new tokens, delta_chunk for prompts) and the
constraints on logits with the greedy pick (constrain_logits).

A thin layer over the C entries of the same names in include/gdn_b200.h,
which say what each operator computes. Calls launch on torch's current stream
of the tensors' device and do not synchronise; they can be captured into a
CUDA graph. Outputs and workspaces come from torch's allocator unless `out`
is given. There is no backward: inputs that require a gradient are refused.
"""
from __future__ import annotations

import struct
from typing import Optional, Tuple

import torch

from . import check, lib

__all__ = ["delta_step", "delta_chunk", "constrain_logits"]

_DTYPE = {torch.float32: 0, torch.bfloat16: 1}
_DELTA = struct.Struct("@13Q13q7I3ifI")     # GdnB200DeltaArgs
_LOGITS = struct.Struct("@13Q6q4I2i")       # GdnB200LogitsArgs
_entries = {}


def _entry(name: str):
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = getattr(lib(), name)
    return fn


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _pointer(t: Optional[torch.Tensor], what: str, dtype, shape: tuple, device) -> int:
    """Address of an optional tensor of this type and shape whose last dimension is contiguous."""
    if t is None:
        return 0
    _need(t.dtype in dtype if isinstance(dtype, tuple) else t.dtype == dtype, f"{what}: type {t.dtype}")
    _need(t.shape == shape, f"{what}: shape {tuple(t.shape)}, expected {shape}")
    _need(t.device == device, f"{what}: on {t.device}, expected {device}")
    _need(t.stride(-1) == 1 or shape[-1] == 1, f"{what}: the last dimension is not contiguous")
    return t.data_ptr()


def _disjoint(t: torch.Tensor, what: str) -> None:
    """Outputs may have any order of dimensions, but no two elements in one place."""
    reach = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz > 1):
        _need(stride >= reach, f"{what}: elements overlap (strides {t.stride()})")
        reach = stride * size


def _delta(name, q, k, v, g, beta, state, starts, slots, fresh, scale, normalize, out):
    _need(q.dim() == 3 and v.dim() == 3 and state.dim() == 4, f"{name}: q, k, v [tokens, heads, dim], state "
          f"[slots, v_heads, value_dim, key_dim] expected")
    device, dtype = q.device, q.dtype
    _need(device.type == "cuda", f"{name}: CUDA tensors expected")
    _need(dtype in _DTYPE, f"{name}: {dtype} is neither float32 nor bfloat16")
    tokens, heads, key_dim = q.shape
    v_heads, value_dim = v.shape[1:]
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or g.requires_grad
                                    or beta.requires_grad or state.requires_grad):
        raise RuntimeError(f"{name}: no gradient is computed (call it under torch.no_grad())")
    pq = _pointer(q, "q", dtype, q.shape, device)
    pk = _pointer(k, "k", dtype, q.shape, device)
    pv = _pointer(v, "v", dtype, (tokens, v_heads, value_dim), device)
    _need(g.shape == (tokens, v_heads) and beta.shape == (tokens, v_heads), f"{name}: g and beta [tokens, v_heads] expected")
    _need(g.dtype == torch.float32 and beta.dtype == torch.float32, f"{name}: g and beta are float32")
    _need(g.device == device and beta.device == device, f"{name}: g or beta is on another device")
    n_slots = state.shape[0]
    ps = _pointer(state, "state", torch.float32, (n_slots, v_heads, value_dim, key_dim), device)
    state_strides = state.stride()
    _need(state_strides[2] == key_dim and (state_strides[1] == value_dim * key_dim or v_heads == 1),
          "state: a slot is not one block [v_heads, value_dim, key_dim]")
    if starts is not None:
        _need(starts.dim() == 1 and starts.numel() >= 1, "starts: [sequences + 1] expected")
        sequences = starts.numel() - 1
    else:
        sequences = tokens
    pst = _pointer(starts, "starts", torch.int32, (sequences + 1,), device)
    psl = _pointer(slots, "slots", torch.int32, (sequences,), device)
    pf = _pointer(fresh, "fresh", (torch.bool, torch.uint8), (sequences,), device)
    if out is None:
        out = torch.empty((tokens, v_heads, value_dim), dtype=dtype, device=device)
    else:
        _disjoint(out, "out")
    po = _pointer(out, "out", dtype, (tokens, v_heads, value_dim), device)
    (qt, qh, _), (kt, kh, _), (vt, vh, _) = q.stride(), k.stride(), v.stride()
    (gt, gh), (bt, bh), (ot, oh, _) = g.stride(), beta.stride(), out.stride()
    stream = torch.cuda.current_stream(device).cuda_stream

    def pack(workspace, workspace_bytes):
        return _DELTA.pack(pq, pk, pv, g.data_ptr(), beta.data_ptr(), ps, po, pst, psl, pf, workspace, workspace_bytes,
                           stream, qt, qh, kt, kh, vt, vh, gt, gh, bt, bh, ot, oh, state_strides[0], sequences, tokens,
                           heads, v_heads, key_dim, value_dim, n_slots, _DTYPE[dtype], 1 if normalize else 0,
                           device.index, key_dim ** -0.5 if scale is None else scale, 0)

    return out, pack


def delta_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
               state: torch.Tensor, *, starts: Optional[torch.Tensor] = None, slots: Optional[torch.Tensor] = None,
               fresh: Optional[torch.Tensor] = None, scale: Optional[float] = None, normalize: bool = False,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """gdn_b200_delta_step: the gated delta rule token by token, for the new
    token (or the few tokens) of every stream. q, k [tokens, heads, key_dim],
    v [tokens, v_heads, value_dim] float32 or bfloat16; g (log decay) and beta
    [tokens, v_heads] float32; state [slots, v_heads, value_dim, key_dim]
    float32, advanced in place. starts int32 [sequences + 1]: the packed
    sequences' bounds (None: one token each); slots int32 [sequences]: their
    distinct states (None: in order); fresh bool [sequences]: start from zero.
    scale defaults to key_dim ** -0.5; normalize divides q and k by their L2
    norms. Returns the outputs [tokens, v_heads, value_dim]."""
    out, pack = _delta("delta_step", q, k, v, g, beta, state, starts, slots, fresh, scale, normalize, out)
    check(_entry("gdn_b200_delta_step")(pack(0, 0)), "gdn_b200_delta_step")
    return out


def delta_chunk(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                state: torch.Tensor, *, starts: Optional[torch.Tensor] = None, slots: Optional[torch.Tensor] = None,
                fresh: Optional[torch.Tensor] = None, scale: Optional[float] = None, normalize: bool = False,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """gdn_b200_delta_chunk: the same rule and arguments as delta_step for
    prompts, 64 tokens at a time on the tensor cores. q, k, v bfloat16 with
    16-byte aligned rows."""
    out, pack = _delta("delta_chunk", q, k, v, g, beta, state, starts, slots, fresh, scale, normalize, out)
    size = _entry("gdn_b200_delta_chunk_workspace")(pack(0, 0))
    workspace = torch.empty(size, dtype=torch.uint8, device=q.device)
    check(_entry("gdn_b200_delta_chunk")(pack(workspace.data_ptr(), size)), "gdn_b200_delta_chunk")
    return out


def constrain_logits(logits: torch.Tensor, *, tokens: Optional[torch.Tensor] = None, lens: Optional[torch.Tensor] = None,
                     prompt_lens: Optional[torch.Tensor] = None, repetition: Optional[torch.Tensor] = None,
                     presence: Optional[torch.Tensor] = None, frequency: Optional[torch.Tensor] = None,
                     bias_ids: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                     mask: Optional[torch.Tensor] = None,
                     out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """gdn_b200_constrain_logits: penalties for repeated tokens, biases and a
    grammar mask on logits [rows, vocab] (float32 or bfloat16), and the greedy
    pick. tokens int32 [rows, history] with the first lens[row] in use, of
    which prompt_lens[row] are the prompt (int32); repetition, presence,
    frequency float32 [rows]; bias_ids int32 and bias float32 [rows, entries]
    (id -1: not used); mask int32 [rows, ceil(vocab / 32)], bit v % 32 of word
    v // 32 set where token v is allowed. Returns (out, picks int32 [rows]);
    out may be the logits themselves, and a pick is -1 where nothing is left."""
    _need(logits.dim() == 2, "constrain_logits: logits [rows, vocab] expected")
    device, dtype = logits.device, logits.dtype
    _need(device.type == "cuda", "constrain_logits: CUDA tensors expected")
    _need(dtype in _DTYPE, f"constrain_logits: {dtype} is neither float32 nor bfloat16")
    if logits.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("constrain_logits: no gradient is computed (call it under torch.no_grad())")
    rows, vocab = logits.shape
    pl = _pointer(logits, "logits", dtype, logits.shape, device)
    if out is None:
        out = torch.empty((rows, vocab), dtype=dtype, device=device)
    elif out is not logits:
        _disjoint(out, "out")
    po = _pointer(out, "out", dtype, logits.shape, device)
    history = biases = 0
    if tokens is not None:
        _need(tokens.dim() == 2, "tokens: [rows, history] expected")
        history = tokens.shape[1]
    else:
        _need(lens is None and prompt_lens is None and repetition is None and presence is None and frequency is None,
              "constrain_logits: lens, prompt_lens and penalties need tokens")
    _need((bias is None) == (bias_ids is None), "constrain_logits: bias and bias_ids go together")
    if bias is not None:
        _need(bias.dim() == 2, "bias: [rows, entries] expected")
        biases = bias.shape[1]
    i32, f32, each = torch.int32, torch.float32, (rows,)
    pt = _pointer(tokens, "tokens", i32, (rows, history), device)
    pln, pp = _pointer(lens, "lens", i32, each, device), _pointer(prompt_lens, "prompt_lens", i32, each, device)
    pr = _pointer(repetition, "repetition", f32, each, device)
    ppr, pfr = _pointer(presence, "presence", f32, each, device), _pointer(frequency, "frequency", f32, each, device)
    pbi, pb = _pointer(bias_ids, "bias_ids", i32, (rows, biases), device), _pointer(bias, "bias", f32, (rows, biases), device)
    pm = _pointer(mask, "mask", i32, (rows, (vocab + 31) // 32), device)
    picks = torch.empty(rows, dtype=i32, device=device)
    check(_entry("gdn_b200_constrain_logits")(_LOGITS.pack(
        pl, po, picks.data_ptr(), pt, pln, pp, pr, ppr, pfr, pbi, pb, pm, torch.cuda.current_stream(device).cuda_stream,
        logits.stride(0), out.stride(0), tokens.stride(0) if tokens is not None else 0,
        bias_ids.stride(0) if biases else 0, bias.stride(0) if biases else 0, mask.stride(0) if mask is not None else 0,
        rows, vocab, history, biases, _DTYPE[dtype], device.index)), "gdn_b200_constrain_logits")
    return out, picks
