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
_F32, _I32 = torch.float32, torch.int32
_DELTA = struct.Struct("@13Q13q7I3ifI")     # GdnB200DeltaArgs
_LOGITS = struct.Struct("@13Q6q4I2i")       # GdnB200LogitsArgs
_entries = {}
try:
    _stream = torch._C._cuda_getCurrentRawStream  # the address alone: a tenth of the time of a stream object
except AttributeError:
    def _stream(device: int) -> int:
        return torch.cuda.current_stream(device).cuda_stream


def _entry(name: str):
    fn = _entries.get(name)
    if fn is None:
        fn = _entries[name] = getattr(lib(), name)
    return fn


def _disjoint(shape, strides) -> bool:
    """Outputs may have any order of dimensions, but no two elements in one place."""
    reach = 1
    for stride, size in sorted((st, sz) for st, sz in zip(strides, shape) if sz > 1):
        if stride < reach:
            return False
        reach = stride * size
    return True


def _no_gradient(name: str, *tensors) -> None:
    for t in tensors:
        if t.requires_grad:
            raise RuntimeError(f"{name}: no gradient is computed (call it under torch.no_grad())")


def _refuse(name: str, device: int, wanted) -> None:
    """Says which argument is not as (argument, tensor, types, shape) of `wanted` ask; the calls test them all at once."""
    for what, t, types, shape in wanted:
        if t is None:
            continue
        if t.dtype not in types:
            raise ValueError(f"{name}: {what} has type {t.dtype}")
        if t.get_device() != device or device < 0:
            raise ValueError(f"{name}: {what} is on {t.device}, all on one CUDA device expected")
        if shape is not None and tuple(t.shape) != tuple(shape):
            raise ValueError(f"{name}: {what} has shape {tuple(t.shape)}, expected {tuple(shape)}")
        if t.dim() == 1 and not t.is_contiguous() or t.dim() > 1 and t.stride(-1) != 1 and what not in ("g", "beta"):
            raise ValueError(f"{name}: the last dimension of {what} is not contiguous")
    raise ValueError(f"{name}: elements of out overlap, or a slot of state is not one block [v_heads, value_dim, key_dim]")


def _delta(name, q, k, v, g, beta, state, starts, slots, fresh, scale, normalize, out):
    """Checks the tensors; returns (out, pack), pack(workspace, bytes) being the C entry's arguments."""
    if q.dim() != 3 or v.dim() != 3 or state.dim() != 4 or k.dim() != 3:
        raise ValueError(f"{name}: q, k, v [tokens, heads, dim], state [slots, v_heads, value_dim, key_dim] expected")
    if torch.is_grad_enabled():
        _no_gradient(name, q, k, v, g, beta, state)
    dtype, device = q.dtype, q.get_device()
    code = _DTYPE.get(dtype, -1)
    q_shape, v_shape = q.shape, v.shape
    tokens, heads, key_dim = q_shape
    _, v_heads, value_dim = v_shape
    n_slots = state.shape[0]
    sequences = tokens if starts is None else starts.shape[0] - 1 if starts.dim() == 1 else -1
    if out is None:
        out = torch.empty_like(v) if v.is_contiguous() else torch.empty(v_shape, dtype=dtype, device=v.device)
        out_ok = True
    else:
        out_ok = (out.dtype is dtype and out.get_device() == device and out.shape == v_shape
                  and _disjoint(v_shape, out.stride()))
    gates = (tokens, v_heads)
    if not (out_ok and code >= 0 and device >= 0 and k.dtype is dtype and v.dtype is dtype and k.shape == q_shape
            and v_shape[0] == tokens and g.dtype is _F32 and beta.dtype is _F32 and g.shape == gates
            and beta.shape == gates and state.dtype is _F32 and state.shape == (n_slots, v_heads, value_dim, key_dim)
            and k.get_device() == device and v.get_device() == device and g.get_device() == device
            and beta.get_device() == device and state.get_device() == device and sequences >= 0
            and (starts is None or starts.dtype is _I32 and starts.get_device() == device and starts.is_contiguous())
            and (slots is None or slots.dtype is _I32 and slots.shape == (sequences,) and slots.get_device() == device
                 and slots.is_contiguous())
            and (fresh is None or fresh.element_size() == 1 and fresh.dtype in (torch.bool, torch.uint8)
                 and fresh.shape == (sequences,) and fresh.get_device() == device and fresh.is_contiguous())):
        _refuse(name, device, (("q", q, _DTYPE, None), ("k", k, (dtype,), q_shape), ("v", v, (dtype,), (tokens, *v_shape[1:])),
                               ("g", g, (_F32,), gates), ("beta", beta, (_F32,), gates),
                               ("state", state, (_F32,), (n_slots, v_heads, value_dim, key_dim)),
                               ("starts", starts, (_I32,), None if sequences >= 0 else ("sequences + 1",)),
                               ("slots", slots, (_I32,), (sequences,)),
                               ("fresh", fresh, (torch.bool, torch.uint8), (sequences,)), ("out", out, (dtype,), v_shape)))
    (qt, qh, q1), (kt, kh, k1), (vt, vh, v1), (ot, oh, o1) = q.stride(), k.stride(), v.stride(), out.stride()
    (gt, gh), (bt, bh), (ss, sh, sv, sk) = g.stride(), beta.stride(), state.stride()
    if not (q1 == k1 == v1 == o1 == sk == 1 and sv == key_dim and (sh == value_dim * key_dim or v_heads == 1)):
        _refuse(name, device, (("q", q, _DTYPE, None), ("k", k, _DTYPE, None), ("v", v, _DTYPE, None),
                               ("out", out, _DTYPE, None), ("state", state, (_F32,), None)))

    def pack(workspace, workspace_bytes):
        return _DELTA.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), beta.data_ptr(), state.data_ptr(),
                           out.data_ptr(), 0 if starts is None else starts.data_ptr(), 0 if slots is None else slots.data_ptr(),
                           0 if fresh is None else fresh.data_ptr(), workspace, workspace_bytes, _stream(device), qt, qh, kt,
                           kh, vt, vh, gt, gh, bt, bh, ot, oh, ss, sequences, tokens, heads, v_heads, key_dim, value_dim,
                           n_slots, code, 1 if normalize else 0, device, key_dim ** -0.5 if scale is None else scale, 0)

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
    rc = _entry("gdn_b200_delta_step")(pack(0, 0))
    if rc:
        check(rc, "gdn_b200_delta_step")
    return out


def delta_chunk(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                state: torch.Tensor, *, starts: Optional[torch.Tensor] = None, slots: Optional[torch.Tensor] = None,
                fresh: Optional[torch.Tensor] = None, scale: Optional[float] = None, normalize: bool = False,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """gdn_b200_delta_chunk: the same rule and arguments as delta_step for
    prompts, 64 tokens at a time on the tensor cores. q, k, v bfloat16 with
    16-byte aligned rows."""
    out, pack = _delta("delta_chunk", q, k, v, g, beta, state, starts, slots, fresh, scale, normalize, out)
    size = _entry("gdn_b200_delta_chunk_workspace")(v.shape[0], v.shape[0] if starts is None else starts.shape[0] - 1, v.shape[1])
    workspace = torch.empty(size, dtype=torch.uint8, device=q.device)
    rc = _entry("gdn_b200_delta_chunk")(pack(workspace.data_ptr(), size))
    if rc:
        check(rc, "gdn_b200_delta_chunk")
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
    name = "constrain_logits"
    if logits.dim() != 2:
        raise ValueError(f"{name}: logits [rows, vocab] expected")
    if torch.is_grad_enabled():
        _no_gradient(name, logits)
    dtype, device, shape = logits.dtype, logits.get_device(), logits.shape
    code = _DTYPE.get(dtype, -1)
    rows, vocab = shape
    if out is None:
        out = torch.empty_like(logits) if logits.is_contiguous() else torch.empty(shape, dtype=dtype, device=logits.device)
    history = biases = 0
    if tokens is not None:
        history = tokens.shape[1] if tokens.dim() == 2 else -1
    elif not (lens is None and prompt_lens is None and repetition is None and presence is None and frequency is None):
        raise ValueError(f"{name}: lens, prompt_lens and penalties need tokens")
    if (bias is None) != (bias_ids is None):
        raise ValueError(f"{name}: bias and bias_ids go together")
    if bias is not None:
        biases = bias.shape[1] if bias.dim() == 2 else -1
    each = (rows,)

    def ok1(t, of):
        return t is None or t.dtype is of and t.shape == each and t.get_device() == device and t.is_contiguous()

    def ok2(t, of, width):
        return t is None or (t.dtype is of and t.shape == (rows, width) and t.get_device() == device
                             and (t.stride(1) == 1 or width <= 1))

    if not (code >= 0 and device >= 0 and ok2(logits, dtype, vocab) and (out is logits or ok2(out, dtype, vocab)
            and _disjoint(shape, out.stride())) and ok2(tokens, _I32, history) and ok1(lens, _I32) and ok1(prompt_lens, _I32)
            and ok1(repetition, _F32) and ok1(presence, _F32) and ok1(frequency, _F32) and ok2(bias_ids, _I32, biases)
            and ok2(bias, _F32, biases) and ok2(mask, _I32, (vocab + 31) // 32)):
        wide = lambda n: ("rows", "width") if n < 0 else (rows, n)  # noqa: E731
        _refuse(name, device, (("logits", logits, _DTYPE, None), ("out", out, (dtype,), shape),
                               ("tokens", tokens, (_I32,), wide(history)), ("lens", lens, (_I32,), each),
                               ("prompt_lens", prompt_lens, (_I32,), each), ("repetition", repetition, (_F32,), each),
                               ("presence", presence, (_F32,), each), ("frequency", frequency, (_F32,), each),
                               ("bias_ids", bias_ids, (_I32,), wide(biases)), ("bias", bias, (_F32,), wide(biases)),
                               ("mask", mask, (_I32,), (rows, (vocab + 31) // 32))))

    def at(t):
        return 0 if t is None else t.data_ptr()

    picks = torch.empty(rows, dtype=_I32, device=logits.device)
    rc = _entry("gdn_b200_constrain_logits")(_LOGITS.pack(
        logits.data_ptr(), out.data_ptr(), picks.data_ptr(), at(tokens), at(lens), at(prompt_lens), at(repetition),
        at(presence), at(frequency), at(bias_ids), at(bias), at(mask), _stream(device), logits.stride(0), out.stride(0),
        tokens.stride(0) if history else 0, bias_ids.stride(0) if biases else 0, bias.stride(0) if biases else 0,
        0 if mask is None else mask.stride(0), rows, vocab, history, biases, code, device))
    if rc:
        check(rc, "gdn_b200_constrain_logits")
    return out, picks
