"""Serving operators on torch CUDA tensors: the gated delta rule over pooled
states (delta_step for new tokens, delta_chunk for prompts) and the
constraints on logits with the greedy pick (constrain_logits).

A thin layer over the C entries of the same names in include/gdn_b200.h,
which say what each operator computes; csrc/gdn_ops_torch.cpp checks the
tensors and makes the calls. Calls launch on torch's current stream of the
tensors' device and do not synchronise; they can be captured into a CUDA
graph. Outputs and workspaces come from torch's allocator unless `out` is
given. There is no backward: inputs that require a gradient are refused.
Arguments that do not fit raise ValueError, what the C entry refuses
RuntimeError.
"""
from __future__ import annotations

import ctypes
import importlib.util
import os
from typing import Optional, Tuple

import torch

from . import HERE, last_error, lib

__all__ = ["delta_step", "delta_chunk", "delta_status", "constrain_logits"]


def _load():
    path = os.path.join(HERE, "_ops_torch.so")
    if not os.path.exists(path):
        raise RuntimeError(f"_ops_torch.so not found at {path}: run `python -m gateddeltanet_b200.build`")
    spec = importlib.util.spec_from_file_location("_ops_torch", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    L = lib()
    module.bind(*(ctypes.cast(getattr(L, name), ctypes.c_void_p).value for name in (
        "gdn_b200_delta_step", "gdn_b200_delta_chunk", "gdn_b200_delta_chunk_workspace", "gdn_b200_constrain_logits",
        "gdn_b200_last_error")))
    return module


_native = _load()


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
    norms. Returns the outputs [tokens, v_heads, value_dim] (`out` if given, in
    memory apart from the inputs)."""
    return _native.delta_step(q, k, v, g, beta, state, starts, slots, fresh, scale, normalize, out)


def delta_chunk(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor,
                state: torch.Tensor, *, starts: Optional[torch.Tensor] = None, slots: Optional[torch.Tensor] = None,
                fresh: Optional[torch.Tensor] = None, scale: Optional[float] = None, normalize: bool = False,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """gdn_b200_delta_chunk: the same rule and arguments as delta_step for
    prompts, 64 tokens at a time on the tensor cores. q, k, v bfloat16 with
    16-byte aligned rows."""
    return _native.delta_chunk(q, k, v, g, beta, state, starts, slots, fresh, scale, normalize, out)


def delta_status(device=None) -> None:
    """gdn_b200_delta_status: waits for the device (None: the current one) and
    raises RuntimeError if a wait inside delta_step or delta_chunk ran out
    there since the last call: the states of that call are then not valid."""
    device = torch.device("cuda" if device is None else device)
    if device.type != "cuda":
        raise ValueError(f"delta_status: {device} is not a CUDA device")
    index = device.index
    if lib().gdn_b200_delta_status(torch.cuda.current_device() if index is None else index) != 0:
        raise RuntimeError(last_error())


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
    out may be the logits themselves or memory apart from them, and a pick is -1
    where nothing is left."""
    return _native.constrain_logits(logits, tokens, lens, prompt_lens, repetition, presence, frequency, bias_ids, bias, mask, out)
