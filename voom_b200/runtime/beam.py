"""Beam search: the choice of the continuations of each step.

  beam_select - the best continuations over a request's beams and the
                vocabulary (csrc/beam.cu).

The rows that the choice names are what PagePool.fork (kv_pool.py) takes as
parents: the beams' cached positions follow without being copied.

Counterpart in the reference: none (its decode loop, runtime/engine.py, samples
one continuation); it stands beside the drafted trees of kv_attention.py.
"""

from __future__ import annotations

import ctypes
import struct
from typing import NamedTuple

import torch

from .. import _device
from .._lib import ELEMENT_TYPES, BeamSelectArgs, check, load

MAX_BEAMS = 64
MAX_WIDTH = 64
MAX_ROWS = 2 ** 27  # beams of all requests, fewer

_ARGS = struct.Struct("5Q2q6I")
assert _ARGS.size == ctypes.sizeof(BeamSelectArgs)


class BeamChoice(NamedTuple):
    """A step's continuations, (B, width) each, the best first: their scores
    (fp32), the rows that they continue (b * beams + beam, int32) and their
    tokens (int32).  Where there are fewer candidates: -inf, -1, -1."""

    scores: torch.Tensor
    parents: torch.Tensor
    tokens: torch.Tensor


def beam_select(logits: torch.Tensor, scores: torch.Tensor, width: int, *,
                stream: torch.cuda.Stream | None = None) -> BeamChoice:
    """The `width` candidates with the largest score + log_softmax(logits) of each
    request.  logits: (B, beams, V) BF16, FP16 or FP32, a row's values adjacent,
    any alignment; scores: (B, beams) fp32, the beams' sums so far.  Compared in
    64 bits; equal candidates: the lower beam, within one the larger logit, then
    the lower token.  A logit of -inf is never chosen, nor is anything of a beam whose score is -inf
    (a first step has one beam alive; an ended one none) or that has a NaN or
    an infinite logit.  width <= 64: twice the beams, to set ended ones aside."""
    index = logits.get_device()
    if index < 0:
        raise ValueError(f"logits: a CUDA tensor wanted, got one on {logits.device}")
    if stream is not None or _device.current_index() != index:
        with _device.on_stream(logits.device, stream):
            return beam_select(logits, scores, width)
    kind = ELEMENT_TYPES.get(logits.dtype)
    if logits.dim() != 3 or kind is None or (logits.stride(2) != 1 and logits.shape[2] > 1):
        raise ValueError(f"logits: (B, beams, V) BF16, FP16 or FP32 with adjacent values wanted, got {tuple(logits.shape)} "
                         f"{logits.dtype}, strides {logits.stride()}")
    (B, beams, V), (sb, si, _) = logits.shape, logits.stride()
    if scores.shape != (B, beams) or scores.dtype != torch.float32 or not scores.is_contiguous() or scores.get_device() != index:
        raise ValueError(f"scores: contiguous fp32 ({B}, {beams}) on {logits.device} wanted, got {tuple(scores.shape)} "
                         f"{scores.dtype} on {scores.device}")
    if not 0 < beams <= MAX_BEAMS or not 0 < width <= MAX_WIDTH or not V:
        raise ValueError(f"{beams} beams, {width} continuations of {V} tokens: 1 to {MAX_BEAMS} beams and 1 to {MAX_WIDTH} "
                         "continuations, one token at least")
    if beams * V >= 2 ** 31 or B * beams >= MAX_ROWS:
        raise ValueError(f"{B} requests of {beams} beams over {V} tokens: fewer than 2^31 candidates each, and 2^27 beams, wanted")
    best = scores.new_empty((B, width))
    parents, tokens = scores.new_empty((2, B, width), dtype=torch.int32).unbind(0)
    if B:
        a = _ARGS.pack(logits.data_ptr(), scores.data_ptr(), best.data_ptr(), parents.data_ptr(), tokens.data_ptr(), sb, si, B,
                       beams, V, width, kind, 0)
        lib = load()
        ws = scores.new_empty(lib.voom_beam_select_scratch_bytes(a), dtype=torch.uint8)
        check(lib.voom_beam_select(a, ws.data_ptr(), ws.numel(), _device.raw_stream(index)), "voom_beam_select")
    return BeamChoice(best, parents, tokens)
