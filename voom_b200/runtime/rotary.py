"""Position rotation of queries and keys, with their per-head norms, in one pass.

  Rotary         - the frequencies of a head: size, rotated part, base, pair
                   layout and long-context scaling.
  qk_norm_rope   - norm + rotation of q and k (csrc/rope.cu).

Counterpart in the reference: the norm and rotation calls of its attention
layers (runtime/layer_runner.py `_attention`), ahead of the KV caches.
"""

from __future__ import annotations

import ctypes
import math
import struct

import torch

from .. import _device
from .._lib import VOOM_E_OVERLAP, ELEMENT_TYPES, QkNormRopeArgs, check, load

LAYOUTS = ("half", "interleaved")
MAX_HEAD_DIM = 512


_COMMON_KEYS = {"rope_type", "type", "factor", "rope_theta", "partial_rotary_factor"}
_SCALING_KEYS = {
    "default": set(),
    "linear": set(),
    "ntk": set(),
    "yarn": {"original_max_position_embeddings", "beta_fast", "beta_slow", "attention_factor", "mscale",
             "mscale_all_dim", "truncate"},
    "llama3": {"original_max_position_embeddings", "low_freq_factor", "high_freq_factor"},
}


def _scaled(freqs: list[float], rot_dim: int, theta: float, scaling: dict,
            head_dim: int | None = None) -> tuple[list[float], float]:
    """Frequencies (radians per position) stretched for a longer context, and
    the factor on the rotated values.  `scaling` uses the names of model
    configurations: rope_type default (no stretching), linear, ntk, yarn or
    llama3.  A key that is not known for its type is refused, and so is one
    (rope_theta, partial_rotary_factor) that contradicts the arguments: each may
    change the angles."""
    kind = scaling.get("rope_type", scaling.get("type"))
    if kind not in _SCALING_KEYS:
        raise ValueError(f"unknown rotary scaling {kind!r} (one of {', '.join(_SCALING_KEYS)})")
    given = {k: v for k, v in scaling.items() if v is not None}
    unknown = sorted(set(given) - _COMMON_KEYS - _SCALING_KEYS[kind])
    if unknown:
        raise ValueError(f"rotary scaling {kind!r} does not take {', '.join(map(repr, unknown))}")
    if float(given.get("rope_theta", theta)) != theta:
        raise ValueError(f"rotary scaling says rope_theta {given['rope_theta']}, the argument theta is {theta}")
    if head_dim and "partial_rotary_factor" in given and \
            abs(head_dim * float(given["partial_rotary_factor"]) - rot_dim) >= 1.0:
        raise ValueError(f"rotary scaling rotates {given['partial_rotary_factor']} of a head of {head_dim}, the argument "
                         f"rot_dim is {rot_dim}")
    factor = float(given.get("factor", 1.0))
    if factor < 1.0:
        raise ValueError(f"rotary scaling factor {factor}: at least 1")
    if kind == "default":
        if factor != 1.0:
            raise ValueError(f"rotary scaling 'default' does not stretch, got factor {factor}")
        return freqs, 1.0
    if kind == "linear":
        return [f / factor for f in freqs], 1.0
    if kind == "ntk":
        base = theta * factor ** (rot_dim / max(rot_dim - 2, 1))
        return [base ** (-2.0 * i / rot_dim) for i in range(rot_dim // 2)], 1.0
    if kind == "yarn":
        orig = float(given["original_max_position_embeddings"])

        def pair_with(turns: float) -> float:  # the pair that makes `turns` turns over the original context
            return rot_dim * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(theta))

        lo, hi = pair_with(float(given.get("beta_fast", 32.0))), pair_with(float(given.get("beta_slow", 1.0)))
        if given.get("truncate", True):  # the ramp starts and ends on whole pairs
            lo, hi = math.floor(lo), math.ceil(hi)
        lo, hi = max(lo, 0), min(hi, rot_dim - 1)
        out = []
        for i, f in enumerate(freqs):
            ramp = min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0)
            out.append(f / factor * ramp + f * (1.0 - ramp))
        if "attention_factor" in given:
            return out, float(given["attention_factor"])
        if "mscale" in given or "mscale_all_dim" in given:
            if not ("mscale" in given and "mscale_all_dim" in given):
                raise ValueError("rotary scaling 'yarn' takes mscale and mscale_all_dim together")

            def gain(m: float) -> float:
                return 0.1 * m * math.log(factor) + 1.0

            return out, gain(float(given["mscale"])) / gain(float(given["mscale_all_dim"]))
        return out, 0.1 * math.log(factor) + 1.0
    orig = float(given["original_max_position_embeddings"])
    low, high = float(given["low_freq_factor"]), float(given["high_freq_factor"])
    out = []
    for f in freqs:
        turns = orig * f / (2 * math.pi)  # turns over the original context
        keep = min(max((turns - low) / (high - low), 0.0), 1.0)
        out.append(f / factor * (1.0 - keep) + f * keep)
    return out, 1.0


class Rotary:
    """The rotation of one head: `rot_dim` of its `head_dim` values (all of
    them by default) in pairs (i, i + rot_dim / 2) for layout "half" or
    (2i, 2i + 1) for "interleaved", pair i turning by theta ** (-2 i / rot_dim)
    radians per position, stretched by `scaling`.

    `turns` holds each pair's turns per position in units of 2^-64, so that
    angles far into a context keep their precision; `factor` multiplies the
    rotated values (1 but for yarn)."""

    def __init__(self, head_dim: int, *, rot_dim: int | None = None, theta: float = 10000.0, layout: str = "half",
                 scaling: dict | None = None, device=None):
        rot_dim = head_dim if rot_dim is None else rot_dim
        if not 0 < head_dim <= MAX_HEAD_DIM:
            raise ValueError(f"head size {head_dim}: 1 to {MAX_HEAD_DIM}")
        if rot_dim % 2 or not 0 <= rot_dim <= head_dim:
            raise ValueError(f"rotated part {rot_dim} of a head of {head_dim}: an even number up to the head's size")
        if layout not in LAYOUTS:
            raise ValueError(f"unknown rotary layout {layout!r} (one of {LAYOUTS})")
        self.head_dim, self.rot_dim, self.theta, self.layout = int(head_dim), int(rot_dim), float(theta), layout
        freqs = [self.theta ** (-2.0 * i / rot_dim) for i in range(rot_dim // 2)]
        self.factor = 1.0
        if scaling is not None:
            freqs, self.factor = _scaled(freqs, rot_dim, self.theta, scaling, head_dim)
        self.freqs = freqs
        turns = [round(f / (2 * math.pi) * 2 ** 64) % 2 ** 64 for f in freqs]
        self.device = _device.require_cuda(device)
        self.index = self.device.index
        self.interleaved = layout == "interleaved"
        self.turns = torch.tensor([t - 2 ** 64 if t >= 2 ** 63 else t for t in turns], dtype=torch.int64,
                                  device=self.device)
        self.turns_ptr = self.turns.data_ptr()


# voom_qk_norm_rope_args as bytes: a packed call costs a third of filling a
# ctypes structure, and one-token calls are bound by the host
_ARGS = struct.Struct("8Q8q10I2f")
assert _ARGS.size == ctypes.sizeof(QkNormRopeArgs)


def _refuse(q, k, positions, rotary, q_weight, k_weight) -> None:
    """Raises what is wrong with the arguments of qk_norm_rope."""
    D, dev = rotary.head_dim, rotary.device
    for name, x in (("q", q), ("k", k)):
        if x.dim() != 3 or x.shape[2] != D:
            raise ValueError(f"{name}: (tokens, heads, {D}) wanted, got {tuple(x.shape)}")
        if x.stride(2) != 1 and x.numel():
            raise ValueError(f"{name}: the values of a head must be contiguous")
    if q.dtype not in ELEMENT_TYPES or k.dtype != q.dtype:
        raise ValueError(f"q and k must both be BF16, FP16 or FP32, got {q.dtype} and {k.dtype}")
    if k.shape[0] != q.shape[0] or positions.shape != (q.shape[0],):
        raise ValueError(f"{q.shape[0]} tokens in q, {k.shape[0]} in k, positions {tuple(positions.shape)}")
    if positions.dtype not in (torch.int64, torch.int32) or not positions.is_contiguous():
        raise ValueError("positions must be contiguous int32 or int64")
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and (w.shape != (D,) or w.dtype not in ELEMENT_TYPES or not w.is_contiguous() or w.device != dev):
            raise ValueError(f"{name}: {D} contiguous BF16, FP16 or FP32 weights on {dev} wanted")
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        raise ValueError("q_weight and k_weight must have one type")
    raise ValueError(f"q, k, positions and the outputs must be on the rotary plan's device {dev}")


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, rotary: Rotary, *,
                 q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps: float = 1e-6,
                 zero_centered: bool = False, out_q: torch.Tensor | None = None, out_k: torch.Tensor | None = None,
                 stream: torch.cuda.Stream | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """q (T, Hq, D) and k (T, Hk, D), normed per head (x rsqrt(mean x^2 + eps)
    times the weight, or 1 + the weight with `zero_centered`; not normed where
    the weight is None) and rotated by their tokens' `positions` (T, int32 or
    int64).  BF16, FP16 or FP32; any token and head strides, so q and k may be
    views of a fused projection.  `out_q` / `out_k` may be views of a cache, or q
    and k themselves (each its own, else no memory of either).  fp32 arithmetic,
    one rounding."""
    if stream is not None or _device.current_index() != rotary.index:
        with _device.on_stream(rotary.device, stream):
            return qk_norm_rope(q, k, positions, rotary, q_weight=q_weight, k_weight=k_weight, eps=eps,
                                zero_centered=zero_centered, out_q=out_q, out_k=out_k)
    D, at, dt = rotary.head_dim, rotary.index, q.dtype
    kind = ELEMENT_TYPES.get(dt)
    if q.dim() != 3 or k.dim() != 3 or kind is None or k.dtype != dt:
        _refuse(q, k, positions, rotary, q_weight, k_weight)
    (T, hq, dq), (tk, hk, dk), (qt, qh, qd), (kt, kh, kd) = q.shape, k.shape, q.stride(), k.stride()
    pt = positions.dtype
    if not (dq == dk == D and tk == T and positions.shape == (T,) and positions.is_contiguous()
            and (pt is torch.int64 or pt is torch.int32) and (qd == kd == 1 or not T * hq * hk)
            and q.get_device() == k.get_device() == positions.get_device() == at):
        _refuse(q, k, positions, rotary, q_weight, k_weight)
    w_type = qw = kw = 0
    if q_weight is not None or k_weight is not None:
        for w in (q_weight, k_weight):
            if w is not None and (w.shape != (D,) or w.dtype not in ELEMENT_TYPES or not w.is_contiguous()
                                  or w.get_device() != at):
                _refuse(q, k, positions, rotary, q_weight, k_weight)
        if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
            _refuse(q, k, positions, rotary, q_weight, k_weight)
        w_type = ELEMENT_TYPES[(k_weight if q_weight is None else q_weight).dtype]
        qw = 0 if q_weight is None else q_weight.data_ptr()
        kw = 0 if k_weight is None else k_weight.data_ptr()
    if out_q is None:
        out_q = q.new_empty((T, hq, D))
        qot, qoh = hq * D, D
    else:
        qot, qoh = _output(out_q, q, "out_q", at)
    if out_k is None:
        out_k = k.new_empty((T, hk, D))
        kot, koh = hk * D, D
    else:
        kot, koh = _output(out_k, k, "out_k", at)
    if T:
        rc = load().voom_qk_norm_rope(
            _ARGS.pack(q.data_ptr(), k.data_ptr(), out_q.data_ptr(), out_k.data_ptr(), qw, kw, positions.data_ptr(),
                       rotary.turns_ptr, qt, qh, kt, kh, qot, qoh, kot, koh, T, hq, hk, D, rotary.rot_dim, kind,
                       w_type, pt is torch.int64, rotary.interleaved, zero_centered, eps, rotary.factor),
            _device.raw_stream(at))
        if rc == VOOM_E_OVERLAP:
            raise ValueError("rows of out_q or out_k overlap one another, or memory of q and k that is not their own")
        check(rc, "voom_qk_norm_rope")
    return out_q, out_k


def _output(x: torch.Tensor, like: torch.Tensor, name: str, device: int) -> tuple[int, int]:
    """Token and head strides of a caller's output."""
    if x.shape != like.shape or x.dtype != like.dtype or (x.stride(2) != 1 and x.numel()):
        raise ValueError(f"{name}: {tuple(like.shape)} {like.dtype} with contiguous heads wanted")
    if x.get_device() != device:
        raise ValueError(f"{name} must be on the rotary plan's device")
    return x.stride(0), x.stride(1)
