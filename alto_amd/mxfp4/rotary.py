"""Rotary positions of Q and K, ahead of the attention (``attention.py``): forward and backward in one HIP kernel.

The reference leaves them to the model's own code; its attention takes Q and K already rotated
(``alto/kernels/dispatch/attention.py:28-77``).
"""
from __future__ import annotations

import ctypes
import math
from typing import NamedTuple, Optional, Tuple

import torch

from . import _runtime as rt
from .._lib import check


class Rotary(NamedTuple):
    """How Q and K are rotated: the arguments of :func:`apply_rotary` that belong to a model and its tokens."""
    inv_freq: torch.Tensor
    positions: Optional[torch.Tensor] = None
    interleaved: bool = False
    factor: float = 1.0


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: Optional[dict] = None, device=None) -> Tuple[torch.Tensor, float]:
    """(radians a position of each of the ``rotary_dim / 2`` pairs, fp64; factor of cosines and sines): ``inv_freq`` and ``factor``
    of :func:`apply_rotary`.

    Frequencies are ``base ** (-2 i / rotary_dim)``, i = 0, 1, ...  ``scaling`` (a dict with a ``"type"``) stretches them for contexts longer than
    a model was trained on, by ``"factor"`` f:

    * ``"linear"``: all of them divided by f.
    * ``"ntk"``: the base becomes ``base * f ** (rotary_dim / (rotary_dim - 2))``: the highest frequency stays, the lowest is divided by f.
    * ``"yarn"``: a pair that turns ``"beta_fast"`` (32) times or more over ``"original_length"`` positions keeps its frequency, one that turns
      ``"beta_slow"`` (1) times or less has it divided by f, and between them the two are blended linearly in the turns; cosines and
      sines are multiplied with ``0.1 ln f + 1`` (or ``"attention_factor"``).  (The blend is linear in the turns, as the method's formula has it.  Models
      trained with a ramp over the pairs' numbers, between the two pairs with those turns, have other frequencies in between: give theirs to
      :func:`apply_rotary` as they are.)
    * ``"wavelength"``: the same blend between ``"high"`` (4) and ``"low"`` (1) wavelengths in ``"original_length"``, factor 1.
    """
    if rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim {rotary_dim}: a positive even number")
    if not base > 0:
        raise ValueError(f"base {base}: positive")
    i = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    kind = "none" if scaling is None else scaling["type"]
    f = 1.0 if scaling is None else float(scaling.get("factor", 1.0))
    if not f > 0:
        raise ValueError(f"scaling factor {f}: positive")
    factor = 1.0
    if kind == "ntk":
        if rotary_dim == 2:
            raise ValueError("'ntk' scaling needs two frequencies at least")
        base = base * f ** (rotary_dim / (rotary_dim - 2))
    freq = base ** (-i / rotary_dim)
    if kind == "linear":
        freq = freq / f
    elif kind in ("yarn", "wavelength"):
        high, low = ((scaling.get("beta_fast", 32.0), scaling.get("beta_slow", 1.0)) if kind == "yarn" else (scaling.get("high", 4.0), scaling.get("low", 1.0)))
        if not high > low:
            raise ValueError(f"{kind!r} scaling blends between {low} and {high} turns: the second must be larger")
        turns = float(scaling["original_length"]) * freq / (2 * math.pi)
        keep = ((turns - low) / (high - low)).clamp(0, 1)
        freq = freq / f * (1 - keep) + freq * keep
        if kind == "yarn":
            factor = float(scaling.get("attention_factor", 0.1 * math.log(f) + 1.0 if f > 1 else 1.0))
    elif kind not in ("none", "ntk"):
        raise ValueError(f"scaling type {kind!r}: 'linear', 'ntk', 'yarn' or 'wavelength'")
    return freq.to(device if device is not None else "cpu"), factor


class _Args(ctypes.Structure):
    """alto_mxfp4_rotary_t of include/alto_mxfp4.h."""
    _fields_ = ([(n, ctypes.c_void_p) for n in ("q", "k", "q_out", "k_out", "inv_freq", "positions")] + [(n, ctypes.c_int64) for n in ("B", "S", "Hq", "Hk", "D", "R")]
                + [(f"{t}_{s}", ctypes.c_int64) for t in ("q", "k", "qo", "ko") for s in ("sb", "sh", "ss")] + [("pos_sb", ctypes.c_int64), ("pos_ss", ctypes.c_int64)]
                + [("factor", ctypes.c_double)] + [(n, ctypes.c_int) for n in ("dtype", "interleaved", "inverse", "positions_are_32")])


# dims of batch, head and row in each layout (None: there is none)
_DIMS = {"bhsd": (0, 1, 2), "bshd": (0, 2, 1), "thd": (None, 1, 0)}
_NATIVE = {"bhsd": 0, "bshd": 1, "thd": 2}


def _strides(t: torch.Tensor, layout: str):
    return [0 if d is None or t.shape[d] == 1 else t.stride(d) for d in _DIMS[layout]]


def _rotate(q: torch.Tensor, k: Optional[torch.Tensor], inv_freq: torch.Tensor, positions: Optional[torch.Tensor], interleaved: bool, factor: float, layout: str,
            inverse: bool):
    batch, head, row = _DIMS[layout]
    q, k = (t if t is None or t.stride(-1) == 1 else t.contiguous() for t in (q, k))
    out = [None if t is None else torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k)]
    if q.numel() == 0:
        return out
    a = _Args(q=q.data_ptr(), k=rt.ptr(k), q_out=out[0].data_ptr(), k_out=rt.ptr(out[1]), inv_freq=inv_freq.data_ptr(), positions=rt.ptr(positions),
              B=1 if batch is None else q.shape[batch], S=q.shape[row], Hq=q.shape[head], Hk=0 if k is None else k.shape[head], D=q.shape[-1], R=2 * inv_freq.shape[0],
              factor=factor, dtype=rt.dtype_code(q.dtype), interleaved=int(interleaved), inverse=int(inverse))
    for name, t in (("q", q), ("k", k), ("qo", out[0]), ("ko", out[1])):
        if t is not None:
            for s, value in zip(("sb", "sh", "ss"), _strides(t, layout)):
                setattr(a, f"{name}_{s}", value)
    if positions is not None:
        a.positions_are_32 = int(positions.dtype == torch.int32)
        a.pos_sb, a.pos_ss = (0 if positions.dim() == 1 or positions.shape[0] == 1 else positions.stride(0)), positions.stride(-1)
    if q.device.index == torch.cuda.current_device():
        check(rt.lib().alto_mxfp4_rotary(ctypes.byref(a), rt.stream_ptr(q.device)), "alto_mxfp4_rotary")
    else:
        with torch.cuda.device(q.device):
            check(rt.lib().alto_mxfp4_rotary(ctypes.byref(a), rt.stream_ptr(q.device)), "alto_mxfp4_rotary")
    return out


class RotaryFunction(torch.autograd.Function):
    """(q, k) rotated; the backward rotates their gradients back with the same kernel and keeps neither Q nor K."""

    @staticmethod
    def forward(ctx, q, k, inv_freq, positions, interleaved, factor, layout, inverse):
        ctx.save_for_backward(inv_freq, positions)
        ctx.more = interleaved, factor, layout, inverse
        out = _rotate(q, k, inv_freq, positions, *ctx.more)
        return tuple(out) if k is not None else out[0]

    @staticmethod
    def backward(ctx, dq, dk=None):
        inv_freq, positions = ctx.saved_tensors
        interleaved, factor, layout, inverse = ctx.more
        back = RotaryFunction.apply(dq, dk, inv_freq, positions, interleaved, factor, layout, not inverse)   # (linear: its gradient is one)
        return (*(back if dk is not None else (back, None)), None, None, None, None, None, None)


def apply_rotary(q: torch.Tensor, k: Optional[torch.Tensor], inv_freq: torch.Tensor, positions: Optional[torch.Tensor] = None, *, interleaved: bool = False,
                 factor: float = 1.0, layout: str = "bhsd"):
    """``q`` and ``k`` with their heads rotated by their tokens' positions, as new tensors (``k`` None: only ``q``); differentiable.

    bf16 or fp32, [B, H, S, D], [B, S, H, D] with ``layout="bshd"`` or [T, H, D] with ``"thd"``, of any strides.  ``inv_freq`` (fp64, on their device,
    :func:`rotary_frequencies`, or a model's own in fp64): radians a position of each pair; twice as many columns, from the first on, are rotated in the pairs
    (i, i + R/2), or (2i, 2i + 1) with ``interleaved``, the others pass.  ``positions``: int32 or int64 [S] or [B, S] ([T] with ``"thd"``) of any
    sign, None for 0, 1, ...  ``factor`` multiplies cosines and sines.  Angles, cosines and sines are taken in 64 bits.
    """
    if torch.compiler.is_compiling():
        return _apply_between_graphs(q, k, inv_freq, positions, interleaved, factor, layout)
    if k is not None and q.is_cuda and layout in _NATIVE:   # one native call; what it declines takes the general way
        out = rt.host().rotary(q, k, inv_freq, positions, bool(interleaved), float(factor), _NATIVE[layout])
        if out is not None:
            return out
    return _apply(q, k, inv_freq, positions, interleaved, factor, layout)


def _apply(q, k, inv_freq, positions, interleaved, factor, layout):
    if layout not in _DIMS:
        raise NotImplementedError(f"layout {layout!r}: 'bhsd', 'bshd' and 'thd' are implemented")
    rt.refuse_transforms("apply_rotary", q, k, inv_freq)
    rt.require_gpu(q, k, inv_freq, positions)
    dims = 3 if layout == "thd" else 4
    batch, head, row = _DIMS[layout]
    rt.dtype_code(q.dtype)
    assert q.dim() == dims and (k is None or (k.dim() == dims and k.dtype == q.dtype)), f"layout {layout!r}: q and k of {dims} dims and one type"
    assert q.shape[head] > 0, "q has no heads"
    assert k is None or all(k.shape[d] == q.shape[d] for d in range(dims) if d != head), f"q of shape {tuple(q.shape)} and k of {tuple(k.shape)}"
    assert inv_freq.dim() == 1 and inv_freq.dtype == torch.float64 and inv_freq.is_contiguous(), "inv_freq: fp64, one frequency for each pair"
    assert 1 <= inv_freq.shape[0] <= 1024 and 2 * inv_freq.shape[0] <= q.shape[-1], f"{inv_freq.shape[0]} frequencies for heads of {q.shape[-1]}"
    if positions is not None:
        assert positions.dtype in (torch.int32, torch.int64), f"positions of type {positions.dtype}: int32 or int64"
        fits = positions.shape == (q.shape[row],) or (batch is not None and positions.dim() == 2 and positions.shape[0] in (1, q.shape[batch]) and positions.shape[1] == q.shape[row])
        assert fits, f"positions of shape {tuple(positions.shape)} for q of {tuple(q.shape)}, layout {layout!r}"
    if inv_freq.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError("the gradient of the frequencies is not implemented: detach them")
    for t in (k, inv_freq, positions):
        assert t is None or t.device == q.device, f"tensors on {q.device} and {t.device}"
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        return RotaryFunction.apply(q, k, inv_freq, positions, bool(interleaved), float(factor), layout, False)
    out = _rotate(q, k, inv_freq, positions, bool(interleaved), float(factor), layout, False)
    return tuple(out) if k is not None else out[0]


@torch.compiler.disable
def _apply_between_graphs(q, k, inv_freq, positions, interleaved, factor, layout):
    """(nothing of the call can be traced: a compiled caller breaks its graph here)"""
    out = rt.host().rotary(q, k, inv_freq, positions, bool(interleaved), float(factor), _NATIVE[layout]) if k is not None and q.is_cuda and layout in _NATIVE else None
    return out if out is not None else _apply(q, k, inv_freq, positions, interleaved, factor, layout)
