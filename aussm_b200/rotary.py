"""Queries and keys: the norm of each head and the rotation by position, in one pass.

``qk_norm_rotate`` normalises every head of ``q`` and ``k`` (mean square or length) and turns pairs of its elements by
``position * frequency``: in the mixers of this package the turn gives a real-valued recurrence the rotating phase that
the unitary scan has by itself.  ``rotary_frequencies`` makes the usual frequencies, also those for contexts longer than
a model was trained on.  CUDA tensors only; all arithmetic runs in libaussm_b200.so.
"""
from __future__ import annotations

import ctypes
import functools
import math
from typing import Optional, Tuple

import torch
from torch import Tensor

from . import _lib
from .delta import _DTYPES, _on, _plain, _raw_stream, _refuse_traced, _strides, _typed
from .ops import _ptr, _workspace

__all__ = ["qk_norm_rotate", "rotary_frequencies", "MAX_HEAD"]

MAX_HEAD = 256
_NORMS = {None: 0, "rms": 1, "l2": 2}


def rotary_frequencies(dim: int, base: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
                       original_length: int = 4096, turns: Tuple[float, float] = (1.0, 32.0),
                       device=None) -> Tuple[Tensor, float]:
    """``(frequencies, magnitude)`` for ``qk_norm_rotate``: ``dim / 2`` float64 radians per position, ``base^(-2i/dim)``.

    ``scaling`` stretches them for contexts ``factor`` times as long as the ``original_length`` steps of training:
    ``"linear"`` divides all by ``factor``; ``"base"`` raises the base so that the slowest is divided by ``factor`` and
    the fastest keeps its pace; ``"ramp"`` divides those that make fewer than ``turns[0]`` turns over the original length
    by ``factor``, keeps those that make more than ``turns[1]`` and blends in between, and returns the magnitude
    ``0.1 ln(factor) + 1`` by which both queries and keys grow (1 otherwise)."""
    if dim <= 0 or dim % 2:
        raise RuntimeError(f"dim must be even and positive, got {dim}")
    if factor <= 0 or base <= 0:
        raise RuntimeError("base and factor must be positive")
    if not turns[0] < turns[1]:
        raise RuntimeError(f"turns must be two rising numbers, got {turns}")
    i = torch.arange(0, dim, 2, device=device, dtype=torch.float64) / dim
    magnitude = 1.0
    if scaling == "base" and dim > 2:
        base = base * factor ** (dim / (dim - 2))
    f = float(base) ** -i
    if scaling == "linear" or (scaling == "base" and dim == 2):
        f = f / factor
    elif scaling == "ramp":
        made = original_length * f / (2 * math.pi)
        keep = ((made - turns[0]) / (turns[1] - turns[0])).clamp(0, 1)
        f = f * keep + f / factor * (1 - keep)
        magnitude = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    elif scaling not in (None, "base"):
        raise RuntimeError(f'scaling must be None, "linear", "base" or "ramp", got {scaling!r}')
    return f, magnitude


@functools.lru_cache(maxsize=256)
def _problem(b, l, hq, hk, d, rot, dtype, norm, interleaved, eps, magnitude, position_stride, *strides):
    """The problem of these sizes, types and strides: read only (the backward call takes a copy)."""
    q, k = ((ctypes.c_longlong * 3)(*strides[i:i + 3]) for i in (0, 3))
    return _lib.RotateProblem(b, l, hq, hk, d, rot, dtype, norm, interleaved, eps, magnitude, position_stride, q, k)


def _forward(q, k, q_weight, k_weight, frequencies, positions, p):
    yq = torch.empty(q.shape, device=q.device, dtype=q.dtype)
    yk = torch.empty(k.shape, device=k.device, dtype=k.dtype)
    if p.B and p.L:
        with _on(q.device):
            rc = _lib.load().aussm_b200_rotate_fwd(p, _ptr(q), _ptr(k), _ptr(frequencies), _ptr(positions), _ptr(q_weight),
                                                   _ptr(k_weight), _ptr(yq), _ptr(yk), _raw_stream(q.device))
        _lib.check(rc, "qk_norm_rotate")
    return yq, yk


class _NormRotate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, frequencies, positions, p):
        ctx.p = p
        ctx.save_for_backward(q, k, q_weight, k_weight, frequencies, positions)
        return _forward(q, k, q_weight, k_weight, frequencies, positions, p)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gq, gk):
        q, k, q_weight, k_weight, frequencies, positions = ctx.saved_tensors
        p = type(ctx.p).from_buffer_copy(ctx.p)         # of this call's own: the gradients' strides go in
        dq, dk = (torch.empty(t.shape, device=t.device, dtype=t.dtype) for t in (q, k))
        dqw = torch.empty_like(q_weight) if ctx.needs_input_grad[2] else None
        dkw = torch.empty_like(k_weight) if ctx.needs_input_grad[3] else None
        if not (p.B and p.L):
            return dq, dk, None if dqw is None else dqw.zero_(), None if dkw is None else dkw.zero_(), None, None, None
        gq, gk = _plain(gq), _plain(gk)
        p.gq_stride, p.gk_stride = _strides(gq), _strides(gk)
        lib = _lib.load()
        with _on(q.device):
            ws = None
            if dqw is not None or dkw is not None:
                ws = _workspace(lib.aussm_b200_rotate_bwd_workspace_bytes(p), q.device)
            rc = lib.aussm_b200_rotate_bwd(p, _ptr(gq), _ptr(gk), _ptr(q), _ptr(k), _ptr(frequencies), _ptr(positions),
                                           _ptr(q_weight), _ptr(k_weight), _ptr(dq), _ptr(dk), _ptr(dqw), _ptr(dkw), _ptr(ws),
                                           0 if ws is None else ws.numel(), _raw_stream(q.device))
        _lib.check(rc, "qk_norm_rotate backward")
        return dq, dk, dqw, dkw, None, None, None


def qk_norm_rotate(q: Tensor, k: Tensor, frequencies: Optional[Tensor] = None, positions: Optional[Tensor] = None, *,
                   q_weight: Optional[Tensor] = None, k_weight: Optional[Tensor] = None, norm: Optional[str] = "rms",
                   eps: float = 1e-6, interleaved: bool = False, magnitude: float = 1.0) -> Tuple[Tensor, Tensor]:
    """``q`` ``(b, l, hq, d)`` and ``k`` ``(b, l, hk, d)`` normalised per head, weighted and rotated; differentiable once in
    ``q, k`` and the weights.

    ``norm``: ``"rms"`` divides a head by ``sqrt(mean(x^2) + eps)``, ``"l2"`` by ``sqrt(sum(x^2) + eps)``, None leaves it.
    ``q_weight, k_weight``: ``(d,)`` float32, shared by the heads.  ``frequencies``: up to ``d / 2`` float64 radians per
    position (None: no rotation); their ``n`` pairs are elements ``(i, i + n)`` of the head, or ``(2i, 2i + 1)`` when
    ``interleaved``; the rest of the head is not rotated.  ``positions``: int64 ``(l,)`` or ``(b, l)`` (None: 0, 1, ...),
    reduced in 64 bits, so far ones are as exact as near ones (up to 2^28; behind it a bit is lost with every doubling).  The
    squares of a head add up in float32: elements below 1e19.  ``magnitude`` multiplies the rotated part.  Types and
    strides as in ``gated_delta_rule``; results are contiguous."""
    _refuse_traced("qk_norm_rotate", q, k, frequencies, positions, q_weight, k_weight)
    if not isinstance(q, Tensor) or not q.is_cuda:
        raise RuntimeError("q must be a CUDA tensor (there is no CPU implementation of this operator)")
    if q.dtype not in _DTYPES:
        raise RuntimeError(f"q must be float32, bfloat16 or float16, got {q.dtype}")
    if q.dim() != 4 or not isinstance(k, Tensor) or k.dim() != 4:
        raise RuntimeError("q and k must be (batch, length, heads, width)")
    if norm not in _NORMS:
        raise RuntimeError(f'norm must be "rms", "l2" or None, got {norm!r}')
    b, l, hq, d = q.shape
    if (b | l | hq | k.shape[2]) >> 31:
        raise RuntimeError(f"batch {b}, length {l}, heads {hq} and {k.shape[2]}: sizes below 2^31 are supported")
    if not 1 <= d <= MAX_HEAD or hq == 0 or k.shape[2] == 0:
        raise RuntimeError(f"heads of {d} elements: 1 to {MAX_HEAD} are supported, and one head at least")
    dev = q.device
    q = _typed("q", q, q.dtype, (b, l, hq, d), dev)
    k = _typed("k", k, q.dtype, (b, l, k.shape[2], d), dev)
    q_weight = None if q_weight is None else _typed("q_weight", q_weight, torch.float32, (d,), dev)
    k_weight = None if k_weight is None else _typed("k_weight", k_weight, torch.float32, (d,), dev)
    n, stride = 0, 0
    if frequencies is not None:
        n = frequencies.numel()
        if frequencies.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("qk_norm_rotate is not differentiable in the frequencies: detach them")
        if 2 * n > d:
            raise RuntimeError(f"{n} frequencies for heads of {d} elements: at most {d // 2}")
        frequencies = _typed("frequencies", frequencies, torch.float64, (n,), dev).contiguous()
    if positions is not None:
        shape = (l,) if positions.dim() == 1 else (b, l)
        positions = _typed("positions", positions, torch.int64, shape, dev).contiguous()
        stride = 0 if positions.dim() == 1 else l
    p = _problem(b, l, hq, k.shape[2], d, 2 * n, _DTYPES[q.dtype], _NORMS[norm], int(bool(interleaved)), float(eps), float(magnitude),
                 stride, *q.stride()[:3], *k.stride()[:3])
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, q_weight, k_weight)):
        return _NormRotate.apply(q, k, q_weight, k_weight, frequencies, positions, p)
    return _forward(q, k, q_weight, k_weight, frequencies, positions, p)
