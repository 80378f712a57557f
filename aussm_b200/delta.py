"""The gated delta rule on B200: a sequence mixer with a matrix state.

Per batch entry and value head, with ``a_t = exp(g_t)`` and the state ``S`` (dk, dv)::

    e_t = beta_t (v_t - a_t S_{t-1}^T k_t)        what the state does not yet answer to the key, times the step size
    S_t = a_t S_{t-1} + k_t e_t^T
    o_t = scale S_t^T q_t

``gated_delta_rule`` takes whole sequences (a chunk of 64 steps at a time, forward and backward),
``gated_delta_step`` one or a few new steps of many sequences, in float32.  The products of the rule carry 22 bits of their
operands (two FP16 parts each) and float32 sums: results differ from the recurrence by about 1e-6, a plain float32 chunk form by
4e-7, for every input type, before the rounding to 16 bits.  CUDA tensors only; all arithmetic runs in libaussm_b200.so.
"""
from __future__ import annotations

import contextlib
import ctypes
import functools
from typing import Optional

import torch
from torch import Tensor

from . import _lib
from .ops import _PLAIN, _eager, _poll_status, _ptr, _workspace

__all__ = ["gated_delta_rule", "gated_delta_step", "MAX_KEY", "MAX_VALUE"]

MAX_KEY, MAX_VALUE = 128, 256            # widths of a head that the kernels take
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _refuse_traced(what: str, *tensors) -> None:
    """A kernel that writes through raw pointers is invisible to tracers and function transforms: refuse them."""
    plain = True
    for t in tensors:
        plain = plain and (t is None or type(t) in _PLAIN)
    if plain and _eager():
        return
    from torch.fx.experimental.proxy_tensor import get_proxy_mode
    if (not plain or torch._C._are_functorch_transforms_active() or torch.autograd.forward_ad._current_level >= 0
            or torch.compiler.is_compiling() or torch._C._is_tracing() or get_proxy_mode() is not None):
        raise RuntimeError(f"{what} runs eagerly on plain tensors: no function transforms, forward-mode differentiation, "
                           "tracing or tensor subclasses")


def _typed(name: str, t: Tensor, dtype, shape, device) -> Tensor:
    """``t`` checked, with unit stride along its last axis (a copy only where it has not)."""
    if (type(t) in _PLAIN and t.device == device and t.dtype is dtype and t.shape == shape and t.stride(-1) == 1
            and not t.is_neg() and t.is_cuda):
        return t                                        # as most are: short calls are bound by the host
    if not isinstance(t, Tensor) or not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor (there is no CPU implementation of this operator)")
    if t.device != device:
        raise RuntimeError(f"{name} is on {t.device}, expected {device}")
    if t.dtype != dtype:
        raise RuntimeError(f"{name} must be {dtype}, got {t.dtype}")
    if tuple(t.shape) != tuple(shape):
        raise RuntimeError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    return _plain(t)


def _plain(t: Tensor) -> Tensor:
    """``t`` with unit stride along its last axis and its sign in memory (parts of conjugate tensors have it in a flag)."""
    if t.is_neg():
        t = t.resolve_neg()
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


_HERE = contextlib.nullcontext()


def _on(device):
    """The device as the current one.  Short calls are bound by the host: nothing is entered where it is already."""
    return _HERE if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def _raw_stream(device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


def _strides(t: Tensor):
    return (ctypes.c_longlong * 3)(*t.stride()[:3])


@functools.lru_cache(maxsize=256)
def _problem(b, l, hk, hv, dk, dv, dtype, scale, *strides):
    """The problem of these sizes, types and strides: read only (the backward call takes a copy)."""
    q, k, v = ((ctypes.c_longlong * 3)(*strides[i:i + 3]) for i in (0, 3, 6))
    return _lib.DeltaProblem(b, l, hk, hv, dk, dv, dtype, scale, q, k, v)


def _check(q, k, v, g, beta, scale):
    """The problem, and the inputs as the kernels take them."""
    if not isinstance(q, Tensor) or not q.is_cuda:
        raise RuntimeError("q must be a CUDA tensor (there is no CPU implementation of this operator)")
    if q.dtype not in _DTYPES:
        raise RuntimeError(f"q must be float32, bfloat16 or float16, got {q.dtype}")
    if q.dim() != 4 or not isinstance(v, Tensor) or v.dim() != 4:
        raise RuntimeError("q, k and v must be (batch, length, heads, width)")
    b, l, hk, dk = q.shape
    hv, dv = v.shape[2:]
    if (b | l | hk | hv) >> 31:
        raise RuntimeError(f"batch {b}, length {l}, heads {hk} and {hv}: sizes below 2^31 are supported")
    if hk == 0 or hv == 0 or hv % hk:
        raise RuntimeError(f"the {hv} value heads must be a multiple of the {hk} key heads")
    if not (1 <= dk <= MAX_KEY and 1 <= dv <= MAX_VALUE):
        raise RuntimeError(f"heads of {dk} keys and {dv} values: 1 to {MAX_KEY} and 1 to {MAX_VALUE} are supported")
    q = _typed("q", q, q.dtype, (b, l, hk, dk), q.device)
    k = _typed("k", k, q.dtype, (b, l, hk, dk), q.device)
    v = _typed("v", v, q.dtype, (b, l, hv, dv), q.device)
    g = _typed("g", g, torch.float32, (b, l, hv), q.device).contiguous()
    beta = _typed("beta", beta, torch.float32, (b, l, hv), q.device).contiguous()
    p = _problem(b, l, hk, hv, dk, dv, _DTYPES[q.dtype], dk ** -0.5 if scale is None else float(scale), *q.stride()[:3],
                 *k.stride()[:3], *v.stride()[:3])
    return p, q, k, v, g, beta


def _state(name: str, s: Tensor, p, device) -> Tensor:
    return _typed(name, s, torch.float32, (p.B, p.HV, p.DK, p.DV), device).contiguous()


def _forward(p, q, k, v, g, beta, state, want_state, train):
    """``(o, final state or None, what the backward call reads or None)``"""
    o = torch.empty((p.B, p.L, p.HV, p.DV), device=q.device, dtype=q.dtype)
    last = torch.empty((p.B, p.HV, p.DK, p.DV), device=q.device, dtype=torch.float32) if want_state else None
    if o.numel() == 0:
        if last is not None:
            last.zero_() if state is None else last.copy_(state)
        return o, last, None
    lib = _lib.load()
    with _on(q.device):
        size = lib.aussm_b200_delta_keep_bytes(p) if train else lib.aussm_b200_delta_workspace_bytes(p, 0)
        room = _workspace(size, q.device)
        rc = lib.aussm_b200_delta_fwd(p, _ptr(q), _ptr(k), _ptr(v), _ptr(g), _ptr(beta), _ptr(state), _ptr(o), _ptr(last),
                                      _ptr(room) if train else None, size if train else 0, None if train else _ptr(room),
                                      0 if train else size, _raw_stream(q.device))
    _lib.check(rc, "gated_delta_rule")
    _poll_status("gated_delta_rule", q.device)
    return o, last, room if train else None


class _GatedDelta(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, beta, state, scale, want_state):
        p, q, k, v, g, beta = _check(q, k, v, g, beta, scale)
        state = None if state is None else _state("initial_state", state, p, q.device)
        o, last, keep = _forward(p, q, k, v, g, beta, state, want_state, True)
        ctx.set_materialize_grads(False)
        ctx.p, ctx.has_state = p, state is not None
        ctx.save_for_backward(q, k, v, g, beta, keep)
        return o, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, go, glast):
        q, k, v, g, beta, keep = ctx.saved_tensors
        p = type(ctx.p).from_buffer_copy(ctx.p)         # of this call's own: the gradient's strides go in
        dq, dk, dv = (torch.empty(t.shape, device=t.device, dtype=t.dtype) for t in (q, k, v))
        dg, dbeta = torch.empty_like(g), torch.empty_like(beta)
        ds0 = None
        if ctx.has_state and ctx.needs_input_grad[5]:
            ds0 = torch.empty(p.B, p.HV, p.DK, p.DV, device=q.device, dtype=torch.float32)
        if glast is not None:
            glast = _plain(glast).contiguous()
        if keep is None:                                # no steps
            if ds0 is not None:
                ds0.zero_() if glast is None else ds0.copy_(glast)
            return dq, dk, dv, dg, dbeta, ds0, None, None
        go = torch.zeros(v.shape, device=v.device, dtype=v.dtype) if go is None else go
        go = _plain(go)
        p.go_stride = _strides(go)
        lib = _lib.load()
        with _on(q.device):
            ws = _workspace(lib.aussm_b200_delta_workspace_bytes(p, 1), q.device)
            rc = lib.aussm_b200_delta_bwd(p, _ptr(go), _ptr(glast), _ptr(q), _ptr(k), _ptr(v), _ptr(g), _ptr(beta), _ptr(keep),
                                          keep.numel(), _ptr(dq), _ptr(dk), _ptr(dv), _ptr(dg), _ptr(dbeta), _ptr(ds0),
                                          _ptr(ws), ws.numel(), _raw_stream(q.device))
        _lib.check(rc, "gated_delta_rule backward")
        _poll_status("gated_delta_rule backward", q.device)
        return dq, dk, dv, dg, dbeta, ds0, None, None


def gated_delta_rule(q: Tensor, k: Tensor, v: Tensor, g: Tensor, beta: Tensor, scale: Optional[float] = None,
                     initial_state: Optional[Tensor] = None, return_final_state: bool = False):
    """The gated delta rule over whole sequences; differentiable once in every tensor.

    ``q, k`` are ``(b, l, hk, dk)`` and ``v`` ``(b, l, hv, dv)``, of one type (float32, bfloat16 or float16) and any
    strides; ``hv`` is a multiple of ``hk`` and value head ``h`` reads key head ``h // (hv // hk)``.  ``g`` (logarithm of
    the decay; -inf forgets the state) and ``beta`` (step size) are ``(b, l, hv)`` float32.  Keys are meant to have unit
    length (``rotary.qk_norm_rotate``) and ``beta`` to lie in 0..2 (larger keys: ``beta |k|^2``): otherwise the recurrence
    itself diverges.  A padded step is one with ``g = beta = 0``: it leaves the state as it is, whatever its key and value hold
    (what is not finite in them counts as zero; of a key, where ``beta`` is zero for all value heads that share it).
    ``scale`` defaults to ``dk ** -0.5``.  ``initial_state`` is ``(b, hv, dk, dv)`` float32 (None: zero).

    Outputs and gradients of ``q`` are right to their own query's size, whatever the other steps hold.  Everything else that
    is summed over the steps of a chunk (64) is rounded to the largest term in the chunk: an outlying value shows in its value column
    with about 1e-7 of itself from its step on (as in any float32 sum), but also with about 1e-11 of itself in the steps
    before it in its chunk, which counts from 1e6 times the others on; so do outlying gradients.  An entry that is not finite
    makes what depends on it non-finite, and may do so for the steps before it in its chunk (a query: only its own output,
    and gradients of the chunks up to its own).

    A step and value head of 128 keys and values takes 2.1 KB of workspace; with gradients 3.6 KB are kept until the backward
    pass, which takes another 1.5 KB (256 values: 5.2 and 3.1 KB).  A very long sequence can be read in pieces that hand the state
    on.

    Returns ``o`` ``(b, l, hv, dv)`` of the inputs' type, or ``(o, final_state)``."""
    _refuse_traced("gated_delta_rule", q, k, v, g, beta, initial_state)
    grad = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, g, beta, initial_state))
    if grad:
        o, last = _GatedDelta.apply(q, k, v, g, beta, initial_state, scale, bool(return_final_state))
    else:
        p, q, k, v, g, beta = _check(q, k, v, g, beta, scale)
        state = None if initial_state is None else _state("initial_state", initial_state, p, q.device)
        o, last, _ = _forward(p, q, k, v, g, beta, state, bool(return_final_state), False)
    return (o, last) if return_final_state else o


def gated_delta_step(q: Tensor, k: Tensor, v: Tensor, g: Tensor, beta: Tensor, state: Tensor, scale: Optional[float] = None,
                     new_state: Optional[Tensor] = None) -> Tensor:
    """One or a few new steps of every sequence, for serving: reads each state once and writes it once.

    Tensors as in ``gated_delta_rule`` with ``l`` the number of new steps.  ``state`` ``(b, hv, dk, dv)`` float32
    contiguous is updated in place, or left alone when ``new_state`` (same shape, no overlap) is given to take the
    result.  Returns ``o``.  Not differentiable."""
    _refuse_traced("gated_delta_step", q, k, v, g, beta, state, new_state)
    tensors = (q, k, v, g, beta, state, new_state)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError("gated_delta_step is not differentiable: call it under torch.no_grad(), or use gated_delta_rule")
    p, q, k, v, g, beta = _check(q, k, v, g, beta, scale)
    out = state if new_state is None else new_state
    state = _state("state", state, p, q.device)
    if not out.is_contiguous() or out.is_neg() or tuple(out.shape) != tuple(state.shape) or out.dtype != torch.float32 or out.device != q.device:
        raise RuntimeError(f"the state that takes the result must be contiguous float32 {tuple(state.shape)} on {q.device}")
    if new_state is not None and state.numel():
        lo, hi, size = sorted((state.data_ptr(), out.data_ptr())) + [4 * state.numel()]
        if lo != hi and hi < lo + size:
            raise RuntimeError("new_state overlaps state in part")
    o = torch.empty((p.B, p.L, p.HV, p.DV), device=q.device, dtype=q.dtype)
    if o.numel() == 0:
        if out.data_ptr() != state.data_ptr():
            out.copy_(state)
        return o
    with _on(q.device):
        rc = _lib.load().aussm_b200_delta_step(p, _ptr(q), _ptr(k), _ptr(v), _ptr(g), _ptr(beta), _ptr(state), _ptr(out),
                                               _ptr(o), _raw_stream(q.device))
    _lib.check(rc, "gated_delta_step")
    if not out.is_inference():                          # written in place: a graph that has saved it must not use it
        torch.autograd.graph.increment_version(out)
    return o
