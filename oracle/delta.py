"""Token-by-token restatement of the gated delta rule, of the per-head norm and of the rotation, for the tests.

Written from the formulas, in plain differentiable torch; run in float64 it is the truth the kernels are held to.
"""
from __future__ import annotations

import math

import torch


def gated_delta_ref(q, k, v, g, beta, scale=None, initial_state=None):
    """``q, k`` (b, l, hk, dk), ``v`` (b, l, hv, dv), ``g, beta`` (b, l, hv) -> (o (b, l, hv, dv), state (b, hv, dk, dv))."""
    b, l, hk, dk = q.shape
    hv, dv = v.shape[2:]
    scale = 1.0 / math.sqrt(dk) if scale is None else scale
    q, k = (x.repeat_interleave(hv // hk, 2) for x in (q, k))
    S = torch.zeros(b, hv, dk, dv, dtype=v.dtype, device=v.device) if initial_state is None else initial_state
    outs = []
    for t in range(l):
        S = S * torch.exp(g[:, t])[..., None, None]
        e = beta[:, t, :, None] * (v[:, t] - torch.einsum("bhkv,bhk->bhv", S, k[:, t]))
        S = S + k[:, t, :, :, None] * e[:, :, None, :]
        outs.append(scale * torch.einsum("bhkv,bhk->bhv", S, q[:, t]))
    o = torch.stack(outs, 1) if outs else v.new_zeros(b, 0, hv, dv)
    return o, S


def norm_rotate_ref(x, frequencies=None, positions=None, weight=None, norm="rms", eps=1e-6, interleaved=False,
                    magnitude=1.0):
    """One of the two tensors of ``qk_norm_rotate``: ``x`` (b, l, h, d) normalised over d and rotated pair by pair."""
    y = x
    if norm == "rms":
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps)
    elif norm == "l2":
        y = y / torch.sqrt((y * y).sum(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight
    if frequencies is None or frequencies.numel() == 0:
        return y
    b, l, _, d = x.shape
    n = frequencies.numel()
    positions = torch.arange(l, device=x.device) if positions is None else positions
    angle = (positions.double()[..., None] * frequencies.double()).expand(b, l, n)[:, :, None]
    cos, sin = (magnitude * torch.cos(angle)).to(y.dtype), (magnitude * torch.sin(angle)).to(y.dtype)
    i = torch.arange(n, device=x.device)
    first, second = (2 * i, 2 * i + 1) if interleaved else (i, i + n)
    a, c = y[..., first], y[..., second]
    return y.index_copy(-1, first, a * cos - c * sin).index_copy(-1, second, c * cos + a * sin)
