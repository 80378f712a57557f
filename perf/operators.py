"""The operators of the gated-delta mixer: what is measured, on which sizes, and their plain forms.

Kinds of work (``case["kind"]``):

``delta``   ``aussm_b200.delta.gated_delta_rule``: a sequence through the gated delta rule.  Per value head, with the
            state S (dk, dv), a_t = exp(g_t) and e_t = beta_t (v_t - a_t S_{t-1}^T k_t):
                S_t = a_t S_{t-1} + k_t e_t^T,     o_t = scale S_t^T q_t
            ``train`` asks for the output and every gradient, otherwise output and final state come back.
``step``    ``aussm_b200.delta.gated_delta_step``: the same recurrence for one or a few new tokens of many sequences.
``rotate``  ``aussm_b200.rotary.qk_norm_rotate``: queries and keys normalised per head and rotated by position.

``dtype`` is the type of queries, keys and values; decays, step sizes and states are float32 whatever it is.
"""
from __future__ import annotations

import math

import torch

own = False

CHUNK = 64
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # A training call of a test-sized model: launches and host work are all there is.
        dict(name="delta_small", kind="delta", b=2, l=48, hk=2, hv=2, dk=32, dv=32, dtype="float32", train=True, state=False),
        # Ragged training data: nothing is a multiple of a chunk, value heads share key heads, a state is handed on.
        dict(name="delta_ragged", kind="delta", b=3, l=1003, hk=3, hv=6, dk=72, dv=100, dtype="float32", train=True, state=True),
        # A training batch of the benchmark's width (inner width 1024 as 8 heads of 128) over 4096 steps.
        dict(name="delta_wide", kind="delta", b=4, l=4096, hk=8, hv=8, dk=128, dv=128, dtype="float32", train=True, state=False),
        # The token classifier's sequence: one row of 65536 tokens at width 512, all parallelism from the time axis.
        dict(name="delta_long", kind="delta", b=1, l=65536, hk=4, hv=4, dk=128, dv=128, dtype="float32", train=True, state=False),
        # Reading a batch of prompts in bfloat16 before single tokens are made: output and final state.
        dict(name="delta_prompt", kind="delta", b=8, l=4096, hk=8, hv=16, dk=128, dv=128, dtype="bfloat16", train=False, state=True),
        # One new token of one sequence: latency.
        dict(name="step_single", kind="step", b=1, l=1, hk=8, hv=8, dk=128, dv=128, dtype="bfloat16"),
        # One new token of a full batch: every state is read and written once.
        dict(name="step_batch", kind="step", b=256, l=1, hk=8, hv=16, dk=128, dv=128, dtype="bfloat16"),
        # One new token of a small batch, normalised and rotated: latency.
        dict(name="rotate_single", kind="rotate", b=16, l=1, hq=8, hk=8, d=128, rot=128, norm="l2", layout="half", far=0, dtype="bfloat16", train=False),
        # Ragged training data, a part of the head rotated in the interleaved layout, positions restarting inside rows.
        dict(name="rotate_ragged", kind="rotate", b=3, l=1021, hq=6, hk=2, d=80, rot=32, norm="rms", layout="interleaved", far=0, dtype="bfloat16", train=True),
        # The queries and keys of delta_wide.
        dict(name="rotate_wide", kind="rotate", b=4, l=4096, hq=8, hk=8, d=128, rot=128, norm="rms", layout="half", far=0, dtype="float32", train=True),
        # A long context read piece by piece: positions around a million, half of each head rotated.
        dict(name="rotate_far", kind="rotate", b=2, l=65536, hq=8, hk=4, d=128, rot=64, norm="rms", layout="half", far=1 << 20, dtype="bfloat16", train=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, hi):
    return rng.choice([16, 32, 64, 64, 96, 128, 128, rng.randint(5, hi)])


def draw(rng):
    kind = rng.choice(["delta", "delta", "delta", "step", "rotate", "rotate"])
    dtype = rng.choice(["float32", "float32", "bfloat16", "bfloat16", "float16"])
    if kind == "rotate":
        b, l, d = _log_int(rng, 1, 32), _log_int(rng, 1, 65536), rng.choice([32, 64, 80, 96, 128, 128, 192, 256, rng.randint(4, 256)])
        hk = _log_int(rng, 1, 16)
        hq = hk * rng.choice([1, 1, 2, 4])
        while b * l * (hq + hk) * d > 1 << 27:
            b, l = max(1, b // 2), max(1, l * 2 // 3)
        rot = rng.choice([d // 2 * 2, d // 2 * 2, d // 4 * 2, 2 * rng.randint(1, d // 2)])
        return dict(kind=kind, b=b, l=l, hq=hq, hk=hk, d=d, rot=rot, norm=rng.choice(["rms", "l2", "none"]),
                    layout=rng.choice(["half", "interleaved"]), far=rng.choice([0, 0, rng.randint(1, 1 << 22)]), dtype=dtype,
                    train=rng.random() < 0.6)
    b, dk, dv = _log_int(rng, 1, 16), _width(rng, 128), _width(rng, 256)
    hk = _log_int(rng, 1, 8)
    hv = hk * rng.choice([1, 1, 2, 3])
    if kind == "step":
        return dict(kind=kind, b=_log_int(rng, 1, 256), l=rng.choice([1, 1, 1, 2, 4]), hk=hk, hv=min(hv, 2 * hk), dk=dk, dv=min(dv, 128), dtype=dtype)
    l = _log_int(rng, 1, 32768)
    while b * l * hv * dk * dv > 1 << 31:               # half of delta_wide's products
        b, l = max(1, b // 2), max(1, l * 2 // 3)
    return dict(kind=kind, b=b, l=l, hk=hk, hv=hv, dk=dk, dv=dv, dtype=dtype, train=rng.random() < 0.6, state=rng.random() < 0.5)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _unit(x):
    return x / x.square().sum(-1, keepdim=True).add(1e-6).sqrt()


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    dtype = TYPES[case["dtype"]]

    def r(*s):
        return torch.randn(*s, device=dev, generator=gen)

    train = case.get("train", False)
    b, l = case["b"], case["l"]
    if case["kind"] == "rotate":
        hq, hk, d, rot = (case[x] for x in ("hq", "hk", "d", "rot"))
        s = dict(case=case, q=r(b, l, hq, d).to(dtype), k=r(b, l, hk, d).to(dtype))
        if case["norm"] == "rms":
            s["q_weight"], s["k_weight"] = 1 + 0.2 * r(d), 1 + 0.2 * r(d)
        # radians per position; far positions come with stretched (slower) angles, as a model read past its length has
        s["frequencies"] = (10000.0 * (8.0 if case["far"] else 1.0)) ** (-torch.arange(rot // 2, device=dev, dtype=torch.float64) * 2 / rot)
        start = torch.randint(0, max(1, l), (b, 1), device=dev, generator=gen)
        s["positions"] = (torch.arange(l, device=dev)[None] + start) % max(1, l) + case["far"]      # packed rows: restarts
        if train:
            s["gq"], s["gk"] = r(b, l, hq, d).to(dtype), r(b, l, hk, d).to(dtype)
            for n in ("q", "k", "q_weight", "k_weight"):
                if n in s:
                    s[n].requires_grad_()
        return s
    hk, hv, dk, dv = (case[x] for x in ("hk", "hv", "dk", "dv"))
    rate = torch.exp(torch.rand(hv, device=dev, generator=gen) * math.log(400.0) + math.log(0.01))   # heads forget fast or slowly
    s = dict(case=case, q=_unit(r(b, l, hk, dk)).to(dtype), k=_unit(r(b, l, hk, dk)).to(dtype), v=r(b, l, hv, dv).to(dtype),
             g=-rate * torch.nn.functional.softplus(r(b, l, hv)), beta=torch.sigmoid(r(b, l, hv)))
    if case["kind"] == "step":
        s["state"] = r(b, hv, dk, dv) / math.sqrt(dk)
        s["new_state"] = torch.empty_like(s["state"])
        return s
    s["state"] = r(b, hv, dk, dv) / math.sqrt(dk) if case["state"] else None
    if train:
        s["go"] = r(b, l, hv, dv).to(dtype)
        for n in ("q", "k", "v", "g", "beta", "state"):
            if s[n] is not None:
                s[n].requires_grad_()
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _inverse(a):
    """(I + a)^-1 for strictly lower triangular a (..., n, n), n a power of two, by halves."""
    n = a.shape[-1]
    if n == 1:
        return torch.ones_like(a)
    h = n // 2
    both = _inverse(torch.stack((a[..., :h, :h], a[..., h:, h:])))
    low = -(both[1] @ a[..., h:, :h] @ both[0])
    return torch.cat((torch.cat((both[0], torch.zeros_like(low)), -1), torch.cat((low, both[1]), -1)), -2)


def _heads(x, r, c):
    """(b, l, h, d) -> (b, h r, chunks, c, d) in 32 bits, zeros behind the end."""
    b, l, h, d = x.shape
    x = torch.nn.functional.pad(x.float(), (0, 0, 0, 0, 0, -l % c))
    x = x.view(b, -1, c, h, d).permute(0, 3, 1, 2, 4)
    return x.repeat_interleave(r, 1) if r > 1 else x


def _delta(q, k, v, g, beta, state):
    """The gated delta rule a chunk at a time: the sums over a chunk's earlier steps as a triangular system."""
    b, l, hk, dk = q.shape
    hv, dv = v.shape[2:]
    c = min(CHUNK, 1 << (l - 1).bit_length())
    Q, K, V = _heads(q * 1.0, hv // hk, c), _heads(k, hv // hk, c), _heads(v, 1, c)
    Q = Q * dk ** -0.5
    be = _heads(beta[..., None], 1, c)
    G = _heads(g[..., None], 1, c)[..., 0].double().cumsum(-1)
    diff = G[..., :, None] - G[..., None, :]
    upto = torch.ones(c, c, device=q.device, dtype=torch.bool).tril()
    D = torch.where(upto, diff, -math.inf).exp().float()
    A = (be * D * (K @ K.transpose(-1, -2))).tril(-1)
    T = _inverse(A)
    since = G.exp().float()[..., None]
    until = (G[..., -1:] - G).exp().float()[..., None]
    U, W = T @ (be * V), T @ (be * since * K)
    P = D * (Q @ K.transpose(-1, -2))
    Kt, whole = (until * K).transpose(-1, -2), since[..., -1:, :]
    S = torch.zeros(b, hv, dk, dv, device=q.device) if state is None else state.float()
    states, news = [], []
    for i in range(U.shape[2]):
        new = U[:, :, i] - W[:, :, i] @ S
        states.append(S)
        news.append(new)
        S = whole[:, :, i] * S + Kt[:, :, i] @ new
    O = (since * Q) @ torch.stack(states, 2) + P @ torch.stack(news, 2)
    return O.permute(0, 2, 3, 1, 4).reshape(b, -1, hv, dv)[:, :l].to(q.dtype), S


def _rotate(x, weight, frequencies, positions, norm, layout):
    d, rot = x.shape[-1], 2 * frequencies.shape[0]
    y = x.float()
    if norm == "rms":
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * weight
    elif norm == "l2":
        y = y * torch.rsqrt(y.square().sum(-1, keepdim=True) + 1e-6)
    angle = (positions[..., None].double() * frequencies)[:, :, None]
    cos, sin = angle.cos().float(), angle.sin().float()
    z = y[..., :rot]
    a, c = (z[..., :rot // 2], z[..., rot // 2:]) if layout == "half" else (z[..., 0::2], z[..., 1::2])
    a, c = a * cos - c * sin, c * cos + a * sin
    z = torch.cat((a, c), -1) if layout == "half" else torch.stack((a, c), -1).flatten(-2)
    return torch.cat((z, y[..., rot:]), -1).to(x.dtype)


# ---------------------------------------------------------------------------
# a pass
# ---------------------------------------------------------------------------
def run(s):
    case = s["case"]
    if case["kind"] == "step":
        if own:
            from aussm_b200.delta import gated_delta_step
            o = gated_delta_step(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"], new_state=s["new_state"])
            return {"o": o, "state": s["new_state"]}
        o, state = _delta(s["q"], s["k"], s["v"], s["g"], s["beta"], s["state"])
        return {"o": o, "state": state}
    if case["kind"] == "delta":
        names = [n for n in ("q", "k", "v", "g", "beta", "state") if s[n] is not None]
        if own:
            from aussm_b200.delta import gated_delta_rule
            got = gated_delta_rule(s["q"], s["k"], s["v"], s["g"], s["beta"], initial_state=s["state"],
                                   return_final_state=not case["train"])
            o, state = (got, None) if case["train"] else got
        else:
            o, state = _delta(*(s[n] for n in ("q", "k", "v", "g", "beta", "state")))
        if not case["train"]:
            return {"o": o, "state": state}
        return {"o": o.detach(), **dict(zip(names, torch.autograd.grad(o, [s[n] for n in names], s["go"])))}
    names = [n for n in ("q", "k", "q_weight", "k_weight") if n in s]
    if own:
        from aussm_b200.rotary import qk_norm_rotate
        q, k = qk_norm_rotate(s["q"], s["k"], s["frequencies"], s["positions"], q_weight=s.get("q_weight"), k_weight=s.get("k_weight"),
                              norm=None if case["norm"] == "none" else case["norm"], eps=1e-6, interleaved=case["layout"] == "interleaved")
    else:
        q, k = (_rotate(s[n], s.get(n + "_weight"), s["frequencies"], s["positions"], case["norm"], case["layout"]) for n in ("q", "k"))
    if not case["train"]:
        return {"yq": q, "yk": k}
    return {"yq": q.detach(), "yk": k.detach(), **dict(zip(names, torch.autograd.grad([q, k], [s[n] for n in names], [s["gq"], s["gk"]])))}


# ---------------------------------------------------------------------------
# work, exact values
# ---------------------------------------------------------------------------
def work(case):
    size = TYPES[case["dtype"]].itemsize
    b, l, train = case["b"], case["l"], case.get("train", False)
    if case["kind"] == "rotate":
        rows, d = b * l * (case["hq"] + case["hk"]), case["d"]
        # forward: in and out; backward: the gradient in and out (the inputs are not read twice); one position a token
        moved = rows * d * size * (4 if train else 2) + 8 * b * l
        return {"bytes": moved, "flops": rows * d * (24 if train else 8)}
    hk, hv, dk, dv = (case[x] for x in ("hk", "hv", "dk", "dv"))
    tokens = b * l
    inputs = tokens * ((2 * hk * dk + hv * dv) * size + 2 * hv * 4)
    states = b * hv * dk * dv * 4
    out = tokens * hv * dv * size
    flops = 6 * tokens * hv * dk * dv                      # S^T k, k e^T, S^T q
    if train:                                              # inputs once, output, its gradient, the inputs' gradients
        return {"bytes": 2 * inputs + 2 * out + (2 * states if case["state"] else 0), "flops": 3 * flops}
    return {"bytes": inputs + out + states * (2 if case["kind"] == "step" or case["state"] else 1), "flops": flops}


def _steps(q, k, v, decay, beta, S):
    """The recurrence itself, a token at a time, on (l, b, h, d) in 64 bits."""
    outs = []
    for t in range(q.shape[0]):
        S = S * decay[t]
        e = beta[t] * (v[t] - (S * k[t][..., :, None]).sum(-2))
        S = S + k[t][..., :, None] * e[..., None, :]
        outs.append((S * q[t][..., :, None]).sum(-2))
    return torch.stack(outs), S


def _exact_delta(case, s):
    b, l, hk, dk = s["q"].shape
    hv, dv = s["v"].shape[2:]
    train = case.get("train", False)
    names = [n for n in ("q", "k", "v", "g", "beta", "state") if s[n] is not None]
    x = {n: s[n].detach().double().requires_grad_(train) for n in names}
    q = x["q"].repeat_interleave(hv // hk, 2).transpose(0, 1) / math.sqrt(dk)
    k = x["k"].repeat_interleave(hv // hk, 2).transpose(0, 1)
    v, decay, beta = x["v"].transpose(0, 1), x["g"].exp().transpose(0, 1)[..., None, None], x["beta"].transpose(0, 1)[..., None]
    S = x.get("state")
    S = torch.zeros(b, hv, dk, dv, device=q.device, dtype=torch.float64) if S is None else S
    pieces = []
    for t in range(0, l, 64):
        part = [y[t:t + 64] for y in (q, k, v, decay, beta)] + [S]
        o, S = torch.utils.checkpoint.checkpoint(_steps, *part, use_reentrant=False) if train else _steps(*part)
        pieces.append(o)
    o = torch.cat(pieces).transpose(0, 1)
    if not train:
        return {"o": o, "state": S}
    return {"o": o.detach(), **dict(zip(names, torch.autograd.grad(o, [x[n] for n in names], s["go"].double())))}


def _exact_rotate(case, s):
    names = [n for n in ("q", "k", "q_weight", "k_weight") if n in s]
    x = {n: s[n].detach().double().requires_grad_(case["train"]) for n in names}
    half = s["frequencies"].shape[0]
    turn = torch.polar(torch.ones((), device=s["q"].device, dtype=torch.float64), s["positions"].double()[..., None] * s["frequencies"])[:, :, None]
    outs = []
    for n in ("q", "k"):
        y = x[n]
        if case["norm"] != "none":
            power = (y * y).sum(-1, keepdim=True) / (y.shape[-1] if case["norm"] == "rms" else 1)
            y = y / torch.sqrt(power + 1e-6)
        if case["norm"] == "rms":
            y = y * x[n + "_weight"]
        first = torch.arange(half, device=y.device) if case["layout"] == "half" else 2 * torch.arange(half, device=y.device)
        second = first + (half if case["layout"] == "half" else 1)
        z = torch.complex(y[..., first], y[..., second]) * turn
        outs.append(y.index_copy(-1, first, z.real).index_copy(-1, second, z.imag))
    got = {"yq": outs[0].detach(), "yk": outs[1].detach()}
    if case["train"]:
        got |= dict(zip(names, torch.autograd.grad(outs, [x[n] for n in names], [s["gq"].double(), s["gk"].double()])))
    return got


def exact(case, seed):
    import torch.utils.checkpoint  # noqa: F401
    if case["kind"] == "rotate":
        return _exact_rotate(case, prepare(case, seed))
    cost = case["l"] * (4 if case.get("train") else 1)     # a token is some launches, a trained one some more
    return None if cost > 24000 else _exact_delta(case, prepare(case, seed))
