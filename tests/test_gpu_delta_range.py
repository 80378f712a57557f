"""Gated delta rule with single entries far out of the range of the others, infinite or NaN, step by step against the
recurrence in float64.

Tolerances.  What a query or its gradient of the output touches is its own row of each product, so the output of step t is
off by at most FWD (see test_gpu_delta.py: 8 products of 2^-21, sqrt(128) between a sum of magnitudes and its result) of
|q_t| times the largest o / |q| of the head, whatever the other queries hold, and its gradient dq_t by BWD of |go_t| times the
largest dq / |go|.  Sums over the steps of a chunk (64) are rounded to the largest of their terms: a large value shows in the
other outputs of its value column and chunk, by FWD of itself, and nowhere else.
"""
import math

import pytest
import torch

import aussm_b200
from aussm_b200.delta import gated_delta_rule, gated_delta_step
from oracle.delta import gated_delta_ref
from tests.test_gpu_delta import BWD, FWD, NAMES, make

pytestmark = pytest.mark.gpu
CHUNK = 64


def run(d, go=None, fn=gated_delta_rule, dtype=None):
    """Output, final state and (with go) the gradients."""
    x = {n: (t if dtype is None else t.to(dtype)).detach().clone().requires_grad_(go is not None) for n, t in d.items()}
    kw = dict(return_final_state=True) if fn is gated_delta_rule else {}
    o, s = fn(*(x[n] for n in NAMES[:5]), initial_state=x["state"], **kw)
    grads = None if go is None else dict(zip(x, torch.autograd.grad(o, list(x.values()), go.to(o.dtype))))
    return o.detach(), s.detach(), grads


def truth(d, go=None):
    return run(d, go, gated_delta_ref, torch.float64)


def go_like(d, seed=5):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(d["v"].shape, device="cuda", generator=gen).to(d["v"].dtype)


def by_rows(name, got, want, size, tol, steps=None):
    """|got - want| of every step within tol of `size` (b, l, heads) times the head's largest |want| / size, and half a step
    of the type; on `steps` (b, l), default all."""
    want = want.double()
    size = size.double()[..., None]
    there = torch.ones(want.shape[:2], dtype=torch.bool, device=want.device) if steps is None else steps
    ratio = torch.where(there[:, :, None, None] & (size > 0), want.abs() / size.clamp(min=1e-300), 0)
    most = ratio.amax((1, 3), keepdim=True)
    half = torch.finfo(got.dtype).eps / 2 if got.dtype != torch.float32 else 0.0
    # results below the normal numbers of their type are rounded to its smallest step
    allowed = tol * size * most + half * want.abs() + torch.finfo(got.dtype).tiny
    err = (got.double() - want).abs()[there]
    assert torch.isfinite(got[there]).all(), name
    assert (err <= allowed.expand(want.shape)[there]).all(), f"{name}: {float((err / allowed.expand(want.shape)[there]).max()):.3g} times the tolerance"


def wide(d, n):
    """(b, l, hk) -> (b, l, hv)"""
    return n.repeat_interleave(d["v"].shape[2] // n.shape[2], 2)


@pytest.mark.parametrize("size", [1e-12, 1e3, 1e6, 1e9, 1e12, 1e30])
@pytest.mark.parametrize("l,hk,hv,dk,dv", [(70, 2, 4, 64, 48), (200, 1, 1, 128, 100), (1100, 1, 2, 72, 64)])
def test_a_query_of_another_size(size, l, hk, hv, dk, dv):
    d = make(61, 1, l, hk, hv, dk, dv)
    for t in (0, 21, l - 1):
        d["q"][:, t, 0] *= size
    d["q"][:, 40, 0, 1:] = 0
    d["q"][:, 40, 0, 0] = size                                   # a single element
    go = go_like(d)
    (o, s, g), (o64, s64, g64) = run(d, go if size < 1e20 else None), truth(d, go if size < 1e20 else None)
    by_rows("o", o, o64, wide(d, d["q"].double().norm(dim=-1)), FWD)
    assert float((s - s64).abs().max()) <= FWD * float(s64.abs().max())
    if g is None:
        return
    by_rows("grad q", g["q"], g64["q"], torch.ones_like(g["q"][..., 0]), BWD)
    # the other gradients are sums over later queries: chunk by chunk within BWD of the chunk's largest
    for n in ("k", "v", "g", "beta"):
        for c in range(0, l, CHUNK):
            a, b = g[n][:, c:c + CHUNK].double(), g64[n][:, c:c + CHUNK]
            assert float((a - b).abs().max()) <= BWD * float(b.abs().max()), (n, c)
    assert aussm_b200.device_status() == 0


@pytest.mark.parametrize("dtype,size", [(torch.bfloat16, 1e9), (torch.float16, 6e4)])
def test_a_query_of_another_size_in_16_bits(dtype, size):
    d = make(62, 2, 150, 2, 2, 64, 64, dtype)
    d["q"][0, 90, 1] *= size
    o, _, _ = run(d)
    by_rows("o", o, truth(d)[0], wide(d, d["q"].double().norm(dim=-1)), FWD)


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_an_infinite_query_stays_with_its_step(bad, dtype):
    d = make(63, 1, 150, 1, 2, 64, 64, dtype)
    clean = {n: t.clone() for n, t in d.items()}
    d["q"][0, 77, 0, 3] = bad
    go = go_like(d)
    (o, s, g), (o64, s64, g64) = run(d, go), truth(clean, go)
    others = torch.ones(1, 150, dtype=torch.bool, device="cuda")
    others[0, 77] = False
    assert not torch.isfinite(o[0, 77]).any()
    by_rows("o", o, o64, wide(d, clean["q"].double().norm(dim=-1)), FWD, others)
    assert float((s - s64).abs().max()) <= FWD * float(s64.abs().max())
    by_rows("grad q", g["q"], g64["q"], torch.ones_like(g["q"][..., 0]), BWD)      # none of them sees a query
    for n in ("k", "v", "g", "beta"):                            # the next chunk does not see it, this one may not hide it
        a, b, half = g[n].double(), g64[n], torch.finfo(g[n].dtype).eps / 2
        most = float(b.abs().max())
        assert ((a - b).abs()[:, 128:] <= BWD * most + half * b.abs()[:, 128:]).all(), n
        assert (((a - b).abs() <= BWD * most + half * b.abs()) | ~torch.isfinite(a))[:, 78:].all(), n
    assert not torch.isfinite(g["v"][0, :78]).any() and not torch.isfinite(g["k"][0, :78]).any()


@pytest.mark.parametrize("bad", [math.inf, math.nan, 1e9])
def test_an_outlying_gradient_stays_with_its_step(bad):
    """One step of the gradient of o: the other steps' dq do not see it."""
    d = make(64, 1, 150, 1, 1, 64, 80)
    go = go_like(d)
    clean = go.clone()
    if math.isfinite(bad):
        go[0, 30] *= bad
    else:
        go[0, 30, 0, 5] = bad
    _, _, g = run(d, go)
    _, _, g64 = truth(d, clean)
    others = torch.ones(1, 150, dtype=torch.bool, device="cuda")
    others[0, 30] = False
    by_rows("grad q", g["q"], g64["q"], torch.ones_like(g["q"][..., 0]), BWD, others)
    if math.isfinite(bad):
        by_rows("grad q", g["q"] / bad, g64["q"], torch.ones_like(g["q"][..., 0]), BWD, ~others)
    for n in ("k", "v", "g", "beta"):
        assert float((g[n][:, 64:] - g64[n][:, 64:]).abs().max()) <= BWD * float(g64[n].abs().max()), n


@pytest.mark.parametrize("l,hk,hv,dk,dv", [(150, 1, 2, 64, 64), (1100, 1, 1, 128, 128), (40, 1, 1, 16, 130)])
@pytest.mark.parametrize("size", [1e4, 1e9, 1e18])
def test_padded_keys_of_any_size(size, l, hk, hv, dk, dv):
    """g = beta = 0 leaves the state alone whatever k and v hold, and the gradients of the other steps with it."""
    d = make(65, 2, l, hk, hv, dk, dv)
    pad = slice(20, 33)
    for n in ("g", "beta"):
        d[n][0, pad] = 0
    d["k"][0, pad] *= size
    d["v"][0, pad] *= size
    go = go_like(d)
    (o, s, g), (o64, s64, g64) = run(d, go), truth(d, go)
    by_rows("o", o, o64, wide(d, d["q"].double().norm(dim=-1)), FWD)
    assert float((s - s64).abs().max()) <= FWD * float(s64.abs().max())
    real = torch.ones(2, l, dtype=torch.bool, device="cuda")
    real[0, pad] = False
    for n in NAMES:
        a, b = g[n].double(), g64[n]
        if n != "state":
            assert (a[~real] == 0).all() or n in ("q", "g", "beta"), n
            a, b = a[real], b[real]
        assert float((a - b).abs().max()) <= BWD * float(b.abs().max()), n
    # of a padded step itself: beta's gradient is a product of its key and value, as large as they are
    a, b = g["beta"][~real].double(), g64["beta"][~real]
    assert float((a - b).abs().max()) <= BWD * float(b.abs().max())


@pytest.mark.parametrize("l,hk,hv,dk,dv", [(150, 1, 2, 64, 64), (1100, 1, 1, 128, 128)])
def test_keys_of_all_sizes(l, hk, hv, dk, dv):
    """With keys times s, values times s and step sizes over s^2 the rule is the same: dk and dv shrink by s, dbeta grows by s^2.
    Powers of two are exact, so the results are held to the recurrence of the unit keys; what is left of a row behind the
    division is 1..2 at its largest element, 1 to 4 times a unit key here: four times the usual bounds for the neighbours."""
    d = make(69, 1, l, hk, hv, dk, dv)
    gen = torch.Generator().manual_seed(3)
    s = 2.0 ** torch.randint(3, 30, (1, l, hk, 1), generator=gen).cuda()
    s[:, ::3] = 1.0
    big = dict(d, k=d["k"] * s, v=d["v"] * wide(d, s), beta=d["beta"] / wide(d, s)[..., 0] ** 2)
    go = go_like(d)
    (o, last, g), (o64, s64, g64) = run(big, go), truth(d, go)
    g = dict(g, k=g["k"] * s, v=g["v"] * wide(d, s), beta=g["beta"] / wide(d, s)[..., 0] ** 2)
    by_rows("o", o, o64, wide(d, d["q"].double().norm(dim=-1)), 4 * FWD)
    assert float((last - s64).abs().max()) <= 4 * FWD * float(s64.abs().max())
    for n in NAMES:
        assert float((g[n] - g64[n]).abs().max()) <= 4 * BWD * float(g64[n].abs().max()), n


@pytest.mark.parametrize("bad", [math.inf, math.nan])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_padded_steps_of_anything(bad, dtype):
    """Unwritten memory in the keys and values of padded steps, in sequences and in single steps."""
    d = make(66, 2, 150, 1, 2, 64, 64, dtype)
    clean = {n: t.clone() for n, t in d.items()}
    pad = torch.zeros(2, 150, dtype=torch.bool, device="cuda")
    pad[0, 100:], pad[1, :7], pad[1, 70] = True, True, True
    for x in (d, clean):
        x["g"][pad] = 0
        x["beta"][pad] = 0
    d["k"][pad], d["v"][pad] = bad, bad
    clean["k"][pad], clean["v"][pad] = 0, 0
    go = go_like(d)
    go[pad] = 0
    (o, s, g), (o64, s64, g64) = run(d, go), truth(clean, go)
    by_rows("o", o, o64, wide(d, d["q"].double().norm(dim=-1)), FWD)
    assert float((s - s64).abs().max()) <= FWD * float(s64.abs().max())
    for n in NAMES[:5]:
        a, b = g[n][~pad].double(), g64[n][~pad]
        assert ((a - b).abs() <= BWD * float(b.abs().max()) + torch.finfo(g[n].dtype).eps / 2 * b.abs()).all(), n
    assert float((g["state"] - g64["state"]).abs().max()) <= BWD * float(g64["state"].abs().max())
    assert (g["k"][pad] == 0).all() and (g["v"][pad] == 0).all()
    state = clean["state"].clone()
    for t in range(100, 104):
        y = gated_delta_step(*(d[n][:1, t:t + 1] for n in NAMES[:5]), state[:1])
        assert torch.isfinite(y).all()
    assert torch.equal(state, clean["state"])


@pytest.mark.parametrize("size", [1e6, 1e12])
def test_a_large_value_shows_in_its_column_and_chunk(size):
    d = make(67, 1, 200, 1, 1, 64, 64)
    d["v"][0, 90, 0, 11] *= size
    put = float(d["beta"][0, 90, 0] * d["v"][0, 90, 0, 11].abs())       # into the state; sqrt(dk) less into an output
    (o, s, _), (o64, s64, _) = run(d), truth(d)
    err = (o - o64).abs()[0, :, 0]
    rest = [c for c in range(64) if c != 11]
    assert float(err[:, rest].max()) <= FWD * float(o64[..., rest].abs().max())
    assert float(err[:64, 11].max()) <= FWD * float(o64[:, :64, 0, 11].abs().max())
    # The state behind the chunk is e^G S + sum_j Kt_j V'_j, whose terms are rounded by 2^-21 of the largest |Kt_j| (at most a
    # unit key) times the largest |V'_j| (the value put in): a decay that follows the value in its chunk does not shrink that
    # error.  Here it shrinks the result to 6e-14 of the value, so the bound is on the value, not on what is left of it.
    assert float(err[64:, 11].max()) <= FWD * put / 8
    assert float((s - s64).abs()[..., 11].max()) <= FWD * put


@pytest.mark.parametrize("size", [1e3, 1e6, 1e9, 1e12])
def test_a_large_value_before_its_step(size):
    """Steps before it in its chunk share its scale: their parts are off by 2^-38 of the value at most, each of up to 64 of them
    that a result adds up."""
    d = make(70, 1, 130, 1, 1, 64, 64)
    d["v"][0, 120, 0, 11] *= size
    put = float(d["beta"][0, 120, 0] * d["v"][0, 120, 0, 11].abs())
    o, _, _ = run(d)
    o64, _, _ = truth(d)
    before = o64[0, 64:120, 0, 11]
    assert float((o[0, 64:120, 0, 11] - before).abs().max()) <= 64 * 2 ** -38 * put + FWD * float(before.abs().max())


@pytest.mark.parametrize("bad", [math.inf, math.nan])
@pytest.mark.parametrize("name", ["v", "k", "beta", "g"])
def test_what_is_not_finite_is_never_hidden(name, bad):
    """From its step on nothing that depends on it is finite; before it, a step of its chunk is right or not finite, and a
    step of an earlier chunk is right."""
    d = make(68, 1, 200, 1, 1, 64, 64)
    clean = truth(d)[0]
    d[name][(0, 90, 0, 5)[:d[name].dim()]] = bad
    o, s, _ = run(d)
    err = (o - clean).abs()
    tol = FWD * float(clean.abs().max())
    assert (err[:, :64] <= tol).all()
    assert ((err <= tol) | ~torch.isfinite(o))[:, :90].all()
    cols = [5] if name == "v" else list(range(64))
    assert not torch.isfinite(o[0, 91:, 0, cols]).any() and not torch.isfinite(s[0, 0, :, cols]).all(0).any()
    if name == "v":
        rest = [c for c in range(64) if c != 5]
        assert (err[..., rest] <= tol).all()
