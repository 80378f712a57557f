"""Gated delta rule against the token-by-token recurrence in float64.

Tolerances.  The kernels' operands carry 22 significant bits or more and all sums 24, so a product's error is at most
2^-21 of the sum of its terms' magnitudes, which exceeds the largest element of the result by sqrt(128) at most where the
terms are as good as independent.  An output is the last of about 8 products in a row (gradients: 16):
8 * 2^-21 * 11.3 = 4.3e-5 of the largest element, twice that for gradients.  Outputs in 16 bits are off by half a step of
their type more.
"""
import math

import pytest
import torch

import aussm_b200
from aussm_b200.delta import gated_delta_rule, gated_delta_step
from oracle.delta import gated_delta_ref

pytestmark = pytest.mark.gpu
NAMES = ["q", "k", "v", "g", "beta", "state"]
FWD, BWD = 5e-5, 1e-4


def make(seed, b, l, hk, hv, dk, dv, dtype=torch.float32, rate=1.0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)
    unit = lambda x: torch.nn.functional.normalize(x, dim=-1)
    d = dict(q=unit(r(b, l, hk, dk)).to(dtype), k=unit(r(b, l, hk, dk)).to(dtype), v=r(b, l, hv, dv).to(dtype),
             g=-rate * torch.nn.functional.softplus(r(b, l, hv)), beta=2 * torch.sigmoid(r(b, l, hv)),
             state=r(b, hv, dk, dv) / math.sqrt(dk))
    return {n: x.cuda() for n, x in d.items()}


def close(name, got, truth, tol):
    truth, half = truth.double(), torch.finfo(got.dtype).eps / 2 if got.dtype != torch.float32 else 0.0
    allowed = half * truth.abs() + tol * float(truth.abs().max()) + 1e-30
    err = (got.double() - truth).abs()
    assert torch.isfinite(got).all(), name
    assert (err <= allowed).all(), f"{name}: {float((err / allowed).max()):.3g} times the tolerance"


def both(d, go_seed=7, scale=None, final=True, state=True):
    """Outputs and gradients of the kernels and of the recurrence in float64, for the same inputs."""
    gen = torch.Generator(device="cuda").manual_seed(go_seed)
    res = []
    for dtype in (None, torch.float64):
        x = {n: t.detach().clone() if dtype is None else t.detach().to(dtype) for n, t in d.items()}
        x = {n: t.requires_grad_() for n, t in x.items() if state or n != "state"}
        fn = gated_delta_rule if dtype is None else gated_delta_ref
        kw = dict(return_final_state=True) if dtype is None else {}
        o, s = fn(x["q"], x["k"], x["v"], x["g"], x["beta"], scale=scale, initial_state=x.get("state"), **kw)
        if dtype is None:
            go = torch.randn(o.shape, device="cuda", generator=gen).to(o.dtype)
            gs = torch.randn(s.shape, device="cuda", generator=gen)
        outs, grads = ([o, s], [go, gs]) if final else ([o], [go])
        grads = torch.autograd.grad(outs, list(x.values()), [t.to(y.dtype) for t, y in zip(grads, outs)])
        res.append(({"o": o.detach(), "s": s.detach()}, dict(zip(x, grads))))
    return res


def compare(res):
    (got, ggot), (truth, gtruth) = res
    for n in got:
        close(n, got[n], truth[n], FWD)
    for n in ggot:
        assert ggot[n].dtype == (got["o"].dtype if n in "qkv" else torch.float32)
        close("grad " + n, ggot[n], gtruth[n], BWD)
    assert aussm_b200.device_status() == 0


@pytest.mark.parametrize("l", [1, 2, 17, 63, 64, 65, 128, 150])
def test_lengths(l):
    compare(both(make(l, 2, l, 2, 2, 32, 32)))


@pytest.mark.parametrize("dk,dv", [(1, 1), (5, 7), (16, 16), (64, 64), (72, 100), (128, 128), (33, 129), (128, 256), (96, 200)])
def test_widths(dk, dv):
    compare(both(make(dk + dv, 1, 130, 1, 2, dk, dv)))


@pytest.mark.parametrize("hk,hv", [(1, 1), (3, 3), (2, 4), (1, 5)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_heads_and_types(hk, hv, dtype):
    compare(both(make(hk + hv, 2, 100, hk, hv, 64, 48, dtype)))


@pytest.mark.parametrize("final,state", [(False, True), (False, False), (True, False)])
def test_without_states(final, state):
    compare(both(make(3, 2, 90, 2, 2, 64, 64), final=final, state=state))


@pytest.mark.parametrize("rate", [1e-3, 0.1, 10.0, 60.0])
def test_decays(rate):
    compare(both(make(5, 1, 200, 2, 2, 64, 64, rate=rate)))


def test_forgetting_and_padding():
    """g = -inf drops the state, also twice in a chunk; steps with g = beta = 0 change nothing, whatever q, k, v hold."""
    d = make(9, 2, 150, 2, 2, 64, 64)
    for t in (5, 6, 70, 149):
        d["g"][:, t] = -math.inf
    d["g"][0, 100:140] = 0.0
    d["beta"][0, 100:140] = 0.0
    x = dict(d)
    o, s = gated_delta_rule(x["q"], x["k"], x["v"], x["g"], x["beta"], initial_state=x["state"], return_final_state=True)
    y = {n: t.double() for n, t in d.items()}
    o64, s64 = gated_delta_ref(y["q"], y["k"], y["v"], y["g"], y["beta"], initial_state=y["state"])
    close("o", o, o64, FWD)
    close("s", s, s64, FWD)
    finite = dict(d, g=d["g"].clamp(min=-300.0))       # -inf itself has no gradient in the recurrence (0 * inf)
    compare(both(finite))


def test_whole_batch_entry_padded():
    d = make(11, 3, 80, 1, 1, 32, 32)
    d["g"][1] = 0.0
    d["beta"][1] = 0.0
    o, s = gated_delta_rule(*(d[n] for n in NAMES[:5]), initial_state=d["state"], return_final_state=True)
    assert torch.equal(s[1], d["state"][1])
    compare(both(d))


def test_scale_and_large_values():
    d = make(13, 1, 100, 1, 1, 64, 64)
    d["v"] *= 1e6
    d["state"] *= 1e6
    compare(both(d, scale=3.0))
    d["v"] *= 1e-18
    d["state"] *= 1e-18
    compare(both(d, scale=1e-3))


@pytest.mark.parametrize("size", [1e36, 1e-30])
def test_ends_of_the_range(size):
    """Values and states near the ends of float32 (the gradients of q, k, g and beta, products of two of them, do not fit)."""
    d = make(14, 1, 100, 1, 1, 64, 64)
    d["v"] *= size
    d["state"] *= size
    o, s = gated_delta_rule(*(d[n] for n in NAMES[:5]), initial_state=d["state"], return_final_state=True)
    y = {n: t.double() for n, t in d.items()}
    o64, s64 = gated_delta_ref(*(y[n] for n in NAMES[:5]), initial_state=y["state"])
    for got, truth in ((o, o64), (s, s64)):
        close("scaled", (got.double() / size).float(), truth / size, FWD)


def test_a_nan_stays_in_its_value_column():
    d = make(17, 1, 130, 1, 1, 64, 64)
    clean, cs = gated_delta_rule(*(d[n] for n in NAMES[:5]), return_final_state=True)
    d["v"][0, 3, 0, 9] = math.nan
    o, s = gated_delta_rule(*(d[n] for n in NAMES[:5]), return_final_state=True)
    rest = [c for c in range(64) if c != 9]
    assert torch.equal(o[..., rest], clean[..., rest]) and torch.equal(s[..., rest], cs[..., rest])
    assert torch.isnan(o[0, 4:, 0, 9]).all()


def test_strides():
    """Views: heads in front of steps, slices of one fused tensor that start anywhere, expanded heads and batches."""
    b, l, h, w = 2, 77, 2, 36
    d = make(19, b, l, h, h, w, w)
    ref = gated_delta_rule(*(d[n] for n in NAMES[:5]))
    front = {n: d[n].transpose(1, 2).contiguous().transpose(1, 2) for n in ("q", "k", "v")}
    assert torch.equal(gated_delta_rule(front["q"], front["k"], front["v"], d["g"], d["beta"]), ref)
    fused = torch.zeros(b, l, h, 3 * w + 1, device="cuda")
    for i, n in enumerate(("q", "k", "v")):
        fused[..., 1 + i * w:1 + (i + 1) * w] = d[n]
    views = [fused[..., 1 + i * w:1 + (i + 1) * w] for i in range(3)]
    assert torch.equal(gated_delta_rule(*views, d["g"], d["beta"]), ref)
    last = [d[n].transpose(1, 3).contiguous().transpose(1, 3) for n in ("q", "k", "v")]      # steps contiguous
    assert torch.equal(gated_delta_rule(*last, d["g"], d["beta"]), ref)
    # one key for all heads and one batch of values for all entries: the gradients of expanded inputs add up
    k1, v1 = d["k"][:, :, :1].clone().requires_grad_(), d["v"][:1].clone().requires_grad_()
    o = gated_delta_rule(d["q"], k1.expand(b, l, h, w), v1.expand(b, l, h, w), d["g"], d["beta"])
    got = torch.autograd.grad(o, [k1, v1], torch.ones_like(o))
    k2, v2 = k1.detach().double().requires_grad_(), v1.detach().double().requires_grad_()
    o2, _ = gated_delta_ref(d["q"].double(), k2.expand(b, l, h, w), v2.expand(b, l, h, w), d["g"].double(), d["beta"].double())
    truth = torch.autograd.grad(o2, [k2, v2], torch.ones_like(o2))
    close("o", o.detach(), o2.detach(), FWD)
    for n, a, t in zip("kv", got, truth):
        close("grad " + n, a, t, BWD)
    # a gradient that is expanded itself
    q = d["q"].clone().requires_grad_()
    o = gated_delta_rule(q, d["k"], d["v"], d["g"], d["beta"])
    one, = torch.autograd.grad(o.sum(), q, retain_graph=True)
    two, = torch.autograd.grad(o, q, torch.ones_like(o))
    assert torch.equal(one, two)


def test_pieces_of_a_sequence_and_determinism():
    """A sequence in pieces through the final state is the sequence; the same call twice is the same bits."""
    d = make(23, 2, 300, 2, 4, 64, 80)
    o, s = gated_delta_rule(*(d[n] for n in NAMES[:5]), initial_state=d["state"], return_final_state=True)
    state, outs = d["state"], []
    for a, z in ((0, 1), (1, 100), (100, 228), (228, 300)):
        y, state = gated_delta_rule(*(d[n][:, a:z] for n in NAMES[:5]), initial_state=state, return_final_state=True)
        outs.append(y)
    close("o", torch.cat(outs, 1), o, FWD)
    close("s", state, s, FWD)
    first, second = both(d), both(d)
    for a, z in zip(first[0], second[0]):
        assert all(torch.equal(a[n], z[n]) for n in a)


def test_gradient_against_differences():
    d = make(29, 1, 70, 1, 1, 16, 16)
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = {n: t.clone().requires_grad_() for n, t in d.items()}
    run = lambda y: gated_delta_rule(y["q"], y["k"], y["v"], y["g"], y["beta"], initial_state=y["state"])
    w = torch.randn(1, 70, 1, 16, device="cuda", generator=gen)
    grads = dict(zip(x, torch.autograd.grad((run(x) * w).sum(), list(x.values()))))
    for n in x:
        way = torch.randn(d[n].shape, device="cuda", generator=gen)
        h = 1e-2
        up, down = (run({**d, n: d[n] + s * h * way}).double() for s in (1, -1))
        slope = float(((up - down) * w.double()).sum() / (2 * h))
        told = float((grads[n].double() * way.double()).sum())
        # the differences' own error: third derivatives times h^2, and rounding of the sums over h
        size = float((grads[n].double().abs() * way.double().abs()).sum())
        assert abs(slope - told) <= 5e-3 * size + 1e-3, n


@pytest.mark.parametrize("t", [1, 2, 5])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dk,dv,hk,hv", [(128, 128, 2, 4), (64, 64, 1, 1), (7, 5, 2, 2), (100, 130, 1, 3), (128, 256, 1, 1)])
def test_step(t, dtype, dk, dv, hk, hv):
    d = make(t + dk, 3, t, hk, hv, dk, dv, dtype)
    y = {n: x.double() for n, x in d.items()}
    o64, s64 = gated_delta_ref(y["q"], y["k"], y["v"], y["g"], y["beta"], initial_state=y["state"])
    before, new = d["state"].clone(), torch.empty_like(d["state"])
    o = gated_delta_step(*(d[n] for n in NAMES), new_state=new)
    assert torch.equal(d["state"], before)
    close("o", o, o64, FWD)
    close("s", new, s64, FWD)
    o2 = gated_delta_step(*(d[n] for n in NAMES))                   # in place
    assert torch.equal(o, o2) and torch.equal(d["state"], new)


def test_step_continues_the_rule():
    d = make(31, 2, 70, 2, 2, 64, 64, torch.bfloat16)
    o, s = gated_delta_rule(*(d[n] for n in NAMES[:5]), return_final_state=True)
    _, state = gated_delta_rule(*(d[n][:, :60] for n in NAMES[:5]), return_final_state=True)
    for t in range(60, 70):
        y = gated_delta_step(*(d[n][:, t:t + 1] for n in NAMES[:5]), state)
    close("s", state, s, FWD)
    close("o", y, o[:, 69:70].double(), 2 ** -8 + FWD)


def test_step_on_an_unaligned_state():
    d = make(37, 1, 1, 1, 1, 64, 64)
    room = torch.zeros(64 * 64 + 1, device="cuda")
    odd = room[1:].view(1, 1, 64, 64)
    odd.copy_(d["state"])
    o = gated_delta_step(*(d[n] for n in NAMES[:5]), odd)
    o2 = gated_delta_step(*(d[n] for n in NAMES))
    close("o", o, o2, FWD)
    close("s", odd, d["state"], FWD)


def test_empty():
    d = make(41, 2, 3, 1, 1, 8, 8)
    z = {n: d[n][:, :0].clone().requires_grad_() for n in NAMES[:5]}
    state = d["state"].clone().requires_grad_()
    o, s = gated_delta_rule(*z.values(), initial_state=state, return_final_state=True)
    assert o.shape == (2, 0, 1, 8) and torch.equal(s, state)
    got = torch.autograd.grad(s, [state, z["q"]], torch.ones_like(s), allow_unused=True)
    assert torch.equal(got[0], torch.ones_like(s)) and got[1].shape == z["q"].shape
    assert gated_delta_step(*(d[n][:, :0] for n in NAMES[:5]), d["state"]).shape == (2, 0, 1, 8)
    none = [d[n][:0] for n in NAMES]
    assert gated_delta_rule(*none[:5]).shape == (0, 3, 1, 8) and gated_delta_step(*none).shape == (0, 3, 1, 8)


def test_refusals():
    d = make(43, 2, 3, 2, 2, 8, 8)
    a = [d[n] for n in NAMES[:5]]
    swap = lambda i, x: a[:i] + [x] + a[i + 1:]
    bad = [swap(0, a[0].cpu()), swap(0, a[0].double()), swap(1, a[1].half()), swap(1, a[1][:, :2]), swap(2, a[2][:, :, :1]),
           swap(3, a[3].double()), swap(4, a[4][:1]), swap(3, a[3].cpu()), swap(0, a[0][0]), swap(2, a[2].cpu()),
           [torch.zeros(1, 2, 1, 129, device="cuda")] * 2 + [torch.zeros(1, 2, 1, 8, device="cuda")] + [torch.zeros(1, 2, 1, device="cuda")] * 2,
           [torch.zeros(1, 2, 1, 8, device="cuda")] * 2 + [torch.zeros(1, 2, 1, 257, device="cuda")] + [torch.zeros(1, 2, 1, device="cuda")] * 2]
    for args in bad:
        with pytest.raises(RuntimeError):
            gated_delta_rule(*args)
    with pytest.raises(RuntimeError):
        gated_delta_rule(*a, initial_state=d["state"][:1])
    with pytest.raises(RuntimeError):
        gated_delta_rule(*a, initial_state=d["state"].double())
    for state, new in ((d["state"].transpose(2, 3), None), (d["state"].half(), None), (d["state"], d["state"].transpose(2, 3)),
                       (d["state"].cpu(), None), (d["state"], d["state"][:1])):
        with pytest.raises(RuntimeError):
            gated_delta_step(*a, state, new_state=new)
    room = torch.zeros(d["state"].numel() + 4, device="cuda")
    with pytest.raises(RuntimeError, match="overlaps"):
        gated_delta_step(*a, room[:-4].view_as(d["state"]), new_state=room[4:].view_as(d["state"]))
    with pytest.raises(RuntimeError, match="not differentiable"):
        gated_delta_step(a[0].clone().requires_grad_(), *a[1:], d["state"])
    q = a[0].clone().requires_grad_()
    first, = torch.autograd.grad(gated_delta_rule(q, *a[1:]).sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first.sum(), q)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda x: gated_delta_rule(x, *a[1:]).sum())(a[0])
    lib, p = aussm_b200._lib.load(), aussm_b200._lib.DeltaProblem(1, 1, 2, 3, 8, 8)
    assert lib.aussm_b200_delta_fwd(p, *([None] * 9), 0, None, 0, None) != 0
    assert lib.aussm_b200_delta_keep_bytes(p) == 0
    p = aussm_b200._lib.DeltaProblem(1, 1, 1, 1, 8, 8)
    ptr = a[0].data_ptr()
    assert lib.aussm_b200_delta_fwd(p, *([ptr] * 5), None, ptr, None, None, 0, None, 0, None) == -2      # no workspace


def test_streams_and_graph_replay():
    """On a stream of its own; captured and replayed on new values, forward, backward and step, while an eager graph of
    the same leaves is alive."""
    d = make(47, 2, 130, 1, 2, 64, 64)
    want = both(d, final=False)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x = {n: t.clone().requires_grad_() for n, t in d.items()}
        alive = gated_delta_rule(*(x[n] for n in NAMES[:5]), initial_state=x["state"])
        go = torch.randn(alive.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(7))
        assert torch.equal(alive, want[0]["o"])
        torch.autograd.grad(gated_delta_rule(*(x[n] for n in NAMES[:5]), initial_state=x["state"]), list(x.values()), go)
    side.synchronize()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        o = gated_delta_rule(*(x[n] for n in NAMES[:5]), initial_state=x["state"])
        grads = torch.autograd.grad(o, list(x.values()), go)
        with torch.no_grad():
            new = torch.empty_like(x["state"])
            y = gated_delta_step(*(x[n][:, :1] for n in NAMES[:5]), x["state"], new_state=new)
    for seed in (47, 48):
        e = make(seed, 2, 130, 1, 2, 64, 64)
        with torch.no_grad():
            for n in NAMES:
                x[n].copy_(e[n])
        graph.replay()
        torch.cuda.synchronize()
        ref = both(e, final=False)[0]
        assert torch.equal(o, ref[0]["o"])
        for n, gr in zip(x, grads):
            assert torch.equal(gr, ref[1][n]), n
        assert torch.equal(y, gated_delta_step(*(e[n][:, :1] for n in NAMES[:5]), e["state"]))
        assert torch.equal(new, e["state"])
    with pytest.raises(RuntimeError, match="inplace"):      # the eager graph's inputs are gone, and torch says so
        torch.autograd.grad(alive.sum(), x["g"])


@pytest.mark.parametrize("l,heads,dk,dv,rate", [(800, 1, 128, 128, 0.01), (1111, 3, 64, 64, 1e-3), (2500, 2, 72, 100, 0.1), (1030, 1, 128, 200, 1.0), (1400, 1, 70, 33, 0.02)])
def test_few_heads_in_segments(l, heads, dk, dv, rate):
    """Long sequences of few heads are cut along time: lengths that fill no segment, states that live through all of it."""
    compare(both(make(l, 1, l, heads, heads, dk, dv, rate=rate)))


@pytest.mark.parametrize("rotary_dim", [0, 32])
def test_block(rotary_dim):
    """The block's operators together, as a model uses them: whole sequences against single tokens, and gradients against
    the same block in float64 with the recurrence in the operators' place."""
    from aussm_b200 import models
    from oracle.delta import norm_rotate_ref
    torch.manual_seed(3)
    block = models.GatedDeltaBlock(128, n_heads=2, rotary_dim=rotary_dim).cuda()
    x = torch.randn(2, 150, 128, device="cuda", requires_grad=True)
    y = block(x)
    gy = torch.randn_like(y)
    names, params = zip(*block.named_parameters())
    grads = torch.autograd.grad(y, (x, *params), gy)
    cache = block.init_cache(2, device="cuda")
    steps = torch.cat([block.step(x[:, t:t + 1].detach(), cache) for t in range(150)], 1)

    def rule(q, k, v, g, beta, **kw):
        return gated_delta_ref(q, k, v, g, beta)[0]

    def rotate(q, k, frequencies=None, positions=None, **kw):
        return tuple(norm_rotate_ref(t, frequencies, positions, **kw) for t in (q, k))

    class Wide(torch.nn.Module):             # float64: the block's gate is cast to float32 by design, so it is restated
        def forward(self, x):
            b, l, d = x.shape
            xs, z = block.in_proj(x).split([3 * d, d], dim=-1)
            conv = models._causal_depthwise_conv(block.conv1d, xs)
            q, k, v = torch.nn.functional.silu(conv).reshape(b, l, 3, 2, 64).unbind(2)
            f = None if not rotary_dim else block._frequencies(x.device)
            q, k = rotate(q, k, f, norm="l2")
            a, beta = block.gate_proj(x).split([2, 2], dim=-1)
            g = -torch.exp(block.A_log) * torch.nn.functional.softplus(a + block.dt_bias)
            o = rule(q, k, v, g, torch.sigmoid(beta))
            o = o * torch.rsqrt(o.square().mean(-1, keepdim=True) + block.norm.eps) * block.norm.weight
            return block.out_proj((o * torch.nn.functional.silu(z.reshape(b, l, 2, 64))).reshape(b, l, d))

    block.double()
    x64 = x.detach().double().requires_grad_()
    y64 = Wide()(x64)
    truth = torch.autograd.grad(y64, (x64, *block.parameters()), gy.double())
    # the operators' tolerance, and as much again for the dozen float32 operations and products around them
    close("y", y.detach(), y64.detach(), 4 * FWD)
    close("steps", steps, y64.detach(), 4 * FWD)
    for n, a, t in zip(("x", *names), grads, truth):
        close("grad " + n, a, t, 4 * BWD)


def test_models_with_delta_layers():
    from aussm_b200 import models
    from aussm_b200.train import GraphedTrainStep
    torch.manual_seed(5)
    net = models.SSMTS(d_model=64, input_dim=3, output_dim=2, layers="a|g|m").cuda()
    x, y = torch.randn(2, 96, 3, device="cuda"), torch.randn(2, 96, 2, device="cuda")
    loss = (net(x) - y).square().mean()
    grads = torch.autograd.grad(loss, list(net.parameters()))
    assert all(torch.isfinite(g).all() for g in grads)
    del loss, grads
    opt = torch.optim.AdamW(net.parameters(), lr=1e-3, capturable=True)
    step = GraphedTrainStep(net, opt, x, y, lambda o, t: (o - t).square().mean())
    assert torch.isfinite(step.step()) and torch.isfinite(step.step(x + 1, y))
    ids = torch.randint(0, 50, (2, 70), device="cuda")
    clf = models.SSMSequenceClassifier(d_model=64, vocab_size=50, output_dim=3, layers="g|a").cuda()
    out = clf(ids, torch.tensor([70, 33], device="cuda"))
    assert out.shape == (2, 3) and torch.isfinite(out).all()
    assert aussm_b200.device_status() == 0


def test_status_word_is_polled(monkeypatch):
    seen = []
    monkeypatch.setattr("aussm_b200.ops.check_device_status", True)
    monkeypatch.setattr("aussm_b200.ops.device_status", lambda device=None: seen.append(device) or 0)
    d = make(1, 1, 70, 1, 1, 8, 8)
    q = d["q"].requires_grad_()
    gated_delta_rule(q, d["k"], d["v"], d["g"], d["beta"]).sum().backward()
    assert seen == [q.device] * 2
    monkeypatch.setattr("aussm_b200.ops.device_status", lambda device=None: 1)
    with torch.no_grad(), pytest.raises(RuntimeError, match="gave up"):
        gated_delta_rule(q, d["k"], d["v"], d["g"], d["beta"])


def test_step_counts_as_a_change_in_place():
    d = make(2, 2, 1, 1, 2, 16, 16)
    w = torch.ones((), device="cuda", requires_grad=True)
    kept = (w * d["state"]).sum()                       # saves the state for w's gradient
    gated_delta_step(*(d[n] for n in NAMES))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        kept.backward()
    with torch.inference_mode():                        # states made there have no count
        x = {n: t.clone() for n, t in d.items()}
        other = gated_delta_step(*(x[n] for n in NAMES))
    assert torch.equal(other, gated_delta_step(*(d[n] for n in NAMES)))


def test_signs_kept_in_a_flag():
    """Parts of conjugate tensors carry their sign in a flag, as inputs and as gradients."""
    d = make(3, 2, 70, 1, 2, 16, 8)
    flagged = lambda t: torch.complex(torch.zeros_like(t), -t).conj().imag
    x = {n: flagged(t) for n, t in d.items()}
    assert all(t.is_neg() for t in x.values())
    a, b = gated_delta_rule(*(d[n] for n in NAMES[:5]), initial_state=d["state"]), gated_delta_rule(
        *(x[n] for n in NAMES[:5]), initial_state=x["state"])
    assert torch.equal(a, b)
    with pytest.raises(RuntimeError, match="takes the result"):
        gated_delta_step(*(x[n][:, :1] for n in NAMES[:5]), x["state"])
    new = torch.empty_like(d["state"])
    assert torch.equal(gated_delta_step(*(x[n][:, :1] for n in NAMES[:5]), x["state"], new_state=new),
                       gated_delta_step(*(d[n][:, :1] for n in NAMES[:5]), d["state"].clone()))
    v = d["v"].requires_grad_()
    o, s = gated_delta_rule(d["q"], d["k"], v, d["g"], d["beta"], return_final_state=True)
    go, gs = torch.randn_like(o), torch.randn_like(s)
    assert torch.equal(torch.autograd.grad([o, s], v, [go, gs], retain_graph=True)[0],
                       torch.autograd.grad([o, s], v, [flagged(go), flagged(gs)])[0])


@pytest.mark.parametrize("rotary_dim", [0, 32])
def test_block_captured_step_and_prompt(rotary_dim):
    """A prompt in one piece, then single tokens from a captured and replayed step, against whole sequences."""
    from aussm_b200 import models
    torch.manual_seed(4)
    block = models.GatedDeltaBlock(128, n_heads=2, rotary_dim=rotary_dim).cuda()
    x = torch.randn(2, 90, 128, device="cuda")
    static = torch.empty(2, 1, 128, device="cuda")
    with torch.no_grad():
        whole = block(x)
        cache = block.init_cache(2, device="cuda")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            block.step(static.zero_(), cache)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = block.step(static, cache)
        for t in cache.values():
            t.zero_()
        got = [block.step(x[:, :70], cache), block.step(x[:, 70:73], cache)]
        for t in range(73, 90):
            static.copy_(x[:, t:t + 1])
            graph.replay()
            got.append(y.clone())
    assert int(cache["position"]) == 90
    # both sides are within the block's tolerance of the exact values
    close("pieces", torch.cat(got, 1), whole, 8 * FWD)
    if rotary_dim:
        fresh = models.GatedDeltaBlock(128, n_heads=2, rotary_dim=rotary_dim).cuda()
        with torch.cuda.graph(torch.cuda.CUDAGraph()), pytest.raises(RuntimeError, match="before it is captured"):
            fresh._frequencies(x.device)


def test_block_in_sixteen_bits():
    """The cache follows the block's type; both ways through the block agree to bfloat16's roundings."""
    from aussm_b200 import models
    torch.manual_seed(6)
    block = models.GatedDeltaBlock(64, n_heads=2, rotary_dim=16).cuda().bfloat16()
    x = torch.randn(2, 30, 64, device="cuda", dtype=torch.bfloat16)
    with torch.no_grad():
        whole, cache = block(x), block.init_cache(2)
        got = torch.cat([block.step(x[:, a:b], cache) for a, b in ((0, 20), (20, 21), (21, 30))], 1)
    assert cache["conv"].dtype == torch.bfloat16 and cache["state"].dtype == torch.float32 and cache["state"].is_cuda
    # In the worst case each of a dozen roundings of 2^-8 stays, for both sides, in the same direction: 24 * 2^-8 of the
    # largest element; a step that took a wrong position, input or state is off by the size of the result.
    assert got.dtype == torch.bfloat16
    assert float((got.float() - whole.float()).abs().max()) <= 24 * 2 ** -8 * float(whole.float().abs().max())


def test_block_under_autocast():
    from aussm_b200 import models
    torch.manual_seed(7)
    block = models.GatedDeltaBlock(64, n_heads=2).cuda()
    x = torch.randn(2, 70, 64, device="cuda")
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = block(x)
        with torch.no_grad():
            cache = block.init_cache(2)
            steps = torch.cat([block.step(x[:, a:b], cache) for a, b in ((0, 40), (40, 41), (41, 70))], 1)
    y.float().square().mean().backward()
    # as in bfloat16 altogether, see above
    assert float((steps.float() - y.detach().float()).abs().max()) <= 24 * 2 ** -8 * float(y.detach().float().abs().max())
    assert torch.isfinite(y).all() and all(torch.isfinite(p.grad).all() for p in block.parameters())
