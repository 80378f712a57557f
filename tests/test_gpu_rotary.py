"""Norm and rotation of queries and keys against plain float64.

Tolerances: a result is a sum of two products of a norm factor, a weight and a cosine, each good to a few 2^-24, so
2^-20 of the head's largest element covers it; gradients add a sum over the head (another factor of 2), the weights'
gradients a sum over all rows in 24 bits (2^-18 of the sum of magnitudes).  16-bit results: half a step of the type more.
"""
import pytest
import torch

from aussm_b200.rotary import qk_norm_rotate, rotary_frequencies
from oracle.delta import norm_rotate_ref

pytestmark = pytest.mark.gpu


def make(seed, b, l, hq, hk, d, rot, dtype=torch.float32, weights=True, far=0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)
    x = dict(q=r(b, l, hq, d).to(dtype), k=r(b, l, hk, d).to(dtype), gq=r(b, l, hq, d).to(dtype), gk=r(b, l, hk, d).to(dtype))
    if weights:
        x["q_weight"], x["k_weight"] = 1 + 0.3 * r(d), 1 + 0.3 * r(d)
    x["positions"] = torch.randint(0, 5000, (b, l), generator=gen) + far
    x = {n: t.cuda() for n, t in x.items()}
    x["frequencies"] = rotary_frequencies(rot, device="cuda")[0] if rot else None
    return x


def terms(x, n, kw):
    """The size of the two terms whose difference a gradient is: dx = r h w - x r^3 mean(h w x).  Each is rounded by a few
    2^-24 of its own size, r |h w|, however far they cancel (in a head of one element dx = r h w eps r^2: all of it
    cancels, 5e-7 is left of a term of 1 and an error of 2^-22 of that term is 0.5 of what is left)."""
    v = x[n].double()
    mean = {"rms": v.square().mean(-1, keepdim=True), "l2": v.square().sum(-1, keepdim=True)}.get(kw.get("norm", "rms"))
    r = 1.0 if mean is None else (mean + kw.get("eps", 1e-6)).rsqrt()
    w = float(x[n + "_weight"].abs().max()) if n + "_weight" in x else 1.0
    return r * x["g" + n].double().abs().amax(-1, keepdim=True) * w * kw.get("magnitude", 1.0)


def check(x, tables=True, **kw):
    leaves = [n for n in ("q", "k", "q_weight", "k_weight") if n in x]
    a = {n: x[n].clone().requires_grad_() for n in leaves}
    yq, yk = qk_norm_rotate(a["q"], a["k"], x["frequencies"], x["positions"] if tables else None, q_weight=a.get("q_weight"),
                            k_weight=a.get("k_weight"), **kw)
    grads = torch.autograd.grad([yq, yk], list(a.values()), [x["gq"], x["gk"]])
    t = {n: x[n].double().requires_grad_() for n in leaves}
    outs = [norm_rotate_ref(t[n], x["frequencies"], x["positions"] if tables else None, t.get(n + "_weight"), **kw) for n in "qk"]
    truth = torch.autograd.grad(outs, list(t.values()), [x["gq"].double(), x["gk"].double()])
    for n, got, want in zip(["yq", "yk"] + leaves, [yq, yk, *grads], [*outs, *truth]):
        got, want = got.detach(), want.detach()
        half = torch.finfo(got.dtype).eps / 2 if got.dtype != torch.float32 else 0.0
        if n.endswith("weight"):
            size = (want.abs().max() + (x["g" + n[0]].double() ** 2).sum((0, 1, 2)).max().sqrt() * 4) * 2 ** -18
        else:
            size = want.abs().amax(-1, keepdim=True) * 2 ** (-20 if n[0] == "y" else -19) + (0 if n[0] == "y" else want.abs().max() * 2 ** -21)
            if n[0] != "y":
                size = size + 2 ** -20 * terms(x, n, kw)
        err = (got.double() - want).abs()
        assert got.dtype == (torch.float32 if n.endswith("weight") else x["q"].dtype)
        assert (err <= half * want.abs() + size).all(), f"{n}: {float((err / (half * want.abs() + size)).max()):.3g}"


@pytest.mark.parametrize("norm", ["rms", "l2", None])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rot", [(128, 128), (64, 32), (80, 32), (6, 4), (5, 2), (256, 256), (36, 8), (250, 126), (1, 0), (96, 0)])
def test_layouts(norm, interleaved, d, rot):
    check(make(d + rot, 2, 9, 3, 2, d, rot), norm=norm, interleaved=interleaved)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b,l,hq,hk", [(1, 1, 1, 1), (4, 1, 8, 8), (1, 700, 9, 3), (2, 1500, 4, 4)])
def test_sizes_and_types(dtype, b, l, hq, hk):
    check(make(l, b, l, hq, hk, 64, 64, dtype))
    check(make(l, b, l, hq, hk, 64, 48, dtype, weights=False), norm="l2", eps=1e-5, magnitude=1.3)


@pytest.mark.parametrize("far", [1 << 20, 1 << 31, -(1 << 22)])
def test_far_positions(far):
    x = make(3, 2, 50, 2, 1, 128, 128, far=far)
    check(x)


def test_positions_of_all_kinds():
    x = make(5, 2, 33, 2, 2, 32, 32)
    check(x, tables=False)
    one = qk_norm_rotate(x["q"], x["k"], x["frequencies"], torch.arange(33, device="cuda"))
    none = qk_norm_rotate(x["q"], x["k"], x["frequencies"])
    row = qk_norm_rotate(x["q"], x["k"], x["frequencies"], torch.arange(33, device="cuda").expand(2, 33))
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(one, none, row))


def test_zero_heads_and_nan():
    """A head of zeros stays zero and has a finite gradient; a NaN stays in its head."""
    x = make(7, 1, 4, 2, 2, 64, 64)
    x["q"][0, 1, 0] = 0.0
    check(x)
    check(x, norm="l2")
    clean = qk_norm_rotate(x["q"], x["k"], x["frequencies"])[0]
    x["q"][0, 2, 1, 5] = float("nan")
    y = qk_norm_rotate(x["q"], x["k"], x["frequencies"])[0]
    assert torch.isnan(y[0, 2, 1]).all() and torch.equal(y[0, :2], clean[0, :2]) and torch.equal(y[0, 2, 0], clean[0, 2, 0])


def test_strides_and_determinism():
    x = make(9, 2, 300, 4, 4, 40, 40)
    ref = qk_norm_rotate(x["q"], x["k"], x["frequencies"], x["positions"], q_weight=x["q_weight"])
    fused = torch.zeros(2, 300, 4, 83, device="cuda")
    fused[..., 1:41], fused[..., 42:82] = x["q"], x["k"]
    odd = qk_norm_rotate(fused[..., 1:41], fused[..., 42:82], x["frequencies"], x["positions"], q_weight=x["q_weight"])
    front = [x[n].permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3) for n in "qk"]
    front = qk_norm_rotate(*front, x["frequencies"], x["positions"], q_weight=x["q_weight"])
    back = [x[n].transpose(1, 3).contiguous().transpose(1, 3) for n in "qk"]
    back = qk_norm_rotate(*back, x["frequencies"], x["positions"], q_weight=x["q_weight"])
    for i in range(2):
        assert torch.allclose(odd[i], ref[i], rtol=0, atol=float(ref[i].abs().max()) * 2 ** -20)     # another order of the norm's sum
        assert torch.equal(front[i], ref[i]) and torch.equal(back[i], ref[i])
    w = x["q_weight"].clone().requires_grad_()
    got = [torch.autograd.grad(qk_norm_rotate(x["q"], x["k"], x["frequencies"], q_weight=w), w, [x["gq"], x["gk"]])[0] for _ in range(2)]
    assert torch.equal(*got)
    # expanded heads and an expanded gradient
    q1 = x["q"][:, :, :1].clone().requires_grad_()
    y = qk_norm_rotate(q1.expand(2, 300, 4, 40), x["k"], x["frequencies"])[0]
    a, = torch.autograd.grad(y.sum(), q1, retain_graph=True)
    b, = torch.autograd.grad(y, q1, torch.ones_like(y))
    assert torch.equal(a, b)


def test_empty_graph_and_refusals():
    x = make(11, 2, 5, 2, 2, 32, 32)
    q, k, f = x["q"], x["k"], x["frequencies"]
    w = x["q_weight"].clone().requires_grad_()
    y = qk_norm_rotate(q[:, :0], k[:, :0], f, q_weight=w)
    assert y[0].shape == (2, 0, 2, 32)
    assert torch.equal(torch.autograd.grad(y[0].sum(), w)[0], torch.zeros_like(w))
    bad = [lambda: qk_norm_rotate(q.cpu(), k, f), lambda: qk_norm_rotate(q, k.half(), f), lambda: qk_norm_rotate(q.double(), k.double(), f),
           lambda: qk_norm_rotate(q, k[:, :2], f), lambda: qk_norm_rotate(q, k[..., :16], f), lambda: qk_norm_rotate(q, k, f.float()),
           lambda: qk_norm_rotate(q, k, torch.ones(17, device="cuda", dtype=torch.float64)), lambda: qk_norm_rotate(q, k, f.cpu()),
           lambda: qk_norm_rotate(q, k, f, x["positions"].int()), lambda: qk_norm_rotate(q, k, f, x["positions"][:, :3]),
           lambda: qk_norm_rotate(q, k, f.clone().requires_grad_()),
           lambda: qk_norm_rotate(q, k, f, norm="layer"), lambda: qk_norm_rotate(q, k, f, q_weight=w.detach()[:5]),
           lambda: qk_norm_rotate(q[0], k[0], f), lambda: qk_norm_rotate(torch.zeros(1, 1, 1, 257, device="cuda"), torch.zeros(1, 1, 1, 257, device="cuda")),
           lambda: torch.func.vmap(lambda a: qk_norm_rotate(a, k, f)[0])(q[None])]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()
    ref = qk_norm_rotate(q, k, f, x["positions"], q_weight=w)
    gref, = torch.autograd.grad(ref, w, [x["gq"], x["gk"]])
    ref, y = [t.detach() for t in ref], None      # torch captures no backward pass while an eager graph made on the default stream holds w
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        y = qk_norm_rotate(q, k, f, x["positions"], q_weight=w)
        gw, = torch.autograd.grad(y, w, [x["gq"], x["gk"]])
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y[0], ref[0]) and torch.equal(y[1], ref[1]) and torch.equal(gw, gref)


def test_differentiable_once():
    q, k = (torch.randn(1, 5, 2, 8, device="cuda").requires_grad_() for _ in range(2))
    yq, yk = qk_norm_rotate(q, k)
    gq, = torch.autograd.grad(yq.sum() + yk.sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(gq.sum(), q)


def test_gradients_with_their_sign_in_a_flag():
    q, k = (torch.randn(1, 5, 2, 8, device="cuda").requires_grad_() for _ in range(2))
    y = qk_norm_rotate(q, k)
    g = [torch.randn_like(t) for t in y]
    flagged = [torch.complex(torch.zeros_like(t), -t).conj().imag for t in g]
    assert all(t.is_neg() for t in flagged)
    for a, b in zip(torch.autograd.grad(y, [q, k], g, retain_graph=True), torch.autograd.grad(y, [q, k], flagged)):
        assert torch.equal(a, b)
