"""Gated delta rule and rotation without a GPU: the oracle against its own chunk form, frequencies, refusals."""
import math

import pytest
import torch

import aussm_b200
from aussm_b200.delta import gated_delta_rule, gated_delta_step
from aussm_b200.rotary import qk_norm_rotate, rotary_frequencies
from oracle.delta import gated_delta_ref, norm_rotate_ref


def test_oracle_against_the_triangular_system():
    """Over one chunk the recurrence is (I + A) e = beta (v - e^G k S): solved directly."""
    torch.manual_seed(0)
    l, dk, dv = 12, 6, 5
    q, k, v = (torch.randn(1, l, 1, d, dtype=torch.float64) for d in (dk, dk, dv))
    k = k / k.norm(dim=-1, keepdim=True)
    g, beta = -torch.rand(1, l, 1, dtype=torch.float64), torch.rand(1, l, 1, dtype=torch.float64)
    S = torch.randn(1, 1, dk, dv, dtype=torch.float64)
    o, last = gated_delta_ref(q, k, v, g, beta, initial_state=S)
    Q, K, V, G, b = q[0, :, 0], k[0, :, 0], v[0, :, 0], g[0, :, 0].cumsum(0), beta[0, :, 0, None]
    D = torch.exp(G[:, None] - G[None])
    e = torch.linalg.solve(torch.eye(l, dtype=torch.float64) + (b * D * (K @ K.T)).tril(-1), b * (V - G.exp()[:, None] * K @ S[0, 0]))
    want = (G.exp()[:, None] * Q @ S[0, 0] + (D * (Q @ K.T)).tril() @ e) / math.sqrt(dk)
    assert torch.allclose(o[0, :, 0], want, atol=1e-12)
    assert torch.allclose(last[0, 0], G[-1].exp() * S[0, 0] + ((G[-1] - G).exp()[:, None] * K).T @ e, atol=1e-12)


def test_rotation_oracle():
    x = torch.randn(1, 7, 2, 8, dtype=torch.float64)
    f, m = rotary_frequencies(8)
    assert m == 1.0 and f.dtype == torch.float64 and torch.allclose(f, 10000.0 ** -(torch.arange(4, dtype=torch.float64) / 4))
    for inter in (False, True):
        y = norm_rotate_ref(x, f, norm=None, interleaved=inter)
        assert torch.allclose(y.norm(dim=-1), x.norm(dim=-1))
        # products of turned vectors depend on the distance alone
        z = norm_rotate_ref(x, f, torch.arange(7) + 100, norm=None, interleaved=inter)
        assert torch.allclose(torch.einsum("bihd,bjhd->bhij", y, y), torch.einsum("bihd,bjhd->bhij", z, z))


def test_stretched_frequencies():
    plain, _ = rotary_frequencies(64)
    linear, _ = rotary_frequencies(64, scaling="linear", factor=4)
    assert torch.allclose(linear, plain / 4)
    base, _ = rotary_frequencies(64, scaling="base", factor=4)
    assert torch.isclose(base[0], plain[0]) and torch.isclose(base[-1], plain[-1] / 4)
    assert torch.allclose(rotary_frequencies(2, scaling="base", factor=4)[0], rotary_frequencies(2)[0] / 4)
    ramp, m = rotary_frequencies(64, scaling="ramp", factor=4, original_length=2048)
    made = 2048 * plain / (2 * math.pi)
    assert torch.allclose(ramp[made > 32], plain[made > 32]) and torch.allclose(ramp[made < 1], plain[made < 1] / 4)
    assert ((ramp <= plain) & (ramp >= plain / 4)).all() and m == pytest.approx(0.1 * math.log(4) + 1)
    for bad in (dict(dim=3), dict(dim=0), dict(dim=4, scaling="other"), dict(dim=4, factor=0.0)):
        with pytest.raises(RuntimeError):
            rotary_frequencies(**bad)


def test_no_cpu_path():
    q = torch.randn(1, 3, 1, 8)
    g = torch.zeros(1, 3, 1)
    for call in (lambda: gated_delta_rule(q, q, q, g, g), lambda: gated_delta_step(q, q, q, g, g, torch.zeros(1, 1, 8, 8)),
                 lambda: qk_norm_rotate(q, q)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_c_entries_refuse_on_the_host():
    """Bad problems come back as codes with a message; nothing is launched for them."""
    lib = aussm_b200._lib.load()
    good = (1, 10, 1, 2, 64, 64, 0)
    assert lib.aussm_b200_delta_keep_bytes(aussm_b200._lib.DeltaProblem(*good)) > 0
    for i, value in ((0, 0), (1, 0), (2, 0), (3, 0), (4, 0), (4, 129), (5, 0), (5, 257), (6, 3), (6, -1)):
        p = aussm_b200._lib.DeltaProblem(*(good[:i] + (value,) + good[i + 1:]))
        assert lib.aussm_b200_delta_keep_bytes(p) == 0 and lib.aussm_b200_delta_workspace_bytes(p, 1) == 0
        assert lib.aussm_b200_delta_step(p, *([None] * 9)) == -1
        assert lib.aussm_b200_last_error()
    assert lib.aussm_b200_delta_fwd(aussm_b200._lib.DeltaProblem(1, 10, 2, 3, 8, 8), *([None] * 9), 0, None, 0, None) == -1
    assert lib.aussm_b200_delta_fwd(None, *([None] * 9), 0, None, 0, None) == -1
    good = (1, 10, 1, 2, 64, 64, 0, 1, 0)
    for i, value in ((0, 0), (4, 257), (5, 3), (5, 66), (6, 5), (7, 3)):
        p = aussm_b200._lib.RotateProblem(*(good[:i] + (value,) + good[i + 1:]))
        assert lib.aussm_b200_rotate_fwd(p, *([None] * 9)) == -1 and lib.aussm_b200_rotate_bwd_workspace_bytes(p) == 0


def _with_oracle(monkeypatch):
    """The block's glue on the CPU: the oracle in place of the operators."""
    from aussm_b200 import models

    def rule(q, k, v, g, beta, **kw):
        return gated_delta_ref(q, k, v, g, beta)[0]

    def step(q, k, v, g, beta, state):
        o, new = gated_delta_ref(q, k, v, g, beta, initial_state=state)
        state.copy_(new)
        return o

    def rotate(q, k, frequencies=None, positions=None, **kw):
        return tuple(norm_rotate_ref(t, frequencies, positions, **kw) for t in (q, k))

    monkeypatch.setattr(models.delta, "gated_delta_rule", rule)
    monkeypatch.setattr(models.delta, "gated_delta_step", step)
    monkeypatch.setattr(models.rotary, "qk_norm_rotate", rotate)
    return models


@pytest.mark.parametrize("rotary_dim,bias", [(0, False), (8, True)])
def test_block_steps_are_its_sequence(monkeypatch, rotary_dim, bias):
    models = _with_oracle(monkeypatch)
    torch.manual_seed(0)
    block = models.GatedDeltaBlock(32, n_heads=2, rotary_dim=rotary_dim, bias=bias).double()
    x = torch.randn(2, 9, 32, dtype=torch.float64)
    whole = block(x)
    cache = block.init_cache(2, dtype=torch.float64)
    cache["state"] = cache["state"].double()
    steps = torch.cat([block.step(x[:, t:t + 1], cache) for t in range(9)], 1)
    assert torch.allclose(steps, whole, atol=1e-12) and cache["position"] == 9
    assert torch.equal(whole[:, :5], block(torch.cat((x[:, :5], torch.randn(2, 4, 32, dtype=torch.float64)), 1))[:, :5])   # causal


def test_block_in_the_models(monkeypatch):
    models = _with_oracle(monkeypatch)
    torch.manual_seed(0)
    net = models.SSMTS(d_model=16, input_dim=3, output_dim=2, layers="g|g")
    y = net(torch.randn(2, 7, 3))
    y.square().mean().backward()
    assert y.shape == (2, 7, 2) and all(torch.isfinite(p.grad).all() for p in net.parameters())
    assert models.GatedDeltaBlock(512).n_heads == 4 and models.GatedDeltaBlock(96).n_heads == 1
    for bad in (dict(d_model=30, n_heads=4), dict(d_model=512, n_heads=2), dict(d_model=32, rotary_dim=3), dict(d_model=32, n_heads=2, rotary_dim=18)):
        with pytest.raises(ValueError):
            models.GatedDeltaBlock(**bad)


def test_block_reads_a_prompt_in_pieces(monkeypatch):
    models = _with_oracle(monkeypatch)
    called = []

    def rule(q, k, v, g, beta, initial_state=None, return_final_state=False):
        called.append(q.shape[1])
        o, s = gated_delta_ref(q, k, v, g, beta, initial_state=initial_state)
        return (o, s) if return_final_state else o

    monkeypatch.setattr(models.delta, "gated_delta_rule", rule)
    torch.manual_seed(1)
    block = models.GatedDeltaBlock(32, n_heads=2, rotary_dim=8, bias=True).double()
    x = torch.randn(2, 60, 32, dtype=torch.float64)
    whole = block(x)
    cache = block.init_cache(2, dtype=torch.float64)
    cache["state"] = cache["state"].double()
    cuts = [0, 37, 38, 40, 43, 60]
    pieces = torch.cat([block.step(x[:, a:b], cache) for a, b in zip(cuts, cuts[1:])], 1)
    # The gates are cast to float32: a product summed in another order (1e-16 off) may round to its neighbour, one step of
    # 2^-23 relative.  |a| < 4 moves softplus(a + dt) and so g by at most 4 * 2^-23 of itself (softplus' <= softplus for
    # arguments below 0.5, and the step sizes start at 0.1 or less), the state, in which a decay of g lasts 1 / |g| steps,
    # by as much of itself, beta by 2^-23: 6e-7 of o, and as much again through the norm of the head and its product.
    assert torch.allclose(pieces, whole, rtol=0, atol=2e-6 * float(whole.detach().abs().max()))
    assert int(cache["position"]) == 60 and called == [60, 37, 17]


def test_sizes_of_the_longest_sequences():
    """Lengths near 2^31: a chunk more is a chunk's bytes more."""
    lib = aussm_b200._lib.load()
    keep = lambda l: lib.aussm_b200_delta_keep_bytes(aussm_b200._lib.DeltaProblem(16, l, 1, 1, 8, 8, 0))
    one = (keep(64 * 2 * 10 ** 6) - keep(64 * 10 ** 6)) // 10 ** 6
    for l in (2 ** 28, 2 ** 31 - 64, 2 ** 31 - 63, 2 ** 31 - 1):
        assert keep(l) - keep(64 * 10 ** 6) == one * ((l + 63) // 64 - 10 ** 6), l
    assert lib.aussm_b200_delta_keep_bytes(aussm_b200._lib.DeltaProblem(33, 2 ** 31 - 1, 1, 1, 8, 8, 0)) == 0      # 33 * 2^25 chunks


def test_the_blocks_frequencies_serve_training_after_inference():
    from aussm_b200 import models
    block = models.GatedDeltaBlock(32, n_heads=2, rotary_dim=8)
    with torch.inference_mode():
        first = block._frequencies(torch.device("cpu"))
    assert block._frequencies(torch.device("cpu")) is first and not first.is_inference()

    class Keep(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, f):
            ctx.save_for_backward(x, f)
            return x * f.sum()

        @staticmethod
        def backward(ctx, g):
            return g * ctx.saved_tensors[1].sum(), None

    x = torch.ones(3, dtype=torch.float64, requires_grad=True)
    Keep.apply(x, first).sum().backward()
    assert torch.equal(x.grad, first.sum().expand(3))


def test_stretch_wants_rising_turns():
    with pytest.raises(RuntimeError, match="rising"):
        rotary_frequencies(8, scaling="ramp", factor=2.0, turns=(4.0, 4.0))
