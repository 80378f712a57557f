"""Gated delta rule, single steps and rotation at sizes whose branches and limits the other tests do not reach.

Beside the bounds on every element (see test_gpu_delta.py) the root mean square of the differences is held: each of about 8
products in a row (gradients: 16) drops lo lo and rounds the lo parts, 2^-22 of its terms where these are as good as
independent, and in the worst case all of them add up in the same direction: 8 * 2^-22 and 16 * 2^-22 of the root mean square
of the result, and half a step of the type in 16 bits.
"""
import pytest
import torch

import aussm_b200
from aussm_b200.delta import gated_delta_rule, gated_delta_step
from aussm_b200.rotary import qk_norm_rotate
from oracle.delta import gated_delta_ref
from tests.test_gpu_delta import BWD, FWD, NAMES, both, close, compare, make
from tests.test_gpu_rotary import check as check_rotation
from tests.test_gpu_rotary import make as make_rotation

pytestmark = pytest.mark.gpu


def rms(x):
    return float(x.double().square().mean().sqrt())


def compare_closely(res):
    compare(res)
    (got, ggot), (truth, gtruth) = res
    for names, a, b, n in (("outputs", got, truth, 8), ("gradients", ggot, gtruth, 16)):
        for x in a:
            half = torch.finfo(a[x].dtype).eps / 2 if a[x].dtype != torch.float32 else 0.0
            assert rms(a[x].double() - b[x].double()) <= (n * 2 ** -22 + half) * rms(b[x]), (names, x)


@pytest.mark.parametrize("shape", [(1, 2 ** 32 + 5, 1), (2 ** 32 + 5, 1, 1), (1, 3, 2 ** 32 + 1)])
def test_sizes_beyond_31_bits_are_refused(shape):
    """Expanded tensors take no memory, and a size must not lose its upper bits on the way to the kernels."""
    x = torch.zeros(1, 1, 1, 1, device="cuda").expand(*shape, 1)
    g = torch.zeros(1, 1, 1, device="cuda").expand(*shape)
    state = torch.zeros(1, 1, 1, 1, device="cuda").expand(shape[0], shape[2], 1, 1)
    with pytest.raises(RuntimeError, match="below 2\\^31"):
        gated_delta_rule(x, x, x, g, g)
    with pytest.raises(RuntimeError, match="below 2\\^31"):
        gated_delta_step(x, x, x, g, g, state)
    with pytest.raises(RuntimeError, match="below 2\\^31"):
        qk_norm_rotate(x, x)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dv", [68, 128, 132, 200])
def test_steps_of_many_states(dtype, dv):
    """600 states of more than 64 values: whole rows a block, with a second slice that is not full."""
    d = make(dv, 300, 2, 1, 2, 16, dv, dtype)
    y = {n: x.double() for n, x in d.items()}
    o64, s64 = gated_delta_ref(*(y[n] for n in NAMES[:5]), initial_state=y["state"])
    before, new = d["state"].clone(), torch.empty_like(d["state"])
    o = gated_delta_step(*(d[n] for n in NAMES), new_state=new)
    assert torch.equal(d["state"], before)
    close("o", o, o64, FWD)
    close("s", new, s64, FWD)
    assert torch.equal(gated_delta_step(*(d[n] for n in NAMES)), o) and torch.equal(d["state"], new)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("b,l,hk,hv,dk,dv", [(6, 1100, 2, 4, 48, 64), (1, 1300, 1, 3, 128, 128), (2, 1024, 1, 1, 64, 256)])
def test_segments_of_shared_heads(dtype, b, l, hk, hv, dk, dv):
    """24 heads of 64 values are chained 16 columns a block, fewer of them 8; value heads that share key heads."""
    compare_closely(both(make(l + hv, b, l, hk, hv, dk, dv, dtype, rate=0.05)))


@pytest.mark.parametrize("l,rate", [(64, 1.0), (700, 0.02)])
def test_typical_differences(l, rate):
    compare_closely(both(make(l, 4, l, 4, 8, 128, 128, rate=rate)))
    compare_closely(both(make(l, 4, l, 4, 4, 64, 64, rate=rate)))


def test_a_long_sequence():
    """65536 steps in 148 segments: heads that remember all of it against the recurrence."""
    d = make(71, 1, 65536, 1, 1, 128, 8, rate=1e-4)
    o, s = gated_delta_rule(*(d[n] for n in NAMES[:5]), initial_state=d["state"], return_final_state=True)
    y = {n: t.double() for n, t in d.items()}
    o64, s64 = gated_delta_ref(*(y[n] for n in NAMES[:5]), initial_state=y["state"])
    close("o", o, o64, FWD)
    close("s", s, s64, FWD)
    assert rms(o - o64) <= 8 * 2 ** -22 * rms(o64) and rms(s - s64) <= 8 * 2 ** -22 * rms(s64)
    assert aussm_b200.device_status() == 0


def test_gradients_of_a_long_sequence():
    compare_closely(both(make(73, 1, 9500, 1, 1, 64, 8, rate=1e-3)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("b,l,hq,hk,d,rot", [(3, 7001, 2, 1, 128, 128), (1, 9973, 1, 2, 256, 128), (1, 9973, 1, 1, 33, 10), (2, 20011, 1, 1, 24, 24)])
def test_rotations_of_many_tokens(dtype, b, l, hq, hk, d, rot):
    """More tokens than the backward kernel's blocks hold at once: further rounds, the last one not full."""
    check_rotation(make_rotation(l, b, l, hq, hk, d, rot, dtype))


@pytest.mark.parametrize("hq,hk", [(5, 9), (9, 1), (16, 4)])
def test_rotations_of_many_heads(hq, hk):
    """A group that walks all heads of a token comes to its loop's second pass and leaves it in the middle."""
    check_rotation(make_rotation(hq, 1, 3000, hq, hk, 64, 64))
    check_rotation(make_rotation(hq, 1, 3000, hq, hk, 64, 32, torch.bfloat16), interleaved=True)
