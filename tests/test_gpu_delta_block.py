"""GatedDeltaBlock: what its first call keeps for the later ones."""
import pytest
import torch

from aussm_b200 import models

pytestmark = pytest.mark.gpu


def block_and_input():
    torch.manual_seed(8)
    return models.GatedDeltaBlock(64, n_heads=2, rotary_dim=32).cuda(), torch.randn(2, 70, 64, device="cuda")


def test_training_after_a_first_call_without_gradients():
    block, x = block_and_input()
    want = block(x)
    want_grads = torch.autograd.grad(want.square().mean(), list(block.parameters()))
    for mode in (torch.inference_mode, torch.no_grad):
        block._angles.clear()
        with mode():
            first = block(x)
        again = block(x)
        grads = torch.autograd.grad(again.square().mean(), list(block.parameters()))
        assert torch.equal(first, want) and torch.equal(again, want)
        assert all(torch.equal(a, b) for a, b in zip(grads, want_grads))


def test_a_first_call_on_a_stream_of_its_own():
    """The other streams may use what it keeps as soon as it returns, whatever lies before it on its own stream."""
    block, x = block_and_input()
    with torch.no_grad():
        want = block(x)
        block._angles.clear()
        busy = torch.randn(4096, 4096, device="cuda")
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(50):
                busy = busy @ busy * 1e-2
            block._frequencies(x.device)
        got = block(x)
        torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
