"""Gated delta rule, single steps and rotation at sizes whose branches and limits the other tests do not reach."""
import pytest
import torch

from aussm_b200.delta import gated_delta_rule, gated_delta_step
from aussm_b200.rotary import qk_norm_rotate

pytestmark = pytest.mark.gpu


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
