"""A state that wants gradients is refused before anything else happens (no GPU)."""
import pytest
import torch

from mamba_amd.ops.gated_linear_scan import gated_linear_state_update


def test_a_state_that_wants_gradients():
    args = [torch.zeros(3, 4) for _ in range(3)] + [torch.zeros(4)]
    state = torch.zeros(3, 4, requires_grad=True)
    for s in (state, 2 * state, (2 * state)[:3]):
        with pytest.raises(RuntimeError, match="state is updated in place"):
            gated_linear_state_update(s, *args)
        with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU fallback"):
            gated_linear_state_update(s, *args)
