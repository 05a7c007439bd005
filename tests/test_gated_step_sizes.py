"""The number of channels that gated_linear_state_update takes: refusals (no GPU), and the largest row."""
import pytest
import torch

from mamba_amd import _lib
from mamba_amd.ops.gated_linear_scan import gated_linear_state_update


@pytest.mark.parametrize("dim", [2 ** 30 + 1, 2 ** 30 + 4, 2 ** 31 - 1024, 2 ** 31 - 1])
@pytest.mark.parametrize("dtype", range(3))
@pytest.mark.parametrize("state_dtype", range(3))
def test_rows_beyond_32_bit_byte_offsets_are_refused(dim, dtype, state_dtype):
    """A lane's place in a row is counted in bytes, 32 bits: 2^30 channels of 4 bytes are the most."""
    p = _lib.GatedStepParams()
    p.batch = p.state_rows = 1
    p.dim, p.dtype, p.state_dtype = dim, dtype, state_dtype
    for n in ("state", "x", "gate_a", "gate_x", "decay", "out"):
        setattr(p, n, 256)  # stand-ins: refused before any launch
    assert _lib.load().gated_state_update(p, None) == -2


@pytest.mark.parametrize("dim", [2 ** 30 + 1, 2 ** 31 - 1])
def test_the_operator_says_so(dim):
    one = torch.zeros(1, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="at most 2\\^30 channels"):
        gated_linear_state_update(*[one.expand(1, dim)] * 4, one.expand(dim))


@pytest.mark.gpu
def test_the_largest_row():
    """Channels at the ends and around every 2^28 of a row of 2^30, against the same channels as a row of their own."""
    dim = 2 ** 30
    big = lambda dtype: torch.zeros(1, dim, dtype=dtype, device="cuda")
    state, x, gate_a, gate_x, decay = big(torch.float32), *[big(torch.bfloat16) for _ in range(4)]
    places = [slice(max(c - 300, 0), min(c + 300, dim)) for c in (0, 2 ** 28, 2 ** 29, 3 * 2 ** 28, dim)]
    g = torch.Generator(device="cuda").manual_seed(0)
    for at in places:
        for t in (state, x, gate_a, gate_x, decay):
            t[:, at] = torch.randn(1, at.stop - at.start, device="cuda", generator=g)
    alone = [state[:, at].clone() for at in places]
    outs = [gated_linear_state_update(s, *[t[:, at].contiguous() for t in (x, gate_a, gate_x)], decay[0, at]) for s, at in zip(alone, places)]
    out = gated_linear_state_update(state, x, gate_a, gate_x, decay[0])
    for at, s, o in zip(places, alone, outs):
        assert torch.equal(state[:, at], s) and torch.equal(out[:, at], o)
    assert int(torch.count_nonzero(state)) <= sum(at.stop - at.start for at in places)
