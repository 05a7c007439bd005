"""Linear attention and attention over a paged cache at the ends of their ranges: weights far below the largest one,
scores near the least number."""
import pytest
import torch

from oracle.linear_attention import U, within

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch", [1, 3100])  # in ranges; a workgroup a sequence, whose waves have a quarter of the positions each
@pytest.mark.parametrize("low", [-8.0, -13.0, -17.5, -20.0])
def test_many_small_weights_beside_a_large_one(batch, low, dtype):
    """A first position that draws nearly all of the weight and has no value: what the others have is the whole result."""
    from mamba_amd.ops.paged_attention import paged_attention_update
    n, page, size = 8000, 16, 64
    k, v = torch.zeros(n // page, page, 1, size), 1 + torch.rand(n // page, page, 1, size, generator=torch.Generator().manual_seed(0))
    k[..., 0], k[0, 0, 0, 0], v[0, 0] = low, 0.0, 0.0
    v = v.to(dtype)
    q = torch.zeros(batch, 1, size)
    q[..., 0] = 1
    table = torch.arange(n // page, dtype=torch.int32, device="cuda").expand(batch, -1)
    out = paged_attention_update(q.to(dtype).cuda(), None, None, k.to(dtype).cuda(), v.cuda(), table,
                                 torch.full((batch,), n, dtype=torch.int32, device="cuda"), scale=1.0)
    w = torch.softmax(k[..., 0].double().flatten(), 0)[:, None] * v.double().flatten(0, 2)
    ref = w.sum(0)
    # The scores are exact but for their factor log2(e), 2 u of them; a weight: 16 u and half a step of the type, in fp16 of numbers of 2^-24
    # at least beside a largest one of 2^15; sums of n positions.
    rounding = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}.get(dtype, 0.0)
    bound = ref * (rounding + (2 * abs(low) + 32 + 2 * n) * U) + (2.0 ** -40 * n * 2 if dtype == torch.float16 else 0.0)
    for row in (0, batch // 2, batch - 1):
        within("out", out[row, 0], ref, bound)
    assert bool((out == out[:1]).all())


@pytest.mark.parametrize("positions", [1, 2, 700])
def test_scores_near_the_least_number(positions):
    """Scores that are all below -3e38 in units of log2: weights are shares of the largest one as ever."""
    from mamba_amd.ops.paged_attention import paged_attention_update
    k = torch.full((positions, 1, 2, 4), 0.0)
    k[..., 0] = -2.25e19  # times 1e19 times log2(e): -3.25e38
    v = torch.rand(positions, 1, 2, 4, generator=torch.Generator().manual_seed(0))
    q = torch.zeros(1, 2, 4)
    q[..., 0] = 1e19
    args = [t.cuda() for t in (k, v, torch.arange(positions, dtype=torch.int32)[None], torch.tensor([positions], dtype=torch.int32))]
    out = paged_attention_update(q.cuda(), None, None, *args, scale=1.0)
    ref = v.double().mean((0, 1))[None]
    within("out", out, ref, ref * (32 + 2 * positions) * U)
