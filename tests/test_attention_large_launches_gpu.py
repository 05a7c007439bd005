"""Linear attention and attention over a paged cache where one workgroup a (sequence, head) makes more workgroups than one dimension
of a launch takes threads for, 2^24 of them: batches of one position and of heads of one value, against 64 bits."""
import pytest
import torch

from oracle.linear_attention import U

pytestmark = pytest.mark.gpu


def _random(seed, *shape):
    return torch.rand(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)) + 0.5


def _near(got, want, terms=1):
    """Products of up to four numbers and their sums: a few roundings each."""
    assert bool(((got.double() - want).abs() <= (8 + terms) * U * want.abs()).all())


def test_linear_attention_forward():
    from mamba_amd.ops.linear_attention import linear_attention_fn
    q, k, v = (_random(n, 2 ** 18 + 3, 1, 64, 1) for n in range(3))
    out = linear_attention_fn(q, k, v, torch.zeros(64, device="cuda"), scale=0.75)
    _near(out, 0.75 * q.double() * k.double() * v.double())


def test_linear_attention_gradients_of_shared_heads():
    from mamba_amd.ops.linear_attention import linear_attention_fn
    batch, heads, kv = 90_000, 64, 32
    q, dout = _random(0, batch, 1, heads, 1), _random(3, batch, 1, heads, 1)
    k, v = _random(1, batch, 1, kv, 1), _random(2, batch, 1, kv, 1)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    dq, dk, dv = torch.autograd.grad(linear_attention_fn(*leaves, torch.zeros(heads, device="cuda"), scale=0.75), leaves, dout)
    q, k, v, dout = (t.detach().double() for t in (q, k, v, dout))
    pairs = (q * dout).unflatten(2, (kv, heads // kv)).sum(3)
    _near(dq, 0.75 * dout * (k * v).repeat_interleave(heads // kv, 2))
    _near(dk, 0.75 * v * pairs, 2)
    _near(dv, 0.75 * k * pairs, 2)


def test_attention_over_a_paged_cache():
    from mamba_amd.ops.paged_attention import paged_attention_update
    batch, heads = 65535, 260
    k_cache, v_cache = (_random(n, 2, 4, heads, 1) for n in (0, 1))
    q = _random(2, batch, heads, 1)
    table = torch.zeros(batch, 1, dtype=torch.int32, device="cuda")
    table[1::2] = 1
    lens = torch.full((batch,), 3, dtype=torch.int32, device="cuda")
    out = paged_attention_update(q, None, None, k_cache, v_cache, table, lens, scale=1.0)
    for first in (0, 1):
        w = torch.softmax(q[first::2, None, :, 0].double() * k_cache[first, :3, :, 0].double(), 1)
        _near(out[first::2, :, 0], (w * v_cache[first, :3, :, 0].double()).sum(1), 32)
