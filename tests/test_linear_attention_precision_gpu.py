"""linear_attention_fn where one product of an operand, a decay and ones makes each result: its bits can be told one by one.

Keys and queries are rows of the unit matrix, so every element of a state, a gradient or (with output gradients that are such rows too) an
output has one term, and nothing but zeros is added to it.  Such an element is off by, u = 2^-24,
 * three factors f^n = 2^x and their products with the operand and one another, 2 u and u each, and their arguments' 3 u |x| ln 2, which
   is 3 u |log_decay| L in all: 9 u, scale and the last product, 2 u;
 * a block that a state goes through: its decay 2 u and u, up to three sums of matrix instructions at 2 u: 9 u;
 * a segment: its decay, product and sum, 4 u;
 * the row that a state takes up in three bf16 parts, u (in two parts it would be up to 2^-17 = 128 u);
or (20 + 9 blocks + 4 segments + 3 |log_decay| L) u.  The general bounds beside the oracle's results, for sums of any terms, are
40 times as wide."""
import pytest
import torch

from oracle.linear_attention import U, linear_attention_oracle, within

DECAYS = torch.tensor([0.0, -1 / 256, -0.02, -0.11])


def _inputs(L, size, dtype, first=0, seed=0):
    """Four heads; the positions from `first` on have a key and a query each."""
    g = torch.Generator().manual_seed(seed)
    one = torch.zeros(3, 1, L, 4, size)
    n = L - first
    assert n <= size
    t = torch.arange(first, L)
    for h in range(4):
        for row, order in zip(one, (t - first, torch.randperm(n, generator=g), torch.randperm(n, generator=g))):
            row[0, t, h, order] = 1
    v = (1 + torch.rand(1, L, 4, size, generator=g)) * torch.randint(0, 2, (1, L, 4, size), generator=g).sub(0.5).sign()
    return one.to(dtype), v.to(dtype)


def _bound(ref, L, blocks, segments, axis):
    heads = (20 + 9 * blocks + 4 * segments + 3 * DECAYS.abs() * L).double() * U
    return ref.abs() * heads.view([-1 if a == axis else 1 for a in range(4)])


def _run(q, k, v, dout):
    from mamba_amd.ops.linear_attention import linear_attention_fn
    start = torch.zeros(1, 4, q.shape[-1], v.shape[-1], device="cuda", requires_grad=True)
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    out, final = linear_attention_fn(*leaves, DECAYS.cuda(), scale=1.0, initial_states=start, return_final_states=True)
    return dict(zip(("out", "final", "dq", "dk", "dv", "dinitial"), (out, final, *torch.autograd.grad(out, [*leaves, start], dout.cuda()))))


@pytest.mark.gpu
@pytest.mark.parametrize("L,size", [(1, 16), (16, 64), (17, 33), (33, 64), (64, 64), (100, 128), (64, 200)])
def test_every_result_in_fp32(L, size):
    (k, q, ones), v = _inputs(L, size, torch.float32, seed=L)
    for dout in (ones, v.roll(1, 1)):
        got = _run(q, k, v, dout)
        ref, _ = linear_attention_oracle(q, k, v, DECAYS, 1.0, None, None, dout)
        for n, x in got.items():
            if n == "dq" or n == "dk":  # products with v: of one term where dout has one value
                if dout is not ones:
                    continue
            within(n, x, ref[n], _bound(ref[n], L, L / 16 + 1, 1, 1 if n in ("final", "dinitial") else 2))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("L,size,first", [(2, 16, 0), (32, 64, 0), (31, 33, 0), (24, 128, 0), (300, 64, 280), (777, 128, 757), (500, 40, 480), (260, 250, 240)])
def test_states_that_are_results_in_16_bit_types(L, size, first, dtype):
    (k, q, _), v = _inputs(L, size, dtype, first, seed=L)
    got = _run(q, k, v, v)
    back = {n: t.flip(1) for n, t in (("q", q), ("k", k), ("v", v))}  # the last positions of the walk are the first of the sequence
    mirrored = _run(back["q"], back["k"], back["v"], back["v"])
    ref, _ = linear_attention_oracle(q, k, v, DECAYS, 1.0, None, None, v)
    within("final", got["final"], ref["final"], _bound(ref["final"], L - first, 2, 1, 1))
    ref, _ = linear_attention_oracle(back["q"], back["k"], back["v"], DECAYS, 1.0, None, None, back["v"])
    within("dinitial", mirrored["dinitial"], ref["dinitial"], _bound(ref["dinitial"], L - first, 2, 1, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("batch,L,heads,kv,dk,dv", [(1, 1, 1, 1, 1, 1), (5, 1, 32, 4, 96, 48), (1, 2, 4, 4, 16, 16), (2, 31, 4, 2, 64, 64), (1, 32, 2, 2, 128, 128),
                                                   (1, 32, 2, 2, 256, 40), (3, 17, 3, 3, 33, 7)])
def test_results_of_one_block_are_rounded_once(batch, L, heads, kv, dk, dv, dtype):
    """Without a state that comes in, a block's results are products of its scores, which are held in two bf16 parts (2^-16 of them; in
    fp16 the products of two second parts are left out, 2^-16 more): what is seen is the rounding of the result."""
    from mamba_amd.ops.linear_attention import linear_attention_fn
    g = torch.Generator().manual_seed(L + dk)
    r = lambda h, d: torch.randn(batch, L, h, d, generator=g).to(dtype)
    q, k, v, dout, decay = r(heads, dk), r(kv, dk), r(kv, dv), r(heads, dv), torch.log1p(-torch.exp2(-torch.linspace(1, 12, heads)))
    ref, _ = linear_attention_oracle(q, k, v, decay, dout=dout)
    # sums of absolute values: the same of absolute operands
    size, _ = linear_attention_oracle(q.abs(), k.abs(), v.abs(), decay, dout=dout.abs())
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    out = linear_attention_fn(*leaves, decay.cuda())
    for n, x in zip(("out", "dq", "dk", "dv"), (out, *torch.autograd.grad(out, leaves, dout.cuda()))):
        within(n, x, ref[n], size[n] * (2.0 ** -15 + (dk + dv + 32 + 60) * U))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("L", [24, 32])
def test_the_bound_tells_two_parts_from_three(dtype, L):
    """What rows in two parts and in three make of the same states, on the CPU."""
    (k, _, _), v = _inputs(L, 64, dtype, seed=L)
    rows = v[0].double() * torch.exp(DECAYS.double()[:, None] * (L - 1 - torch.arange(L).double()[:, None, None]))
    left, inside = rows.float(), []
    bound = _bound(rows[None], L, 2, 1, 2)[0]
    for part in range(3):
        left = left - left.bfloat16().float()
        inside.append(left.abs().double() <= bound)
    assert not bool(inside[0].all()) and not bool(inside[1].all()) and bool(inside[2].all())
    assert float(inside[1].double().mean()) < 0.9
