"""Linear attention layers and an attention layer over a paged cache, as a hybrid model uses them: prompts of several users in
one packed row, their states and keys taken into pools, then tokens one by one, with users that come and go, against every user's
whole sequence in 64 bits."""
import pytest
import torch

from oracle.linear_attention import linear_attention_oracle, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompts_then_tokens(dtype):
    from mamba_amd.ops.linear_attention import linear_attention_fn, linear_attention_state_update
    from mamba_amd.ops.paged_attention import paged_attention_update
    heads, kv, dk, dv, page = 4, 2, 32, 48, 16
    prompts, steps = [70, 1, 130, 15], 20
    g = torch.Generator().manual_seed(0)
    users = [{n: torch.randn(p + steps, h, d, generator=g).to(dtype) for n, h, d in
              (("q", heads, dk), ("k", kv, dk), ("v", kv, dv))} for p in prompts]
    decay = torch.tensor([-0.7, -0.1, -0.01, 0.0])
    lin = [linear_attention_oracle(*(u[n][None] for n in "qkv"), decay) for u in users]

    # the prompts: one packed row; the attention layer's keys and values go to the users' pages
    row = {n: torch.cat([u[n][:p] for u, p in zip(users, prompts)])[None].cuda() for n in "qkv"}
    cu = torch.tensor([0, *torch.tensor(prompts).cumsum(0).tolist()], dtype=torch.int32, device="cuda")
    out, final = linear_attention_fn(row["q"], row["k"], row["v"], decay.cuda(), cu_seqlens=cu, return_final_states=True)
    for n, p in enumerate(prompts):
        at = slice(int(cu[n]), int(cu[n]) + p)
        within("prompt", out[0, at], lin[n][0]["out"][0, :p], lin[n][1]["out"][0, :p])
    slots = [5, 0, 3, 1]
    pool = torch.full((7, heads, dk, dv), 9.0, device="cuda")
    pool[slots] = final
    wide = 10
    order = torch.randperm(4 * wide, generator=g)
    table = order.view(4, wide).to(torch.int32).cuda()
    caches = {n: torch.full((4 * wide, page, kv, d), float("nan"), dtype=dtype, device="cuda") for n, d in (("k", dk), ("v", dv))}
    for u, p, pages in zip(users, prompts, table):
        pos = torch.arange(p, device="cuda")
        for n in "kv":
            caches[n][pages[pos // page].long(), pos % page] = u[n][:p].cuda()

    # tokens: in every step some users wait (empty places), the others go on by one
    done = list(prompts)
    for step in range(steps + 4):
        active = [done[n] < prompts[n] + steps and (step + n) % 6 != 0 for n in range(4)]
        token = {n: torch.stack([users[i][n][min(done[i], prompts[i] + steps - 1)] for i in range(4)]).cuda() for n in "qkv"}
        rows = torch.tensor([slots[i] if active[i] else -1 for i in range(4)], dtype=torch.int32, device="cuda")
        lens = torch.tensor([done[i] if active[i] else -1 for i in range(4)], dtype=torch.int32, device="cuda")
        out = linear_attention_state_update(pool, token["q"], token["k"], token["v"], decay.cuda(), state_batch_indices=rows)
        att = paged_attention_update(token["q"], token["k"], token["v"], caches["k"], caches["v"], table, lens)
        for i in range(4):
            if not active[i]:
                assert torch.count_nonzero(out[i]) == 0 and torch.count_nonzero(att[i]) == 0
                continue
            t = done[i]
            within("linear", out[i], lin[i][0]["out"][0, t], lin[i][1]["out"][0, t])
            keys, values = (users[i][n][:t + 1].double().repeat_interleave(heads // kv, 1) for n in "kv")
            p = torch.softmax(dk ** -0.5 * (keys * users[i]["q"][t].double()).sum(-1), 0)[..., None]
            # weights and outputs are rounded to the type, everything else is fp32
            bound = (p * values.abs()).sum(0) * ((2.0 ** -8 if dtype == torch.bfloat16 else 0.0) + 1000 * 2.0 ** -24)
            within("attention", att[i], (p * values).sum(0), bound)
            done[i] += 1
    assert all(d > p + 10 for d, p in zip(done, prompts))
    for i in range(4):
        ref, bound = linear_attention_oracle(*(users[i][n][None, :done[i]] for n in "qkv"), decay)
        within("state", pool[slots[i]], ref["final"][0], bound["final"][0])
    assert bool((pool[[2, 4, 6]] == 9.0).all())
