"""paged_attention_update against the 64-bit oracle: outputs within the bounds that stand beside the oracle's plus half a step
of the result's type, the caches bit for bit."""
import pytest
import torch

from oracle.linear_attention import paged_attention_oracle, within

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _fn(*args, **kw):
    from mamba_amd.ops.paged_attention import paged_attention_update
    return paged_attention_update(*args, **kw)


@pytest.fixture(params=["ext", "ctypes"])
def host(request, monkeypatch):
    from mamba_amd import _lib
    if request.param == "ctypes":
        monkeypatch.setattr(_lib, "_torch_ext", None)
    return request.param


def _inputs(lens, heads, kv, dk, dv, page, dtype, wide=None, seed=0, spare=3):
    """Caches whose unused positions hold no numbers, and tables in disorder whose unused entries are none."""
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype)
    batch = len(lens)
    wide = wide or max(1, max(n // page + 1 for n in lens))
    pages = sum(min(max(n, 0) // page + 1, wide) for n in lens) + spare
    order = torch.randperm(pages, generator=g).tolist()
    table, k_cache, v_cache = [], r(pages, page, kv, dk), r(pages, page, kv, dv)
    used = torch.zeros(pages, page, dtype=torch.bool)
    for n in lens:
        mine = [order.pop() for _ in range(min(max(n, 0) // page + 1, wide))] if n >= 0 else []
        for p in range(min(max(n, 0), wide * page)):
            used[mine[p // page], p % page] = True
        table.append(mine + [-1 if len(table) % 2 else 2 ** 30] * (wide - len(mine)))
    k_cache[~used], v_cache[~used] = float("nan"), float("nan")
    return dict(q=2 * r(batch, heads, dk), k=r(batch, kv, dk), v=r(batch, kv, dv), k_cache=k_cache, v_cache=v_cache), table, lens


def _call(t, table, lens, int_dtype=torch.int32, **kw):
    d = {k: (v.cuda() if v is not None else None) for k, v in t.items()}
    out = _fn(**d, block_table=torch.tensor(table, dtype=int_dtype, device="cuda"),
              cache_seqlens=torch.tensor(lens, dtype=int_dtype, device="cuda"), **kw)
    return out, d["k_cache"], d["v_cache"]


def _same(a, b):
    return torch.equal(a.cpu().nan_to_num(nan=123.0), b.cpu().nan_to_num(nan=123.0))


def _check(inputs, **kw):
    t, table, lens = inputs
    out, k_cache, v_cache = _call(t, table, lens, **kw)
    kw.pop("int_dtype", None)
    ref, bound = paged_attention_oracle(block_table=table, cache_seqlens=lens, **t, **kw)
    assert out.dtype == t["q"].dtype and torch.equal(out.isnan().cpu(), ref["out"].isnan())  # (a row that is read past what is in it)
    within("out", out.nan_to_num(), ref["out"].nan_to_num(), bound["out"].nan_to_num())
    assert _same(k_cache, ref["k_cache"]) and _same(v_cache, ref["v_cache"])
    return out


# lengths around the positions of a tile, of a page and of several parts; head sizes around those the kernels are made for
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv,dk,dv,page", [(4, 4, 64, 64, 16), (8, 2, 128, 128, 32), (6, 3, 33, 7, 5), (4, 1, 80, 104, 64), (2, 1, 256, 256, 24),
                                                 (16, 1, 16, 130, 128), (20, 1, 100, 36, 1), (40, 2, 8, 200, 7), (3, 3, 1, 1, 3)])
def test_sizes(heads, kv, dk, dv, page, dtype):
    _check(_inputs([0, 1, 15, -1, 16, 31, 32, 33, 100, 257], heads, kv, dk, dv, page, dtype, seed=dk))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,page", [([4999], 64), ([1, 3000, 2047], 16), ([1023, 1024, 1025], 256), ([0], 16), ([-1], 16), ([2500, 0, -1], 7)])
def test_lengths_in_parts(lens, page, dtype):
    _check(_inputs(lens, 4, 2, 64, 64, page, dtype, seed=len(lens), wide=6000 // page))


@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 100, 1000, 10 ** 6])
@pytest.mark.parametrize("page", [16, 48])
def test_windows(window, page):
    _check(_inputs([0, 1, 31, 32, 64, 65, 300, 1500, -1], 4, 2, 64, 40, page, torch.bfloat16, seed=window), window=window)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [None, 20])
def test_the_cache_as_it_is(dtype, window):
    """Without a new token: the sequence ends with the cache, nothing is written, and an empty one gives 0."""
    t, table, lens = _inputs([0, 1, 33, -1, 200], 6, 2, 48, 32, 16, dtype)
    t["k"] = t["v"] = None
    out = _check((t, table, lens), window=window)
    assert torch.count_nonzero(out[0]) == 0 and torch.count_nonzero(out[3]) == 0


def test_scales():
    for scale in (0.0, 1.0, -0.5):
        _check(_inputs([40, 7], 4, 2, 32, 32, 16, torch.float32), scale=scale)


def test_large_scores():
    """Weights of one position only, and scores that differ by more than the exponent's range."""
    t, table, lens = _inputs([100, 33], 4, 2, 64, 64, 16, torch.float32)
    t["q"] *= 60
    _check((t, table, lens), scale=1.0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinite_scores(dtype):
    """A key whose score is minus infinity has no weight; sequences and heads without it do not see it."""
    t, table, lens = _inputs([100, 50], 2, 2, 32, 32, 16, dtype)
    t["q"] = t["q"].abs()
    want = _call(t, table, lens)[0]
    for p in (5, 40, 70):
        t["k_cache"][table[0][p // 16], p % 16, 1] = -float("inf")
    got = _call(t, table, lens)[0]
    assert torch.equal(got[1], want[1]) and torch.equal(got[0, 0], want[0, 0])
    assert bool(got.isfinite().all())
    finite = {**t, "k_cache": t["k_cache"].clone()}
    finite["k_cache"][finite["k_cache"] == -float("inf")] = -1e4 if dtype != torch.float16 else -3e4
    ref, bound = paged_attention_oracle(block_table=table, cache_seqlens=lens, **finite)
    within("out", got, ref["out"], bound["out"])


def test_no_number_stays_in_its_sequence_and_head():
    t, table, lens = _inputs([100, 90], 4, 2, 32, 32, 16, torch.bfloat16)
    want = _call(t, table, lens)[0]
    t["v_cache"][table[0][2], 3, 1, 5] = float("nan")
    t["k_cache"][table[1][1], 3, 0, 5] = float("nan")
    got = _call(t, table, lens)[0]
    assert torch.equal(got[0, :2], want[0, :2]) and torch.equal(got[1, 2:], want[1, 2:])
    assert bool(got[1, :2].isnan().all()) and bool(got[0, 2:, 5].isnan().all())
    other = torch.arange(32) != 5
    assert torch.equal(got[0, 2:][:, other], want[0, 2:][:, other])


def test_pages_that_are_none_and_lengths_beyond_the_table():
    t, table, _ = _inputs([100, 100, 100, 100], 4, 2, 32, 32, 16, torch.float32)
    table[0][2], table[1][0], table[2] = -1, 2 ** 31 - 1, [-7] * len(table[2])
    _check((t, table, [100, 90, 60, 5000]))
    _check((t, table, [40, 10, 0, len(table[0]) * 16]), window=9)
    t["k"] = t["v"] = None
    out = _check((t, table, [100, 90, 60, 5000]))
    assert torch.count_nonzero(out[2]) == 0


def test_pages_shared_by_sequences_and_named_twice():
    t, table, _ = _inputs([70, 70, 70], 4, 2, 32, 32, 16, torch.bfloat16)
    table[1][:2] = table[0][:2]
    table[2][0] = table[2][1]
    _check((t, table, [70, 50, 64]))


@pytest.mark.parametrize("dtype", DTYPES)
def test_other_layouts(dtype, host):
    """Heads before positions, pages of a larger buffer, keys and values in one, operands by strides."""
    t, table, lens = _inputs([70, 20, 33], 4, 2, 32, 32, 16, dtype)
    want, want_k, want_v = _call(t, table, lens)
    pages = t["k_cache"].shape[0]
    both = torch.zeros(pages + 1, 2, 2, 16, 40, dtype=dtype, device="cuda")
    caches = [both[1:, n, :, :, 3:35].transpose(1, 2) for n in (0, 1)]
    for c, n in zip(caches, ("k_cache", "v_cache")):
        c.copy_(t[n])
    q = torch.empty(4, 3, 32, dtype=dtype, device="cuda").transpose(0, 1).copy_(t["q"])
    k = torch.empty(3, 32, 2, dtype=dtype, device="cuda").transpose(1, 2).copy_(t["k"])
    v = torch.empty(3, 2, 37, dtype=dtype, device="cuda")[..., 1:33].copy_(t["v"])
    wide = torch.full((3, 9), -1, dtype=torch.int32, device="cuda")
    wide[:, 2:2 + len(table[0])] = torch.tensor(table, dtype=torch.int32)
    out = _fn(q, k, v, *caches, wide[:, 2:2 + len(table[0])], torch.tensor(lens, dtype=torch.int32, device="cuda"))
    assert torch.equal(out, want) and _same(caches[0], want_k) and _same(caches[1], want_v)
    assert torch.count_nonzero(both[0]) == 0 and torch.count_nonzero(both[..., :3]) == 0 and torch.count_nonzero(both[..., 35:]) == 0


def test_types_of_tables_and_new_tokens():
    t, table, lens = _inputs([70, 20, 33, -1], 4, 2, 32, 32, 16, torch.bfloat16)
    want = _call(t, table, lens)
    got = _call(t, [[p if p >= 0 else p - 2 ** 32 for p in row] for row in table], [70, 20, 33, -(2 ** 32) + 5], torch.int64)
    assert torch.equal(got[0], want[0]) and _same(got[1], want[1]) and _same(got[2], want[2])
    t["k"], t["v"] = t["k"].float(), t["v"].float()
    assert torch.equal(_call(t, table, lens)[0], want[0])


def test_caches_beyond_32_bit_offsets():
    t, table, lens = _inputs([40, 17], 2, 1, 64, 64, 16, torch.bfloat16)
    want, want_k, want_v = _call(t, table, lens)
    big = torch.zeros(2 ** 31 + 2 ** 21, dtype=torch.bfloat16, device="cuda")
    pages = t["k_cache"].shape[0]
    step = 2 ** 31 // (pages - 1)
    caches = [big.as_strided((pages, 16, 1, 64), (step, 64, 64, 1), offset) for offset in (0, 2 ** 20)]
    for c, n in zip(caches, ("k_cache", "v_cache")):
        c.copy_(t[n])
    out = _fn(t["q"].cuda(), t["k"].cuda(), t["v"].cuda(), *caches, torch.tensor(table, dtype=torch.int32, device="cuda"),
              torch.tensor(lens, dtype=torch.int32, device="cuda"))
    assert torch.equal(out, want) and _same(caches[0], want_k) and _same(caches[1], want_v)


def test_results_repeat_and_host_sides_agree(monkeypatch):
    from mamba_amd import _lib
    inputs = _inputs([3000, 100, 5], 8, 2, 64, 64, 16, torch.bfloat16)
    want = _call(*inputs)
    for _ in range(3):
        assert torch.equal(_call(*inputs)[0], want[0])
    monkeypatch.setattr(_lib, "_torch_ext", None)
    got = _call(*inputs)
    assert torch.equal(got[0], want[0]) and _same(got[1], want[1])


def test_batches_of_none():
    t, table, lens = _inputs([5, 6], 4, 2, 32, 32, 16, torch.float32)
    d = {k: v.cuda() for k, v in t.items()}
    table, lens = torch.tensor(table, dtype=torch.int32, device="cuda"), torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = _fn(d["q"][:0], d["k"][:0], d["v"][:0], d["k_cache"], d["v_cache"], table[:0], lens[:0])
    assert out.shape == (0, 4, 32)


def test_the_caches_have_a_new_version(host):
    t, table, lens = _inputs([5, 6], 4, 2, 32, 32, 16, torch.float32)
    d = {k: v.cuda() for k, v in t.items()}
    at = torch.tensor(table, dtype=torch.int32, device="cuda"), torch.tensor(lens, dtype=torch.int32, device="cuda")
    versions = [d[n]._version for n in ("k_cache", "v_cache")]
    _fn(**d, block_table=at[0], cache_seqlens=at[1])
    assert [d[n]._version for n in ("k_cache", "v_cache")] == [v + 1 for v in versions]
    _fn(d["q"], None, None, d["k_cache"], d["v_cache"], *at)
    assert [d[n]._version for n in ("k_cache", "v_cache")] == [v + 1 for v in versions]


@pytest.mark.parametrize("which", ["q", "k", "v"])
def test_a_gradient_is_refused_not_dropped(host, which):
    t, table, lens = _inputs([5, 6], 4, 2, 32, 32, 16, torch.float32)
    d = {k: v.cuda() for k, v in t.items()}
    d[which].requires_grad_()
    at = torch.tensor(table, dtype=torch.int32, device="cuda"), torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = _fn(**d, block_table=at[0], cache_seqlens=at[1])
    assert out.requires_grad
    with pytest.raises(RuntimeError, match="no gradients"):
        out.sum().backward()
    with torch.no_grad():
        assert not _fn(**d, block_table=at[0], cache_seqlens=at[1]).requires_grad


def test_caches_that_want_gradients_are_refused(host):
    t, table, lens = _inputs([5, 6], 4, 2, 32, 32, 16, torch.float32)
    d = {k: v.cuda() for k, v in t.items()}
    d["v_cache"].requires_grad_()
    at = torch.tensor(table, dtype=torch.int32, device="cuda"), torch.tensor(lens, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="takes no gradients"):
        _fn(**d, block_table=at[0], cache_seqlens=at[1])
    out = _fn(d["q"], None, None, d["k_cache"], d["v_cache"], *at)
    with pytest.raises(RuntimeError, match="no gradients"):
        out.sum().backward()


def test_transforms_are_refused_and_traces_replay(host):
    import torch.autograd.forward_ad as fwAD
    t, table, lens = _inputs([5, 6], 4, 2, 32, 32, 16, torch.float32)
    d = {k: v.cuda().nan_to_num() for k, v in t.items()}
    at = torch.tensor(table, dtype=torch.int32, device="cuda"), torch.tensor(lens, dtype=torch.int32, device="cuda")
    call = lambda q, k: _fn(q, k, d["v"], d["k_cache"], d["v_cache"], *at)
    with fwAD.dual_level(), pytest.raises(NotImplementedError):
        call(fwAD.make_dual(d["q"], torch.ones_like(d["q"])), d["k"])
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda s: call(d["q"], d["k"]) + s)(torch.zeros(2, 1, device="cuda"))
    with torch.no_grad():
        traced = torch.jit.trace(call, (d["q"], d["k"]), check_trace=False)
        for seed in range(3):
            q, k = torch.randn_like(d["q"]), torch.randn_like(d["k"])
            assert torch.equal(traced(q, k), call(q, k))


def test_calls_in_a_captured_graph():
    """A graph that is replayed while the sequences grow, one of them into its next page, and places empty and fill."""
    t, table, _ = _inputs([2000, 90, 33], 4, 2, 64, 64, 16, torch.bfloat16)
    d = {k: v.cuda().nan_to_num() for k, v in t.items()}
    table = torch.tensor(table, dtype=torch.int32, device="cuda").clamp(0, len(t["k_cache"]) - 1)
    lens = torch.zeros(3, dtype=torch.int32, device="cuda")
    other = [d[n].clone() for n in ("k_cache", "v_cache")]
    call = lambda: _fn(**d, block_table=table, cache_seqlens=lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    lens.fill_(-1)
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for n, now in enumerate([[1999, 88, 15], [2000, 89, 16], [0, -1, 17], [1500, 90, 18]]):
        lens.copy_(torch.tensor(now))
        d["q"].copy_(torch.randn(d["q"].shape, generator=torch.Generator().manual_seed(n)))
        d["k"].copy_(torch.randn(d["k"].shape, generator=torch.Generator().manual_seed(n + 10)))
        graph.replay()
        want = _fn(d["q"], d["k"], d["v"], *other, table, lens)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(d["k_cache"], other[0]) and torch.equal(d["v_cache"], other[1])


def test_two_streams_at_once():
    calls = [_inputs([3000, 50], 4, 1, 64, 64, 16, torch.bfloat16, seed=s) for s in range(2)]
    want = [_call(*c)[0] for c in calls]
    ready = [({k: v.cuda() for k, v in t.items()}, torch.tensor(table, dtype=torch.int32, device="cuda"),
              torch.tensor(lens, dtype=torch.int32, device="cuda")) for t, table, lens in calls]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for n, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[n].append(_fn(**ready[n][0], block_table=ready[n][1], cache_seqlens=ready[n][2]))
    torch.cuda.synchronize()
    for n in range(2):
        assert all(torch.equal(g, want[n]) for g in got[n])
