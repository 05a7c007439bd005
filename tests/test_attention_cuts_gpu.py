"""linear_attention_fn and paged_attention_update at the sizes where they change how they divide their work, against the 64-bit
oracle: rows in one piece and in segments, one or two tiles a wave, ranges of a batch and a workgroup a sequence, rows far apart."""
import pytest
import torch

from oracle.linear_attention import linear_attention_oracle, within
from test_linear_attention_gpu import _check as _check_linear, _inputs as _linear_inputs, _run as _run_linear
from test_paged_attention_gpu import _check as _check_paged, _inputs as _paged_inputs

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("batch,L,heads,kv,dk,dv,dtype", [
    (5, 900, 8, 8, 128, 128, torch.bfloat16),  # two tiles a wave, seven segments
    (5, 901, 8, 4, 112, 96, torch.float16),    # the same in part of the columns, heads that share
    (4, 131, 128, 128, 128, 100, torch.bfloat16),  # two tiles, whole rows
    (3, 259, 40, 20, 96, 128, torch.float16),
    (2, 700, 6, 2, 33, 50, torch.bfloat16),    # shared heads of odd sizes, in segments
    (1, 300, 6, 3, 6, 10, torch.float32)])
def test_rows(batch, L, heads, kv, dk, dv, dtype):
    _check_linear(_linear_inputs(batch, L, heads, dk, dv, dtype, kv=kv, seed=L))


@pytest.mark.parametrize("heads,kv,dk,dv,dtype", [(16, 8, 112, 96, torch.bfloat16), (16, 16, 128, 128, torch.float16), (16, 4, 64, 64, torch.bfloat16)])
def test_packed_rows(heads, kv, dk, dv, dtype):
    cu = [3, 131, 131, 1500, 1501, 2777, 2778, 4090]
    _check_linear(_linear_inputs(1, 4100, heads, dk, dv, dtype, kv=kv, seed=dk, seqs=len(cu) - 1), cu)


@pytest.mark.parametrize("stride", [1 << 22, (1 << 22) + 8])
def test_rows_far_apart(stride):
    """On both sides of the largest distance that 32-bit places of a lane reach.  (Rows beyond it are walked block by block with
    weights f^(a + b) where the others have f^a f^b, two roundings of 2^-24 more: the oracle's bounds hold both, which are not the
    same bit for bit.)"""
    t = _linear_inputs(1, 130, 2, 32, 32, torch.bfloat16, states=False)
    wide = torch.empty(130 * stride + 64, dtype=torch.bfloat16, device="cuda")
    ref, bound = linear_attention_oracle(t["q"], t["k"], t["v"], t["log_decay"], None, None, None, t["dout"], None)
    for n in ("q", "k", "v", "dout"):
        far = wide.as_strided(t[n].shape, (130 * stride, stride, 32, 1))
        far.copy_(t[n])
        for name, v in _run_linear({**t, n: far}).items():
            within(name, v, ref[name], bound[name])


def _lens(n, most, seed):
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(0, most, (n,), generator=g)
    lens[torch.randint(0, n, (n // 10,), generator=g)] = -1
    return lens.tolist()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,most,heads,kv,dk,dv,page,wide", [
    (150, 700, 2, 1, 64, 64, 16, 60),       # ranges with one sequence and with many, lengths read 64 at a time
    (130, 40, 4, 2, 32, 32, 8, 100),        # many sequences a range
    (260, 300, 16, 8, 104, 120, 32, 12),    # a workgroup a sequence
    (5, 900, 100, 100, 16, 16, 32, 30)])    # more heads than ranges
def test_batches(batch, most, heads, kv, dk, dv, page, wide, dtype):
    _check_paged(_paged_inputs(_lens(batch, most, batch), heads, kv, dk, dv, page, dtype, wide=wide, seed=batch))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv,dk,dv", [(4, 2, 96, 72), (6, 3, 65, 95), (20, 1, 88, 96), (2, 2, 3, 90)])
def test_heads_of_up_to_96(heads, kv, dk, dv, dtype):
    _check_paged(_paged_inputs([1500, 0, 33, -1, 300], heads, kv, dk, dv, 16, dtype, wide=100, seed=dk))


@pytest.mark.parametrize("window", [40, 500])
def test_windows_in_ranges(window):
    _check_paged(_paged_inputs(_lens(40, 1200, 7), 12, 12, 80, 80, 16, torch.float16, wide=80, seed=window), window=window)
