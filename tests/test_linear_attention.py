"""What linear_attention_fn, linear_attention_state_update and paged_attention_update refuse, and their C entry points' argument
checks (no GPU)."""
import ctypes
import os
import subprocess
import tempfile

import pytest
import torch

from mamba_amd import _lib
from mamba_amd.ops.linear_attention import linear_attention_fn, linear_attention_state_update
from mamba_amd.ops.paged_attention import paged_attention_update

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "mamba_hip.h")
Z = torch.zeros
INT = lambda *v: torch.tensor(v, dtype=torch.int32)


def _linear(**changes):
    a = dict(q=Z(1, 6, 4, 8), k=Z(1, 6, 2, 8), v=Z(1, 6, 2, 5), log_decay=Z(4))
    return linear_attention_fn(**{**a, **changes})


def _step(**changes):
    a = dict(state=Z(3, 4, 8, 5), q=Z(2, 4, 8), k=Z(2, 2, 8), v=Z(2, 2, 5), log_decay=Z(4))
    return linear_attention_state_update(**{**a, **changes})


def _paged(**changes):
    a = dict(q=Z(2, 4, 8), k=Z(2, 2, 8), v=Z(2, 2, 5), k_cache=Z(7, 4, 2, 8), v_cache=Z(7, 4, 2, 5), block_table=INT([0, 1], [2, 3]),
             cache_seqlens=INT(3, 5))
    return paged_attention_update(**{**a, **changes})


@pytest.mark.parametrize("call,changes,kind,text", [
    (_linear, {}, RuntimeError, "no CPU fallback"),
    (_linear, dict(cu_seqlens=INT(0, 6)), RuntimeError, "no CPU fallback"),
    (_linear, dict(q=Z(6, 4, 8)), RuntimeError, "q must be"),
    (_linear, dict(q=Z(1, 6, 4, 8, dtype=torch.float64)), RuntimeError, "q must be"),
    (_linear, dict(k=Z(1, 5, 2, 8)), RuntimeError, "k must be"),
    (_linear, dict(v=Z(1, 6, 2)), RuntimeError, "v must be"),
    (_linear, dict(k=Z(1, 6, 2, 8, dtype=torch.int32)), RuntimeError, "k must be"),
    (_linear, dict(k=Z(1, 6, 2, 7)), RuntimeError, "same head size"),
    (_linear, dict(k=Z(1, 6, 1, 8)), RuntimeError, "same number of heads"),
    (_linear, dict(k=Z(1, 6, 3, 8), v=Z(1, 6, 3, 5)), RuntimeError, "must divide"),
    (_linear, dict(k=Z(1, 6, 0, 8), v=Z(1, 6, 0, 5)), RuntimeError, "must divide"),
    (_linear, dict(v=Z(1, 6, 2, 257)), RuntimeError, "head sizes of 1 to 256"),
    (_linear, dict(v=Z(1, 6, 2, 0)), RuntimeError, "head sizes of 1 to 256"),
    (_linear, dict(log_decay=Z(5)), RuntimeError, "log_decay must be"),
    (_linear, dict(log_decay=Z(4, dtype=torch.float64)), RuntimeError, "log_decay must be"),
    (_linear, dict(log_decay=Z(4).requires_grad_()), RuntimeError, "takes no gradients"),
    (_linear, dict(scale=float("nan")), ValueError, "scale"),
    (_linear, dict(scale=float("inf")), ValueError, "scale"),
    (_linear, dict(initial_states=Z(2, 4, 8, 5)), RuntimeError, "initial_states"),
    (_linear, dict(cu_seqlens=INT(0, 3, 6), initial_states=Z(1, 4, 8, 5)), RuntimeError, "initial_states"),
    (_linear, dict(cu_seqlens=INT(0)), RuntimeError, "cu_seqlens"),
    (_linear, dict(cu_seqlens=torch.tensor([0.0, 6.0])), RuntimeError, "cu_seqlens"),
    (_linear, dict(q=Z(2, 6, 4, 8), k=Z(2, 6, 2, 8), v=Z(2, 6, 2, 5), cu_seqlens=INT(0, 6)), RuntimeError, "batch 1"),
    (_step, {}, RuntimeError, "no CPU fallback"),
    (_step, dict(q=Z(2, 4, 8, 1)), RuntimeError, "q must be"),
    (_step, dict(k=Z(1, 2, 8)), RuntimeError, "k must be"),
    (_step, dict(state=Z(3, 4, 5, 8)), RuntimeError, "state must be"),
    (_step, dict(state=Z(3, 4, 8, 5, dtype=torch.float64)), RuntimeError, "state must be"),
    (_step, dict(state=Z(1, 4, 8, 5)), RuntimeError, "rows"),
    (_step, dict(state=Z(3, 4, 5, 8).transpose(2, 3)), RuntimeError, "contiguous"),
    (_step, dict(state=Z(1, 4, 8, 5).expand(3, 4, 8, 5)), RuntimeError, "must not overlap"),
    (_step, dict(state=Z(3, 4, 8, 5).requires_grad_()), RuntimeError, "takes no gradients"),
    (_step, dict(log_decay=Z(3)), RuntimeError, "log_decay"),
    (_step, dict(log_decay=Z(4).requires_grad_()), RuntimeError, "takes no gradients"),
    (_step, dict(scale=float("-inf")), ValueError, "scale"),
    (_step, dict(state_batch_indices=INT(0, 1, 2)), RuntimeError, "state_batch_indices"),
    (_step, dict(state_batch_indices=Z(2)), RuntimeError, "state_batch_indices"),
    (_paged, {}, RuntimeError, "no CPU fallback"),
    (_paged, dict(k=None, v=None), RuntimeError, "no CPU fallback"),
    (_paged, dict(k=None), RuntimeError, "come together"),
    (_paged, dict(q=Z(2, 1, 4, 8)), RuntimeError, "q must be"),
    (_paged, dict(q=Z(2, 1, 4, 8), k=None, v=None), RuntimeError, "q must be"),
    (_paged, dict(q=Z(2, 3, 8)), RuntimeError, "must divide"),
    (_paged, dict(q=Z(2, 3, 8), k=None, v=None), RuntimeError, "must divide"),
    (_paged, dict(k_cache=Z(7, 4, 2, 8, dtype=torch.float16)), RuntimeError, "k_cache must be"),
    (_paged, dict(v_cache=Z(7, 4, 10)), RuntimeError, "v_cache must be"),
    (_paged, dict(v_cache=Z(7, 3, 2, 5)), RuntimeError, "same pages"),
    (_paged, dict(v_cache=Z(7, 4, 2, 6)), RuntimeError, "heads of k and v"),
    (_paged, dict(k_cache=Z(0, 4, 2, 8), v_cache=Z(0, 4, 2, 5)), RuntimeError, "a page at least"),
    (_paged, dict(k_cache=Z(0, 4, 2, 8), v_cache=Z(0, 4, 2, 5), k=None, v=None), RuntimeError, "a page at least"),
    (_paged, dict(k_cache=Z(7, 4, 8, 2).transpose(2, 3)), RuntimeError, "unit stride"),
    (_paged, dict(v_cache=Z(1, 4, 2, 5).expand(7, 4, 2, 5)), RuntimeError, "must not overlap"),
    (_paged, dict(k_cache=Z(7, 4, 2, 8).requires_grad_()), RuntimeError, "takes no gradients"),
    (_paged, dict(block_table=INT(0, 1)), RuntimeError, "block_table"),
    (_paged, dict(block_table=INT([0, 1])), RuntimeError, "block_table"),
    (_paged, dict(block_table=Z(2, 0, dtype=torch.int32)), RuntimeError, "block_table"),
    (_paged, dict(block_table=Z(2, 2)), RuntimeError, "block_table"),
    (_paged, dict(block_table=INT([0], [1]).expand(2, 2 ** 29)), RuntimeError, "2\\^30 positions"),
    (_paged, dict(cache_seqlens=INT(3)), RuntimeError, "cache_seqlens"),
    (_paged, dict(cache_seqlens=Z(2)), RuntimeError, "cache_seqlens"),
    (_paged, dict(scale=float("nan")), ValueError, "scale"),
    (_paged, dict(window=0), ValueError, "window"),
    (_paged, dict(window=-1), ValueError, "window"),
])
def test_refusals(call, changes, kind, text):
    with pytest.raises(kind, match=text):
        call(**changes)


@pytest.mark.parametrize("name", ["LinearAttnParams", "LinearAttnStepParams", "PagedAttnParams"])
def test_ctypes_structs_match_c_layout(name):
    cls = getattr(_lib, name)
    fields = [f[0] for f in cls._fields_]
    prog = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{HEADER}"', "int main(void){",
            f'printf("%zu\\n", sizeof({name}));']
    prog += [f'printf("%zu\\n", offsetof({name}, {f}));' for f in fields] + ["return 0;}"]
    with tempfile.TemporaryDirectory() as d:
        src, exe = os.path.join(d, "t.c"), os.path.join(d, "t")
        open(src, "w").write("\n".join(prog))
        subprocess.run(["gcc", "-std=c99", src, "-o", exe], check=True)
        vals = [int(v) for v in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    assert vals[0] == ctypes.sizeof(cls)
    for f, off in zip(fields, vals[1:]):
        assert getattr(cls, f).offset == off, f"{name}.{f}"


def _filled(cls, ints, pointers):
    p = cls()
    for k, v in ints.items():
        setattr(p, k, v)
    for k in pointers:
        setattr(p, k, 256)  # stand-ins: the checks below run before any launch
    return p


LINEAR = dict(ints=dict(batch=1, seqlen=4, nheads=4, nkvheads=2, headdim_k=8, headdim_v=8, scale=1.0),
              pointers=["q", "k", "v", "log_decay", "out", "ws", "dout", "dq", "dk", "dv"])
STEP = dict(ints=dict(batch=2, nheads=4, nkvheads=2, headdim_k=8, headdim_v=8, state_rows=2, scale=1.0),
            pointers=["state", "q", "k", "v", "log_decay", "out"])
PAGED = dict(ints=dict(batch=2, nheads=4, nkvheads=2, headdim_k=8, headdim_v=8, num_pages=3, page_size=4, max_pages=2, nsplit=1, scale=1.0),
             pointers=["q", "k", "v", "k_cache", "v_cache", "block_table", "cache_seqlens", "out"])
HEADS = [dict(batch=0), dict(nheads=0), dict(nkvheads=0), dict(nkvheads=3), dict(headdim_k=0), dict(headdim_v=-1), dict(dtype=3), dict(dtype=-1),
         dict(scale=float("nan")), dict(scale=float("inf"))]


@pytest.mark.parametrize("fn,cls,base,changes,code", [
    *[("linear_attn_fwd", "LinearAttnParams", LINEAR, c, -1) for c in (
        *HEADS, dict(seqlen=0), dict(nseq=-1), dict(nseq=2), dict(cu_seqlens=256), dict(batch=2, nseq=1, cu_seqlens=256), dict(q=None),
        dict(k=None), dict(v=None), dict(log_decay=None), dict(out=None))],
    *[("linear_attn_fwd", "LinearAttnParams", LINEAR, c, -2) for c in (dict(headdim_k=257), dict(headdim_v=257), dict(seqlen=2 ** 30 + 1))],
    *[("linear_attn_bwd", "LinearAttnParams", LINEAR, c, -1) for c in (
        dict(dout=None), dict(dq=None), dict(dk=None), dict(dv=None), dict(ws=None), dict(ws=8))],
    *[("linear_attn_fwd_ws_bytes", "LinearAttnParams", LINEAR, c, -1) for c in HEADS],
    *[("linear_attn_state_update", "LinearAttnStepParams", STEP, c, -1) for c in (
        *HEADS, dict(state_rows=0), dict(state_rows=1), dict(state_dtype=3), dict(state=None), dict(q=None), dict(k=None), dict(v=None),
        dict(log_decay=None), dict(out=None))],
    *[("linear_attn_state_update", "LinearAttnStepParams", STEP, c, -2) for c in (dict(headdim_k=257), dict(nheads=65538))],
    *[("paged_attn_update", "PagedAttnParams", PAGED, c, -1) for c in (
        *HEADS, dict(num_pages=0), dict(page_size=0), dict(max_pages=0), dict(window=-1), dict(nsplit=0), dict(nsplit=65536), dict(nsplit=2),
        dict(nsplit=2, ws=8), dict(q=None), dict(k=None), dict(v=None), dict(k_cache=None), dict(v_cache=None), dict(block_table=None),
        dict(cache_seqlens=None), dict(out=None))],
    *[("paged_attn_update", "PagedAttnParams", PAGED, c, -2) for c in (
        dict(headdim_v=300), dict(max_pages=2 ** 29), dict(batch=65536))],
    *[("paged_attn_parts", "PagedAttnParams", PAGED, c, -1) for c in HEADS],
    ("paged_attn_ws_bytes", "PagedAttnParams", PAGED, dict(nsplit=0), -1),
])
def test_c_entry_points_refuse(fn, cls, base, changes, code):
    p = _filled(getattr(_lib, cls), **base)
    for k, v in changes.items():
        setattr(p, k, v)
    fn = getattr(_lib.load(), fn)
    assert (fn(p, None) if len(fn.argtypes) == 2 else fn(p)) == code


def test_c_entry_points_without_a_struct():
    lib = _lib.load()
    for fn in ("linear_attn_fwd", "linear_attn_bwd", "linear_attn_state_update", "paged_attn_update"):
        assert getattr(lib, fn)(None, None) == -1
    for fn in ("linear_attn_fwd_ws_bytes", "linear_attn_bwd_ws_bytes", "paged_attn_parts", "paged_attn_ws_bytes"):
        assert getattr(lib, fn)(None) == -1
