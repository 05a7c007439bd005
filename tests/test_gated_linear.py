"""What gated_linear_scan_fn, gated_linear_state_update and block_norm_fn refuse, and their C entry points' argument checks
(no GPU)."""
import ctypes
import os
import subprocess
import tempfile

import pytest
import torch

from mamba_amd import _lib
from mamba_amd.ops.block_norm import block_norm_fn
from mamba_amd.ops.gated_linear_scan import gated_linear_scan_fn, gated_linear_state_update

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "mamba_hip.h")


def _scan(**changes):
    a = dict(x=torch.zeros(1, 6, 4), gate_a=torch.zeros(1, 6, 4), gate_x=torch.zeros(1, 6, 4), decay=torch.zeros(4))
    return gated_linear_scan_fn(**{**a, **changes})


def _step(**changes):
    a = dict(state=torch.zeros(3, 4), x=torch.zeros(2, 4), gate_a=torch.zeros(2, 4), gate_x=torch.zeros(2, 4), decay=torch.zeros(4))
    return gated_linear_state_update(**{**a, **changes})


def _norm(**changes):
    a = dict(x=torch.zeros(2, 4), residual=torch.zeros(2, 4), norm_weight=torch.ones(4), next_weight=torch.ones(4))
    return block_norm_fn(**{**a, **changes})


Z = torch.zeros


@pytest.mark.parametrize("call,changes,kind,text", [
    (_scan, {}, RuntimeError, "no CPU fallback"),
    (_scan, dict(x=Z(6, 4)), RuntimeError, "x must be"),
    (_scan, dict(x=Z(1, 6, 4, dtype=torch.float64)), RuntimeError, "x must be"),
    (_scan, dict(gate_a=Z(1, 5, 4)), RuntimeError, "gate_a must have x's shape"),
    (_scan, dict(gate_x=Z(1, 6, 1)), RuntimeError, "gate_x must have x's shape"),
    (_scan, dict(decay=Z(5)), RuntimeError, "decay must be"),
    (_scan, dict(decay=Z(4, dtype=torch.float64)), RuntimeError, "decay must be"),
    (_scan, dict(rate=-1.0), ValueError, "rate"),
    (_scan, dict(rate=float("nan")), ValueError, "rate"),
    (_scan, dict(rate=float("inf")), ValueError, "rate"),
    (_scan, dict(initial_states=Z(2, 4)), RuntimeError, "initial_states"),
    (_scan, dict(cu_seqlens=torch.tensor([0, 6], dtype=torch.int32), initial_states=Z(2, 4)), RuntimeError, "initial_states"),
    (_scan, dict(cu_seqlens=torch.tensor([0], dtype=torch.int32)), RuntimeError, "cu_seqlens"),
    (_scan, dict(cu_seqlens=torch.tensor([0.0, 6.0])), RuntimeError, "cu_seqlens"),
    (_scan, dict(x=Z(2, 6, 4), gate_a=Z(2, 6, 4), gate_x=Z(2, 6, 4), cu_seqlens=torch.tensor([0, 6], dtype=torch.int32)),
     RuntimeError, "batch 1"),
    (_scan, dict(cu_seqlens=torch.tensor([0, 6], dtype=torch.int32)), RuntimeError, "no CPU fallback"),
    (_step, {}, RuntimeError, "no CPU fallback"),
    (_step, dict(state=Z(1, 4)), RuntimeError, "rows"),
    (_step, dict(state=Z(3, 5)), RuntimeError, "state must be"),
    (_step, dict(state=Z(3, 4, dtype=torch.float64)), RuntimeError, "fp32, fp16 or bf16"),
    (_step, dict(state=Z(4, 3).t()), RuntimeError, "unit channel stride"),
    (_step, dict(gate_a=Z(1, 4)), RuntimeError, "gate_a"),
    (_step, dict(decay=Z(3)), RuntimeError, "decay"),
    (_step, dict(rate=float("nan")), ValueError, "rate"),
    (_step, dict(state_batch_indices=torch.zeros(3, dtype=torch.int32)), RuntimeError, "state_batch_indices"),
    (_step, dict(state_batch_indices=torch.zeros(2)), RuntimeError, "state_batch_indices"),
    (_norm, {}, RuntimeError, "no CPU fallback"),
    (_norm, dict(x=Z(2, 4, dtype=torch.float64), residual=Z(2, 4, dtype=torch.float64)), RuntimeError, "x must be"),
    (_norm, dict(residual=Z(1, 4)), RuntimeError, "residual must have x's shape"),
    (_norm, dict(z=Z(2, 3)), RuntimeError, "z must have x's shape"),
    (_norm, dict(residual=Z(2, 4, dtype=torch.bfloat16)), RuntimeError, "residual stream"),
    (_norm, dict(norm_weight=torch.ones(3)), RuntimeError, "norm_weight"),
    (_norm, dict(next_bias=torch.ones(1)), RuntimeError, "next_bias"),
    (_norm, dict(scale=torch.ones(1)), RuntimeError, "scale"),
    (_norm, dict(x=Z(2, 0), residual=Z(2, 0)), RuntimeError, "channels"),
    (_norm, dict(x=Z(1, 32769), residual=Z(1, 32769)), RuntimeError, "channels"),
])
def test_refusals(call, changes, kind, text):
    with pytest.raises(kind, match=text):
        call(**changes)


@pytest.mark.parametrize("name", ["GatedScanParams", "GatedStepParams", "NormBlockParams"])
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


SCAN = dict(ints=dict(batch=1, seqlen=4, dim=4), pointers=["x", "gate_a", "gate_x", "decay", "out", "ckpt", "dout", "dx", "dgate_a",
                                                           "dgate_x", "ddecay", "ws"])
STEP = dict(ints=dict(batch=2, dim=4, state_rows=2), pointers=["state", "x", "gate_a", "gate_x", "decay", "out"])
NORM = dict(ints=dict(rows=2, dim=4, nparts=1), pointers=["x", "residual", "norm_weight", "next_weight", "out", "residual_out", "stats",
                                                          "dout", "dx", "dresidual", "dnorm_weight", "dnext_weight", "parts"])


@pytest.mark.parametrize("fn,cls,base,changes", [
    *[("gated_scan_fwd", "GatedScanParams", SCAN, c) for c in (
        dict(batch=0), dict(seqlen=0), dict(dim=-1), dict(nseq=-1), dict(nseq=2), dict(batch=2, nseq=1, cu_seqlens=256), dict(dtype=3),
        dict(decay_dtype=-1), dict(x=None), dict(gate_a=None), dict(gate_x=None), dict(decay=None), dict(ckpt=None), dict(ckpt=8),
        dict(out=None), dict(cu_seqlens=256), dict(rate=-1.0), dict(rate=float("nan")))],
    *[("gated_scan_bwd", "GatedScanParams", SCAN, c) for c in (
        dict(dout=None), dict(dx=None), dict(dgate_a=None), dict(dgate_x=None), dict(ddecay=None), dict(ws=None), dict(ws=8))],
    *[("gated_state_update", "GatedStepParams", STEP, c) for c in (
        dict(batch=0), dict(dim=0), dict(state_rows=0), dict(state_rows=1), dict(dtype=7), dict(state_dtype=3), dict(decay_dtype=3),
        dict(state=None), dict(x=None), dict(gate_a=None), dict(gate_x=None), dict(decay=None), dict(out=None), dict(rate=-1.0))],
    *[("norm_block_fwd", "NormBlockParams", NORM, c) for c in (
        dict(rows=0), dict(dim=0), dict(dtype=3), dict(weight_dtype=4), dict(x=None), dict(residual=None), dict(norm_weight=None),
        dict(next_weight=None), dict(out=None), dict(residual_out=None), dict(stats=8))],
    *[("norm_block_bwd", "NormBlockParams", NORM, c) for c in (
        dict(stats=None), dict(dout=None), dict(dx=None), dict(dresidual=None), dict(dnorm_weight=None), dict(dnext_weight=None),
        dict(parts=None), dict(nparts=0), dict(nparts=65537), dict(z=256), dict(dz=256), dict(scale=256), dict(dscale=256),
        dict(norm_bias=256), dict(dnext_bias=256))],
])
def test_c_entry_points_refuse(fn, cls, base, changes):
    p = _filled(getattr(_lib, cls), **base)
    for k, v in changes.items():
        setattr(p, k, v)
    assert getattr(_lib.load(), fn)(p, None) == -1


def test_c_entry_points_without_a_struct():
    lib = _lib.load()
    for fn in ("gated_scan_fwd", "gated_scan_bwd", "gated_state_update", "norm_block_fwd", "norm_block_bwd", "gated_scan_ckpt_bytes",
               "gated_scan_bwd_ws_bytes", "norm_block_bwd_nparts"):
        assert getattr(lib, fn)(*([None] if fn.endswith(("bytes", "nparts")) else [None, None])) == -1


def test_c_entry_points_refuse_what_they_do_not_serve():
    lib = _lib.load()
    p = _filled(_lib.NormBlockParams, **NORM)
    p.dim = 32769
    assert lib.norm_block_fwd(p, None) == -2
    p.dim, p.dtype, p.res_dtype = 4, 1, 2      # a bf16 block on an fp16 stream
    assert lib.norm_block_fwd(p, None) == -2


def test_more_workgroups_than_a_launch_takes():
    lib = _lib.load()
    p = _filled(_lib.GatedScanParams, **SCAN)
    p.batch, p.seqlen, p.dim = 2 ** 23 - 1, 1, 1
    assert lib.gated_scan_ckpt_bytes(p) > 0 and lib.gated_scan_bwd_ws_bytes(p) > 0
    p.batch += 1                                # 2^32 threads
    assert lib.gated_scan_ckpt_bytes(p) == lib.gated_scan_bwd_ws_bytes(p) == lib.gated_scan_fwd(p, None) == lib.gated_scan_bwd(p, None) == -2


BIG = torch.zeros(1, dtype=torch.bfloat16)


@pytest.mark.parametrize("call", [
    lambda: gated_linear_scan_fn(*[BIG.expand(2 ** 31, 1, 1)] * 3, BIG),
    lambda: gated_linear_scan_fn(*[BIG.expand(1, 2 ** 31, 1)] * 3, BIG),
    lambda: gated_linear_state_update(torch.zeros(1, 1), *[BIG.expand(2 ** 31, 1)] * 3, BIG, state_batch_indices=BIG),
    lambda: block_norm_fn(*[BIG.expand(2 ** 31, 1)] * 2, BIG, BIG)])
def test_sizes_beyond_32_bits(call):
    with pytest.raises(RuntimeError, match="counted in 32 bits"):
        call()


def test_overlapping_state_rows():
    with pytest.raises(RuntimeError, match="must not overlap"):
        _step(state=Z(1, 4).expand(3, 4))
    with pytest.raises(RuntimeError, match="must not overlap"):
        _step(state=Z(9).as_strided((3, 4), (2, 1)))
