"""Transformer-layer operators without a GPU: refusals at the ends of their ranges, decided from the arguments alone."""
import ctypes as C
import os
import re
import subprocess

import pytest

from dorado_amd import capi
from tests.test_ops_cpu import ATTN, call


@pytest.mark.parametrize("change", [dict(softcap=1e30, scale=1e-10), dict(softcap=1.0, scale=1e-38), dict(softcap=1e-35, scale=1e5)])
def test_attention_refuses_caps_beyond_f32(change):
    rc, text = call(2, {**ATTN, "out": 1 << 21}, **change)
    assert rc == -1 and "for this scale" in text


@pytest.mark.parametrize("change", [dict(scale=1e-20), dict(softcap=1e-20, scale=1e-10), dict(scale=1e-40, softcap=1e-30)])
def test_attention_refuses_slopes_beyond_f32(change):
    # slope / scale is infinite there, and infinity times a distance of 0 is NaN
    rc, text = call(2, {**ATTN, "out": 1 << 21}, slopes=1 << 22, **change)
    assert rc == -1 and ("slopes need" in text or "for this scale" in text)


@pytest.mark.parametrize("rc,text,seen", [(-2, "attention: out of memory", (-2, "attention: out of memory")), (-1, "rope: null pointer", (-1, "rope: null pointer")),
                                          (1, "attention: head_dim", (1, "tx attention shape")), (0, "old", (0, "old"))])
def test_engine_keeps_an_operators_error(rc, text, seen):
    lib = capi.dbg_lib()
    lib.mibc_last_error.restype = C.c_char_p
    lib.mibc_last_error.argtypes = [C.c_void_p]
    assert (lib.mibc_debug_tx_op_status(rc, text.encode()), lib.mibc_last_error(None).decode()) == seen


def test_nothing_but_the_lds_loads_uses_m0(tmp_path):
    # att_dma16 writes M0 in assembly, which cannot name it as overwritten: the compiler must have no use of its own for it
    csrc = os.path.join(os.path.dirname(capi.LIB_PATH), "csrc")
    make = subprocess.check_output(["make", "-n", "-B", "-C", csrc, "ops_att_32.o"], text=True)
    command = next(line for line in make.splitlines() if "ops_attention_kernels.hip" in line).split()
    jobs = []
    for d in (32, 64, 96, 128):
        out = str(tmp_path / f"{d}.s")
        args = [a.replace("ATT_D=32", f"ATT_D={d}") for a in command[:command.index("-c")]]
        jobs.append((out, subprocess.Popen(args + ["--offload-device-only", "-S", "ops_attention_kernels.hip", "-o", out], cwd=csrc, stderr=subprocess.DEVNULL)))
    for out, job in jobs:
        assert job.wait() == 0
        lines = [line.strip() for line in open(out)]
        at = [i for i, line in enumerate(lines) if re.search(r"\bm0\b", line)]
        assert len(at) == sum("global_load_lds" in line for line in lines) > 100
        for i in at:
            assert re.match(r"s_mov_b32 m0, s\d+$", lines[i]) and lines[i + 1] == "s_nop 0" and lines[i + 2].startswith("global_load_lds_dwordx4")
