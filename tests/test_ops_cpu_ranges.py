"""Transformer-layer operators without a GPU: refusals at the ends of their ranges, decided from the arguments alone."""
import ctypes as C
import os
import random
import re
import subprocess

import numpy as np
import pytest

from dorado_amd import capi, ops
from tests.test_ops_cpu import ATTN, NORM, ROPE, call


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


def bytes_of(base, run, *dims):
    at = np.array([base], dtype=np.int64)
    for n, s in dims:
        at = (at[:, None] + np.arange(n) * s).reshape(-1)
    return np.unique((at[:, None] + np.arange(run)).reshape(-1))


def on_no_device(which, base, **change):
    """The entry point's refusal, or None: device 99 stops a call that is not refused before anything is launched."""
    flat = []
    for v in {**base, **change}.values():
        flat += list(v) if isinstance(v, tuple) else [v]
    rc = ops._entry()[which](99, 0, (ops._NORM_ARGS, ops._ROPE_ARGS, ops._ATTN_ARGS)[which].pack(*flat))
    text = capi.lib().mibc_last_error(None).decode()
    assert rc == -2 or (rc == -1 and "overlap" in text), (rc, text)
    return text if rc == -1 else None


def test_overlaps_are_refused_wherever_they_lie():
    # random places and layouts (tokens or heads outermost, gaps, neighbours in one buffer) of two tensors, f32: refused wherever a byte
    # is shared, and let through where the bytes are apart and the layouts are those of views of one buffer
    r = random.Random(1)
    shared = apart = 0
    for _ in range(4000):
        b, n, h, d = r.randint(1, 3), r.randint(1, 4), r.randint(1, 3), 2 * r.randint(1, 2)
        room = h + r.randint(0, 3)                          # heads of the buffer
        strides = (n * room * d, room * d, d) if r.random() < 0.5 else (n * room * d, d, n * d)
        if r.random() < 0.3:
            strides = tuple(s * 2 for s in strides)
        off = r.choice([0, strides[2] * r.randint(0, room), strides[1] * r.randint(-2, 2), strides[0] * r.randint(-2, 2), 2 * r.randint(-40, 40), 10**4])
        other = strides if r.random() < 0.7 else (n * h * d, h * d, d)
        x, o = 1 << 20, (1 << 20) + 4 * off
        dims = [(b, strides), (n, strides), (h, strides)]
        mine = bytes_of(x, 4 * d, *[(m, 4 * strides[i]) for i, (m, _) in enumerate(dims)])
        theirs = bytes_of(o, 4 * d, *[(m, 4 * other[i]) for i, (m, _) in enumerate(dims)])
        said = on_no_device(1, ROPE, x0=x, out0=o, freqs=1 << 30, batch=b, tokens=n, h0=h, head_dim=d, rot_dim=d, type=2, xs=strides + (0, 0, 0), os=other + (0, 0, 0))
        same = off == 0 and all(m == 1 or other[i] == strides[i] for i, (m, _) in enumerate(dims))
        touch = np.intersect1d(mine, theirs).size > 0
        if touch and not same:
            shared += 1
            assert said is not None, (b, n, h, d, strides, other, off)
        elif other == strides and off % strides[2] == 0 and (off == 0 or not touch):
            apart += 1
            assert said is None, (b, n, h, d, strides, off)
    assert shared > 500 and apart > 500


N, B = 1 << 20, 128          # an address, and the bytes of a row of NORM


@pytest.mark.parametrize("change,refused", [
    (dict(), False), (dict(out=N + 4 * B), False), (dict(out=N + B), True), (dict(out=N - B), True), (dict(out=N + 2), True), (dict(out=N + 4 * B - 2), True),
    (dict(x_stride=128, out_stride=128, out=N + B), False), (dict(x_stride=128, out_stride=128, out=N + B + 2), True), (dict(out_stride=128), True),
    (dict(residual=N, residual_stride=64), False), (dict(residual=N + B, residual_stride=64), True), (dict(residual=N + 8 * B, residual_stride=0), False),
    (dict(residual=N, residual_stride=0), True), (dict(x=N + 8 * B, residual=N, residual_stride=64, sum_out=N + 8 * B, sum_stride=64), False),
    (dict(sum_out=N, sum_stride=64), True), (dict(weight=N + B), True), (dict(weight=N + 4 * B), False), (dict(weight=N + 4 * B - 4, weight_type=2), True),
    (dict(out_type=3, scale_out=N + 8 * B, scale_stride=1, out=N), True), (dict(out_type=3, scale_out=N + 8 * B, scale_stride=1, out=N + 4 * B), False),
    (dict(out_type=3, scale_out=N + 4 * B + 8, scale_stride=1, out=N + 4 * B), True), (dict(out_type=3, scale_out=N + 8, scale_stride=1, out=N + 4 * B), True)])
def test_rms_norm_overlaps(change, refused):
    assert (on_no_device(0, {**NORM, "x": N, "out": N}, **change) is not None) == refused


F = 1 << 30


@pytest.mark.parametrize("change,refused", [
    (dict(), False), (dict(x1=N + 256, out1=N + 256, h1=2), False), (dict(x1=N + 256, out1=N + 128, h1=2), True), (dict(x1=N, out1=N + 256, h1=2), True),
    (dict(x1=N + 256, out1=N, h1=2), True), (dict(freqs=N + 512), True), (dict(freqs=N + 256), False), (dict(freqs=N + 128), True), (dict(positions=N + 64), True), (dict(positions=N + 4096), False)])
def test_rope_overlaps(change, refused):
    # q and k beside one another in rows of four heads of 64, f16
    base = {**ROPE, "x0": N, "out0": N, "freqs": F, "xs": (1024, 256, 64, 1024, 256, 64), "os": (1024, 256, 64, 1024, 256, 64)}
    assert (on_no_device(1, base, **change) is not None) == refused


@pytest.mark.parametrize("change,refused", [
    (dict(), False), (dict(out=N + 128), True), (dict(out=N + 1536), False), (dict(out=N + 256), False), (dict(out=N + 384), True), (dict(out=N + 512), True), (dict(out=N + 640), True),
    (dict(out=N + 2048 * 16, out_stride=(1024, 128, 64)), False), (dict(out=N + 2048 * 15, out_stride=(1024, 128, 64)), True), (dict(lse=N + 2048 * 16), False),
    (dict(lse=N + 2048 * 15 + 1276), True), (dict(lse=N + 2048 * 15 + 1280), False), (dict(lse=F, slopes=F), True), (dict(lse=F, slopes=F + 2 * 2 * 8 * 4), False), (dict(k_len=N), True),
    (dict(q_tokens=1, k_tokens=1 << 14, k=F, v=F + (1 << 28), workspace=F + (1 << 29), workspace_bytes=1 << 40), False),
    (dict(q_tokens=1, k_tokens=1 << 14, k=F, v=F + (1 << 28), workspace=F + (1 << 28), workspace_bytes=1 << 40), True),
    (dict(q_tokens=1, k_tokens=1 << 14, k=F, v=F + (1 << 28), workspace=N - 256, workspace_bytes=1 << 40), True)])
def test_attention_overlaps(change, refused):
    # q, k, v of two heads of 64 each beside one another in rows of 1024 elements, 16 rows
    wide = (8192, 1024, 64)
    base = {**ATTN, "q": N, "k": N + 512, "v": N + 1024, "out": N, "q_stride": wide, "k_stride": wide, "v_stride": wide, "out_stride": wide}
    assert (on_no_device(2, base, **change) is not None) == refused


def test_outputs_that_overlap_themselves_are_refused():
    # strides of at least a head each, as the sizes allow: refused wherever two of the output's heads share a byte, views of one buffer not
    r = random.Random(2)
    bad = good = 0
    for _ in range(3000):
        b, n, h, d = r.randint(1, 3), r.randint(1, 4), r.randint(1, 4), 2
        if r.random() < 0.5:
            dense = [(r.randint(m, m + 2), i) for i, m in enumerate((b, n, h))]
            r.shuffle(dense)
            strides, step = [0, 0, 0], d + 2 * r.randint(0, 1)
            for m, i in dense:
                strides[i] = step
                step *= m
        else:
            dense, strides = None, [2 * r.randint(1, 14) for _ in range(3)]
        x = bytes_of(0, 4 * d, *[(m, 4 * s) for m, s in zip((b, n, h), strides)])
        touch = x.size < 4 * d * b * n * h
        said = on_no_device(1, ROPE, x0=1 << 28, out0=1 << 20, freqs=1 << 30, batch=b, tokens=n, h0=h, head_dim=d, rot_dim=d, type=2,
                            xs=(n * h * d, h * d, d, 0, 0, 0), os=tuple(strides) + (0, 0, 0))
        if touch:
            bad += 1
            assert said is not None, (b, n, h, strides)
        elif dense is not None:
            good += 1
            assert said is None, (b, n, h, strides)
    assert bad > 300 and good > 500
    said = on_no_device(2, ATTN, q=1 << 28, k=1 << 29, v=1 << 30, out=1 << 20, out_stride=(1024, 64, 64))
    assert said == "attention: output heads overlap"
