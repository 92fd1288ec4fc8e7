"""Transformer-layer operators without a GPU: what the entry points refuse (decided from the arguments alone, before any device
call), the layout of the argument structures, the host-only frequencies, and the 64-bit reference itself."""
import ctypes as C
import math
import os
import re
import subprocess

import pytest
import torch

from dorado_amd import capi, ops
from tests import ops_reference as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20          # a pointer that nothing follows: every case here is refused before a launch
NORM = dict(x=P, residual=0, weight=0, sum_out=0, out=P, scale_out=0, rows=4, x_stride=64, residual_stride=0, sum_stride=0, out_stride=64,
            scale_stride=0, cols=64, type=0, weight_type=0, out_type=0, group=0, alpha=1.0, eps=1e-5, reserved=0)
ROPE = dict(x0=P, x1=0, out0=P, out1=0, positions=0, freqs=P, start=0, xs=(256, 128, 64, 0, 0, 0), os=(256, 128, 64, 0, 0, 0), batch=2, tokens=2,
            h0=2, h1=0, head_dim=64, rot_dim=64, type=0, interleaved=0, positions_64=0, amplitude=1.0)
ATTN = dict(q=P, k=P, v=P, out=P, lse=0, k_len=0, prefix=0, doc_offsets=0, slopes=0, workspace=0, workspace_bytes=0, q_stride=(1024, 128, 64),
            k_stride=(1024, 128, 64), v_stride=(1024, 128, 64), out_stride=(1024, 128, 64), batch=2, heads=2, kv_heads=2, q_tokens=8, k_tokens=8,
            head_dim=64, n_docs=0, type=0, back=-1, ahead=-1, q_start=ops.ATTN_END, scale=0.125, softcap=0.0, reserved=0)


def call(which, base, **change):
    a = {**base, **change}
    flat = []
    for v in a.values():
        flat += list(v) if isinstance(v, tuple) else [v]
    s = (ops._NORM_ARGS, ops._ROPE_ARGS, ops._ATTN_ARGS)[which]
    return ops._entry()[which](0, 0, s.pack(*flat)), capi.lib().mibc_last_error(None).decode()


def test_structures_match_the_header(tmp_path):
    hdr = os.path.join(ROOT, "include", "mibc.h")
    names = {"mibc_rms_norm_args": ops._NORM_ARGS, "mibc_rope_args": ops._ROPE_ARGS, "mibc_attention_args": ops._ATTN_ARGS}
    src = tmp_path / "s.c"
    src.write_text('#include "%s"\n#include <stdio.h>\nint main(void){%s return 0;}\n' %
                   (hdr, "".join('printf("%%zu\\n", sizeof(%s));' % n for n in names)))
    subprocess.check_call(["gcc", "-std=c99", "-o", str(tmp_path / "s"), str(src)])
    sizes = [int(x) for x in subprocess.check_output([str(tmp_path / "s")]).split()]
    assert sizes == [s.size for s in names.values()]
    text = open(hdr).read()
    assert ops.ATTN_END == -2147483647 - 1 and re.search(r"#define MIBC_ATTN_END \(-2147483647 - 1\)", text)


@pytest.mark.parametrize("change,code", [
    (dict(type=3), 1), (dict(type=9), 1), (dict(cols=0), -1), (dict(cols=-5), -1), (dict(rows=-1), -1), (dict(cols=32769, x_stride=32769, out_stride=32769), 1),
    (dict(rows=1 << 31), 1), (dict(weight=P, weight_type=1), 1), (dict(out_type=1), 1), (dict(out_type=7), 1), (dict(group=32), -1),
    (dict(out_type=3, scale_out=P, scale_stride=1, group=16), 1), (dict(out_type=3, scale_out=P, scale_stride=1, group=128), -1),
    (dict(out_type=4, scale_stride=1), -1), (dict(out_type=4, scale_out=P, group=32, scale_stride=1), -1), (dict(eps=-1.0), -1), (dict(eps=math.nan), -1),
    (dict(x=0), -1), (dict(out=0), -1), (dict(out_stride=63), -1), (dict(out_stride=0), -1), (dict(sum_out=P, sum_stride=8), -1), (dict(x_stride=-64), -1),
    (dict(x=P + 1), -1), (dict(weight=P + 2, weight_type=2), -1), (dict(reserved=1), -1)])
def test_rms_norm_refuses(change, code):
    rc, text = call(0, NORM, **change)
    assert rc == code and text.startswith("rms_norm: ")


@pytest.mark.parametrize("change,code", [
    (dict(type=4), 1), (dict(head_dim=63, rot_dim=63), -1), (dict(rot_dim=0), -1), (dict(rot_dim=66), -1), (dict(rot_dim=7), -1), (dict(h0=0), -1), (dict(h1=2), -1),
    (dict(x1=P), -1), (dict(batch=-1), -1), (dict(tokens=-1), -1), (dict(batch=1 << 16, tokens=1 << 16), 1), (dict(freqs=0), -1), (dict(freqs=P + 4), -1),
    (dict(amplitude=math.inf), -1), (dict(amplitude=math.nan), -1), (dict(x0=0), -1), (dict(out0=0), -1), (dict(os=(256, 128, 0, 0, 0, 0)), -1),
    (dict(xs=(256, -128, 64, 0, 0, 0)), -1), (dict(x0=P + 1), -1), (dict(positions=P + 4, positions_64=1), -1), (dict(head_dim=8192, os=(1 << 20, 1 << 18, 8192, 0, 0, 0)), 1)])
def test_rope_refuses(change, code):
    rc, text = call(1, ROPE, **change)
    assert rc == code and text.startswith("rope: ")


@pytest.mark.parametrize("change,code", [
    (dict(type=2), 1), (dict(type=4), 1), (dict(head_dim=48), 1), (dict(head_dim=256), 1), (dict(heads=0), -1), (dict(kv_heads=0), -1), (dict(heads=3), -1),
    (dict(batch=-1), -1), (dict(q_tokens=-1), -1), (dict(k_tokens=-1), -1), (dict(scale=0.0), -1), (dict(scale=-1.0), -1), (dict(scale=math.nan), -1),
    (dict(scale=math.inf), -1), (dict(softcap=-1.0), -1), (dict(softcap=math.inf), -1), (dict(softcap=math.nan), -1), (dict(softcap=1e-40), -1), (dict(q=0), -1), (dict(k=0), -1), (dict(out=0), -1),
    (dict(q=P + 8), 1), (dict(v=P + 2), 1), (dict(q_stride=(1024, 129, 64)), 1), (dict(k_stride=(1024, 128, 63)), 1), (dict(k_stride=(1024, -128, 64)), -1),
    (dict(out_stride=(1024, 128, 0)), -1), (dict(out_stride=(0, 128, 64)), -1), (dict(k_stride=(1024, 1 << 25, 64)), 1), (dict(lse=P + 2), -1),
    (dict(doc_offsets=P, n_docs=1), -1), (dict(doc_offsets=P, n_docs=-1, batch=1), -1), (dict(doc_offsets=P, n_docs=1, batch=1, q_tokens=4), -1),
    (dict(doc_offsets=P, n_docs=1, batch=1, k_len=P), -1), (dict(doc_offsets=P, n_docs=1, batch=1, q_start=0), -1), (dict(n_docs=1), -1), (dict(reserved=1), -1),
    (dict(q_tokens=(1 << 30) + 1), 1), (dict(q_start=-(1 << 31) + 1), 1),
    (dict(q_tokens=1, k_tokens=1 << 20), -1), (dict(q_tokens=1, k_tokens=1 << 20, workspace=P, workspace_bytes=64), -1)])
def test_attention_refuses(change, code):
    rc, text = call(2, ATTN, **change)
    assert rc == code and text.startswith("attention: ")


@pytest.mark.parametrize("change", [dict(k=P, v=P + 64), dict(k=P + 64, v=P), dict(k=P, v=P)])
def test_attention_refuses_to_write_its_keys(change):
    rc, text = call(2, ATTN, out=P, **change)
    assert rc == -1 and "not k or v" in text


def test_workspace_follows_the_sizes():
    ws = ops._entry()[3]

    def need(**change):
        a = {**ATTN, **change}
        flat = []
        for v in a.values():
            flat += list(v) if isinstance(v, tuple) else [v]
        return ws(ops._ATTN_ARGS.pack(*flat))

    assert need() == 0 and need(head_dim=48) == 0 and need(batch=0) == 0
    one = need(q_tokens=1, k_tokens=1 << 17)
    assert one > 0 and one % (4 * 65 * 2 * 2) == 0      # [batch * heads][splits][head_dim + 1] f32
    assert need(q_tokens=1, k_tokens=1 << 17, batch=4096) == 0


def test_python_checks():
    x = torch.zeros((2, 64), dtype=torch.float16)
    with pytest.raises(capi.MibcError, match="no CPU form"):
        ops.rms_norm(x)
    q = torch.zeros((1, 2, 2, 64), dtype=torch.float16)
    with pytest.raises(capi.MibcError, match="no CPU form"):
        ops.attention(q, q, q)
    with pytest.raises(capi.MibcError, match="no CPU form"):
        ops.rope(q, freqs=torch.ones(32, dtype=torch.float64))


def test_rope_frequencies():
    f = ops.rope_frequencies(64, device="cpu")
    want = torch.tensor([10000.0 ** (-2 * i / 64) for i in range(32)], dtype=torch.float64)
    tol = 4 * 2.0 ** -52 * want
    assert ((f - want).abs() <= tol).all()
    assert ((ops.rope_frequencies(64, scaling="linear", factor=4.0, device="cpu") - want / 4).abs() <= tol).all()
    base = ops.rope_frequencies(64, scaling="base", factor=8.0, device="cpu")
    assert float(base[0]) == 1.0 and abs(float(base[-1] * 8 / want[-1]) - 1) < 1e-13
    parts = ops.rope_frequencies(64, scaling="by_parts", factor=8.0, original_length=4096, device="cpu")
    turns = 4096 * want / (2 * math.pi)
    assert torch.equal(parts[turns >= 32], f[turns >= 32])
    assert ((parts[turns <= 1] - want[turns <= 1] / 8).abs() <= tol[turns <= 1]).all()
    assert (parts[1:] < parts[:-1]).all()
    for bad in (dict(rot_dim=7), dict(rot_dim=0), dict(rot_dim=8, theta=0.0), dict(rot_dim=8, scaling="linear", factor=0.0),
                dict(rot_dim=2, scaling="base", factor=2.0), dict(rot_dim=8, scaling="by_parts", factor=2.0),
                dict(rot_dim=8, scaling="by_parts", factor=2.0, original_length=10, turns_low=3, turns_high=3), dict(rot_dim=8, scaling="x")):
        with pytest.raises(capi.MibcError):
            ops.rope_frequencies(**bad, device="cpu")


def test_reference_against_torch():
    """The 64-bit reference of the GPU tests against torch's own modules in f64."""
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn((2, 9, 4, 32), generator=g, dtype=torch.float64) for _ in range(3))
    out = R.attention(q, k, v, window=(-1, 0))[0]
    want = torch.nn.functional.scaled_dot_product_attention(*(x.transpose(1, 2) for x in (q, k, v)), is_causal=True).transpose(1, 2)
    assert float((out - want).abs().max()) < 1e-13
    x = torch.randn((3, 40), generator=g, dtype=torch.float64)
    assert float((R.rms_norm(x)[0] - torch.nn.functional.rms_norm(x, (40,), eps=1e-5)).abs().max()) < 1e-13
    see, pos = R.visible(1, 3, 5, (1, 0), k_len=torch.tensor([4]))
    assert see[0].tolist() == [[True, True, False, False, False], [False, True, True, False, False], [False, False, True, True, False]]
    p = torch.arange(9)
    f = torch.tensor([1.0, 0.1], dtype=torch.float64)
    y = R.rope(q, f, p)
    assert float((y.norm(dim=-1) - q.norm(dim=-1)).abs().max()) < 1e-12 and float((R.rope(y, f, -p) - q).abs().max()) < 1e-12
