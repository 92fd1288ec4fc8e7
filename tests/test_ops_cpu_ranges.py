"""Transformer-layer operators without a GPU: refusals at the ends of their ranges, decided from the arguments alone."""
import ctypes as C

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
