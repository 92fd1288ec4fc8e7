"""Transformer encoders on the operators at the ends of what is accepted: windows as wide as the limits' type, widths up to 2048
(same contract as tests/test_gpu_ops_encoder.py), pytest -m gpu."""
import copy

import numpy as np
import pytest

from dorado_amd import capi, config, synth
from oracle import oracle_py as O
from tests.test_gpu_ops_encoder import _err

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window", [(2**31 - 1, 2**31 - 1), (2**31 - 1, 15), (15, 2**31 - 1), (2**31 - 65, 1), (200, 57)])
def test_windows_of_any_width(window):
    # heads of 64: limits whose sum leaves 32 bits are windows over all tokens, not narrow ones
    cfg = config.tiny_tx(128, 2, window=window)
    plain = copy.deepcopy(cfg)
    plain.tx.attn_window = tuple(min(w, 512) for w in window)      # as far as 512 tokens see
    ws = synth.make_weights(cfg, seed=73)
    x16 = synth.make_signal(2, 6144, seed=74)
    eng = capi.Engine(cfg, ws)
    scores = eng.forward(x16)
    same = capi.Engine(plain, ws)
    assert np.array_equal(scores, same.forward(x16))
    s_o = O.tx_forward(plain, ws, x16.astype(np.float32)[:, None, :])
    mx, rms = _err(scores, s_o)
    print(f"scores max-abs {mx:.4f} rms {rms:.5f}")
    assert rms <= 0.03 and mx <= 0.5
    eng.close()
    same.close()
