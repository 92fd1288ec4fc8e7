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


@pytest.mark.parametrize("d_model,nhead,ff,depth,n,t_in", [
    (640, 10, 256, 2, 2, 1536),         # the 128 x 128 projections, heads of 64: window kernels and the norm operator
    (640, 20, 1024, 2, 2, 1536),        # heads of 32
    (768, 8, 512, 2, 3, 1500),          # heads of 96, 125 tokens
    (1024, 8, 1024, 1, 2, 3000),        # the persistent projections of K = 1024
    (1920, 15, 256, 1, 2, 1536),        # neither a power of two nor a multiple of 256 columns
    (2048, 16, 2048, 1, 4, 6144),       # the widest: persistent projections of K = 2048 (2048 rows), four chunks of a norm row a lane
])
def test_wide_encoders_vs_oracle(d_model, nhead, ff, depth, n, t_in):
    cfg = config.tiny_tx(d_model, nhead, depth=depth, ff=ff)
    ws = synth.make_weights(cfg, seed=75)
    x16 = synth.make_signal(n, t_in, seed=76)
    eng = capi.Engine(cfg, ws)
    scores = eng.forward(x16)
    t_tok = eng.output_steps(t_in) // cfg.tx.up_scale_factor
    tok = eng.tap(3, (n, t_tok, d_model), np.float16)
    m = min(n, 2)                       # the oracle's time grows with the rows
    s_o, tok_o = O.tx_forward(cfg, ws, x16[:m].astype(np.float32)[:, None, :], want_tokens=True)
    mx, rms = _err(tok[:m], tok_o)
    print(f"tokens max-abs {mx:.4f} rms {rms:.5f} (|x| rms {np.sqrt((tok_o ** 2).mean()):.3f})", flush=True)
    assert rms <= 0.01 and mx <= 0.15
    mx, rms = _err(scores[:m], s_o)
    print(f"scores max-abs {mx:.4f} rms {rms:.5f}", flush=True)
    assert rms <= 0.03 and mx <= 0.5
    for x in (0, n - 1):
        assert np.array_equal(eng.forward(x16[x:x + 1])[0], scores[x]), "a chunk's scores must not depend on the batch"
    got, want = eng.call(x16), O.decode(scores.astype(np.float32), det=1)
    for a, b in zip(got, want):
        assert a[0] == b[0] and (a[2] == b[2]).all()
    eng.close()


def test_operators_need_no_transposed_values():
    # the same width with heads of 64 (window kernels, which read V transposed) and of 32 (the operators, which read it as it lies)
    need = []
    for nhead in (4, 8):
        cfg = config.tiny_tx(256, nhead)
        eng = capi.Engine(cfg, synth.make_weights(cfg, seed=77))
        need.append(eng.query_memory(1536)[0])
        tokens = eng.output_steps(1536) // cfg.tx.up_scale_factor
        eng.close()
    assert need[0] - need[1] == tokens * 256 * 2
