"""Transformer encoders whose attention, rotary positions or norms run on the operators (csrc/ops_*.hip): head sizes other than 64,
windows beyond the window kernels' 256 keys, widths other than 128 / 256 / 512.  Same contract as
test_gpu_parity.py::test_transformer_model_vs_oracle, pytest -m gpu."""
import numpy as np
import pytest

from dorado_amd import capi, config, synth
from oracle import oracle_py as O

pytestmark = pytest.mark.gpu


def _err(a, b):
    d = a.astype(np.float64) - b.astype(np.float64)
    return np.abs(d).max(), np.sqrt((d * d).mean())


@pytest.mark.parametrize("d_model,nhead,window,n,t_in", [
    (128, 4, (15, 16), 4, 1536),        # heads of 32
    (256, 2, (15, 16), 3, 1500),        # heads of 128, 125 tokens
    (384, 4, (40, 30), 2, 1536),        # heads of 96; 384 columns: the norm operator
    (384, 6, (15, 16), 2, 1536),        # heads of 64: window kernels, the norm operator
    (128, 2, (300, 200), 2, 6144),      # a window of 501 of the 512 tokens
    (512, 4, (127, 128), 2, 6144),      # the full width with heads of 128 (fused layer tail behind the operators)
])
def test_encoder_on_the_operators_vs_oracle(d_model, nhead, window, n, t_in):
    cfg = config.tiny_tx(d_model, nhead, window=window)
    if d_model == 512:
        cfg.tx.dim_feedforward = 2048
    ws = synth.make_weights(cfg, seed=71)
    x16 = synth.make_signal(n, t_in, seed=72)
    eng = capi.Engine(cfg, ws)
    scores = eng.forward(x16)
    t_tok = eng.output_steps(t_in) // cfg.tx.up_scale_factor
    tok = eng.tap(3, (n, t_tok, d_model), np.float16)
    s_o, tok_o = O.tx_forward(cfg, ws, x16.astype(np.float32)[:, None, :], want_tokens=True)
    assert s_o.shape == scores.shape
    mx, rms = _err(tok, tok_o)
    print(f"tokens max-abs {mx:.4f} rms {rms:.5f} (|x| rms {np.sqrt((tok_o ** 2).mean()):.3f})")
    assert rms <= 0.01 and mx <= 0.15
    mx, rms = _err(scores, s_o)
    print(f"scores max-abs {mx:.4f} rms {rms:.5f}")
    assert rms <= 0.03 and mx <= 0.5
    one = eng.forward(x16[:1])
    assert np.array_equal(one[0], scores[0]), "a chunk's scores must not depend on the batch"
    got, want = eng.call(x16), O.decode(scores.astype(np.float32), det=1)
    for a, b in zip(got, want):
        assert a[0] == b[0] and (a[2] == b[2]).all()
    eng.close()


@pytest.mark.parametrize("d_model,nhead", [(128, 8), (256, 1), (384, 5)])
def test_encoder_head_sizes_refused(d_model, nhead):
    cfg = config.tiny_tx(d_model, nhead)
    with pytest.raises(capi.MibcNotSupported):
        capi.Engine(cfg, synth.make_weights(cfg, seed=1))
