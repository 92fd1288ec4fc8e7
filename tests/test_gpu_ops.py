"""Transformer-layer operators (dorado_amd.ops -> mibc_rms_norm, mibc_rope, mibc_attention) against plain 64-bit
implementations (tests/ops_reference.py, where the tolerances are derived), pytest -m gpu."""
import math

import pytest
import torch

from dorado_amd import capi, ops
from tests import ops_reference as R

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def rnd(shape, t, seed, mul=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * mul).to(t).cuda()


# ---------------------------------------------------------------------------------------------------------------- RMS norm
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 64), (33, 128), (7, 130), (4, 512), (9, 1000), (2, 1024), (3, 2048),
                                       (2, 4096), (3, 5000), (2, 8192), (1, 16384), (2, 32768), (513, 256)])
@pytest.mark.parametrize("t", [F16, BF16, F32])
def test_rms_norm(rows, cols, t):
    x, r = rnd((rows, cols), t, 1, 2.0), rnd((rows, cols), t, 2)
    for res, alpha, w in ((None, 1.0, None), (r, 2.5, rnd((cols,), F32, 3) + 1), (r, -0.5, rnd((cols,), t, 4))):
        y, h = ops.rms_norm(x, w, residual=res, alpha=alpha, return_sum=True)
        want, wsum = R.rms_norm(x, w, res, alpha)
        R.close(y, want, R.rms_norm_tolerance(want, x, w, res, alpha, t), "y")
        terms = x.cpu().double().abs() + (0 if res is None else abs(alpha) * res.cpu().double().abs())
        R.close(h, wsum, R.u(t) * wsum.abs() + 2.0 ** -23 * terms + 2.0 ** -38, "h")
        assert y.dtype is t and h.dtype is t


@pytest.mark.parametrize("rows,cols,group", [(1, 1, 0), (3, 77, 0), (4, 128, 0), (4, 128, 128), (5, 512, 64), (2, 4096, 128), (3, 2080, 32),
                                             (2, 5000, 0), (2, 32768, 128), (65, 256, 32)])
@pytest.mark.parametrize("quant,most", [("int8", 127.0), ("e4m3", 448.0)])
@pytest.mark.parametrize("t", [F16, BF16, F32])
def test_rms_norm_8bit(rows, cols, group, quant, most, t):
    x, r, w = rnd((rows, cols), t, 5), rnd((rows, cols), t, 6), rnd((cols,), F32, 7) + 1
    q, s = ops.rms_norm(x, w, residual=r, quant=quant, group=group)
    want, _ = R.rms_norm(x, w, r)
    g = want.view(rows, -1, group or cols)
    ws = g.abs().amax(-1) / most
    f32 = R.rms_norm_tolerance(want, x, w, r, 1.0, F32).view(g.shape)
    R.close(s, ws, f32.amax(-1) / most + 2.0 ** -23 * ws, "scales")
    got = q.cpu().double().view(g.shape) * s.cpu().double()[..., None]
    step = ws[..., None]
    half = 0.5 * step if quant == "int8" else 2.0 ** -4 * g.abs() + 2.0 ** -10 * step
    # half a step of the code, the f32 error of the value, of the scale (128 codes of it at most) and of the quotient
    tol = half + 2 * f32 + (f32.amax(-1, keepdim=True) / most + 2.0 ** -22 * step) * most
    R.close(got, g, tol, quant)
    assert float(q.double().abs().max()) == most or cols == 1 or rows * cols > 0


def test_rms_norm_values():
    x = rnd((6, 256), F16, 8)
    x[1] = 0
    x[2, 5] = math.nan
    x[3, 6] = math.inf
    x[4] = 6e-8                                    # the smallest f16
    y = ops.rms_norm(x)
    want, _ = R.rms_norm(x)
    assert (y[1] == 0).all() and y[2].isnan().all() and y[3, 6].isnan() and (y[3, :6] == 0).all()
    rows = [0, 1, 4, 5]
    R.close(y[rows], want[rows], R.rms_norm_tolerance(want, x, None, None, 1.0, F16)[rows], "y")
    for quant in ("int8", "e4m3"):
        q, s = ops.rms_norm(x, quant=quant, group=64)
        assert (s[1] == 1).all() and (q[1].float() == 0).all()
        assert s[2].isnan().all() and (q[2].float() == 0).all()
        assert s[3, 0].isnan() and (s[3, 1:] == 1).all()
    # values below 448 of f32's smallest: their scale would be 0
    w = torch.full((64,), 1e-41, device="cuda")
    for quant in ("int8", "e4m3"):
        q, s = ops.rms_norm(torch.ones((1, 64), device="cuda"), w * 1e-3, quant=quant)
        assert float(s) == 1 and (q.float() == 0).all()
        q, s = ops.rms_norm(torch.ones((1, 64), device="cuda"), w, quant=quant)       # a scale of few bits: codes stay finite
        assert q.float().isfinite().all() and 0 < float(s) < 1e-40
    b = rnd((2, 64), BF16, 9)
    b[0] = torch.finfo(BF16).min                  # squares beyond f32: the root is infinite and y is 0, as in f32 arithmetic
    assert (ops.rms_norm(b)[0] == 0).all()


def test_rms_norm_layouts():
    base = rnd((4, 5, 3 * 96), BF16, 10)
    x = base[:, :, 96:192].reshape(20, 96)
    view = base.view(20, 288)[:, 96:192]           # row stride 288
    assert torch.equal(ops.rms_norm(view), ops.rms_norm(x.contiguous()))
    odd = base.view(20, 288)[:, 1:96]              # misaligned rows, 95 columns
    assert torch.equal(ops.rms_norm(odd), ops.rms_norm(odd.contiguous()))
    one = x[3].clone()
    assert torch.equal(ops.rms_norm(one), ops.rms_norm(x.contiguous())[3])
    r = x[:1].expand(20, 96)                       # the same residual for all rows
    assert torch.equal(ops.rms_norm(x, residual=r), ops.rms_norm(x, residual=r.contiguous()))
    out = torch.full((20, 300), 7.0, dtype=BF16, device="cuda")
    ops.rms_norm(x, out=out[:, 100:196])
    assert torch.equal(out[:, 100:196], ops.rms_norm(x)) and (out[:, :100] == 7).all() and (out[:, 196:] == 7).all()
    a, s = x.clone(), rnd((20, 96), BF16, 11)      # in place: x <- y, residual <- sum
    wy, wh = ops.rms_norm(a, residual=s, return_sum=True)
    ops.rms_norm(a, residual=s, out=a, sum_out=s)
    assert torch.equal(a, wy) and torch.equal(s, wh)
    assert ops.rms_norm(x[:0]).shape == (0, 96)
    assert ops.rms_norm(base.transpose(0, 1)[:, :1, :288]).shape == (5, 1, 288)


# -------------------------------------------------------------------------------------------------------------------- rope
@pytest.mark.parametrize("t", [F16, BF16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("b,n,h,kh,d,rot", [(1, 1, 1, 1, 64, 64), (2, 5, 8, 8, 64, 64), (3, 7, 6, 2, 128, 64), (1, 33, 5, 1, 80, 80),
                                            (2, 3, 3, 3, 80, 40), (1, 4, 2, 1, 10, 6), (2, 9, 32, 8, 128, 128), (1, 2, 4, 4, 256, 192),
                                            (1, 3, 1, 1, 2, 2), (1, 301, 40, 2, 96, 96)])
def test_rope(t, interleaved, b, n, h, kh, d, rot):
    both = rnd((b, n, h + kh, d), t, 20)
    q, k = both[:, :, :h], both[:, :, h:]
    f = ops.rope_frequencies(rot)
    g = torch.Generator().manual_seed(21)
    for start, positions, amplitude in ((0, None, 1.0), (100000, None, 1.25), (0, torch.randint(-5000, 2000000, (b, n), generator=g), 1.0),
                                        (0, torch.randint(0, 2**31 - 1, (b, n), generator=g, dtype=torch.int32), -0.5),
                                        (0, torch.arange(n) * 3, 1.0)):
        p = torch.arange(start, start + n) if positions is None else positions
        gq, gk = ops.rope(q, k, freqs=f, positions=None if positions is None else positions.cuda(), start=start,
                          interleaved=interleaved, amplitude=amplitude)
        for x, got in ((q, gq), (k, gk)):
            want = R.rope(x, f, p, interleaved, amplitude)
            want[..., rot:] = x[..., rot:].cpu().double()
            R.close(got, want, R.rope_tolerance(want, x, f, p, amplitude, t, interleaved), "rope")
            assert torch.equal(got[..., rot:], x[..., rot:])


def test_rope_in_place_and_back():
    both = rnd((2, 50, 10, 64), F32, 22)
    f = ops.rope_frequencies(48, 500.0).cuda()
    want = ops.rope(both[:, :, :8], both[:, :, 8:], freqs=f, start=7)
    x = both.clone()
    got = ops.rope(x[:, :, :8], x[:, :, 8:], freqs=f, start=7, out=(x[:, :, :8], x[:, :, 8:]))
    assert torch.equal(x[:, :, :8], want[0]) and torch.equal(x[:, :, 8:], want[1]) and got[0].data_ptr() == x.data_ptr()
    p = -torch.arange(7, 57).cuda()
    back = ops.rope(x, freqs=f, positions=p)
    assert float((back - both).abs().max()) <= 2.0 ** -20 * 6.0     # two turns of pairs below 6 in f32
    odd = rnd((1, 4, 3, 65), F16, 23)[:, :, :, 1:]                  # misaligned heads
    assert torch.equal(ops.rope(odd, freqs=f), ops.rope(odd.contiguous(), freqs=f))
    assert ops.rope(both[:, :0], freqs=f).shape == (2, 0, 10, 64)
    wide = both[:, :, :1].expand(2, 50, 4, 64)                      # one head for four
    assert torch.equal(ops.rope(wide, freqs=f), ops.rope(wide.contiguous(), freqs=f))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("h,kh,d,rot", [(20, 3, 40, 40), (8, 0, 40, 20), (1, 9, 36, 10)])
def test_rope_in_place_other_sizes(h, kh, d, rot, interleaved):
    x = rnd((2, 9, h + kh, d), BF16, 24)
    q, k, f = x[:, :, :h], x[:, :, h:] if kh else None, ops.rope_frequencies(rot)
    want = ops.rope(q.clone(), None if k is None else k.clone(), freqs=f, start=3, interleaved=interleaved)
    got = ops.rope(q, k, freqs=f, start=3, interleaved=interleaved, out=q if k is None else (q, k))
    for a, b in zip((got,) if k is None else got, (want,) if k is None else want):
        assert torch.equal(a, b)
    R.close(q, R.rope(rnd((2, 9, h + kh, d), BF16, 24)[:, :, :h], f, torch.arange(3, 12), interleaved),
            R.rope_tolerance(q.cpu().double(), rnd((2, 9, h + kh, d), BF16, 24)[:, :, :h], f, torch.arange(3, 12), 1.0, BF16, interleaved)
            + 2.0 ** -8 * R.u(BF16) * q.cpu().double().abs(), "in place")      # the tolerance of the rounded value, not of the exact one


# --------------------------------------------------------------------------------------------------------------- attention
def qkv(b, n, m, h, kh, d, t, seed, mul=1.0):
    return rnd((b, n, h, d), t, seed, mul), rnd((b, m, kh, d), t, seed + 1, mul), rnd((b, m, kh, d), t, seed + 2)


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def check(q, k, v, **kw):
    out, lse = ops.attention(q, k, v, return_lse=True, **kw)
    if kw.pop("causal", False):
        kw["window"] = (-1, 0)
    kw = {x: (y.cpu() if isinstance(y, torch.Tensor) else y) for x, y in kw.items()}
    want, wlse, tol, ltol = R.attention(q, k, v, **kw)
    R.close(out, want, tol, "out")
    R.close(lse, wlse, ltol, "lse")
    return out, lse


@pytest.mark.parametrize("t", [F16, BF16])
@pytest.mark.parametrize("d", [32, 64, 96, 128])
@pytest.mark.parametrize("n,m", [(1, 1), (1, 2), (1, 200), (2, 3), (17, 63), (64, 64), (65, 65), (130, 129), (31, 257), (300, 300), (1, 1100)])
def test_attention_sizes(t, d, n, m):
    q, k, v = qkv(2, n, m, 4, 2, d, t, 30, 1.5)
    check(q, k, v)
    check(q, k, v, causal=True)


MASKS = {
    "window": dict(window=(5, 3)), "back": dict(window=(40, 0)), "ahead": dict(window=(-1, 70)), "zero": dict(window=(0, 0)),
    "wide": dict(window=(2**31 - 1, 2**31 - 1)), "lengths": dict(k_len=i32, lens=(0, 1, 70, 150)), "over": dict(k_len=i32, lens=(-3, 64, 1000, 149)),
    "causal lengths": dict(causal=True, k_len=i32, lens=(0, 1, 70, 150)), "prefix": dict(causal=True, prefix=i32, lens=(0, 1, 90, 1000)),
    "sinks": dict(window=(10, 0), prefix=i32, lens=(0, 4, 64, 150)), "start": dict(window=(30, 0), q_start=20), "before": dict(causal=True, q_start=-40),
    "beyond": dict(window=(30, 0), q_start=140),
}


@pytest.mark.parametrize("extra", [dict(), dict(softcap=5.0), dict(slopes=True), dict(softcap=20.0, slopes=True)], ids=["plain", "cap", "slopes", "both"])
@pytest.mark.parametrize("mask", sorted(MASKS))
@pytest.mark.parametrize("t,d,n", [(F16, 64, 100), (BF16, 128, 100), (BF16, 128, 3), (F16, 32, 1), (BF16, 96, 150)])
def test_attention_masks(mask, extra, t, d, n):
    q, k, v = qkv(4, n, 150, 6, 2, d, t, 40, 1.5)
    kw = dict(MASKS[mask])
    lens = kw.pop("lens", None)
    for x in ("k_len", "prefix"):
        if x in kw:
            kw[x] = i32(*lens)
    extra = dict(extra)
    if "slopes" in extra:
        extra["slopes"] = torch.tensor([0.5, 0.25, 0.0, 1.0, -0.01, 2.0]).cuda()
    out, lse = check(q, k, v, **kw, **extra)
    if lens == (0, 1, 70, 150) and "k_len" in kw:
        assert (out[0] == 0).all() and (lse[0] == -math.inf).all()


@pytest.mark.parametrize("offsets,prefix", [((0, 300), None), ((0, 1, 1, 1, 65, 200, 290), None), ((7, 7, 100, 280), (3, 40, 500)),
                                            ((0,), None), ((0, 0), None), (tuple(range(0, 301, 3)), None), ((0, 150, 900), None)])
@pytest.mark.parametrize("window", [(-1, -1), (-1, 0), (20, 10)])
@pytest.mark.parametrize("t,d", [(F16, 64), (BF16, 128)])
def test_attention_documents(offsets, prefix, window, t, d):
    q, k, v = qkv(1, 300, 300, 4, 2, d, t, 50, 1.5)
    kw = dict(window=window, doc_offsets=i32(*offsets), prefix=None if prefix is None else i32(*prefix))
    out, _ = check(q, k, v, **kw)
    inside = torch.zeros(300, dtype=torch.bool)
    for a, z in zip(offsets, offsets[1:]):
        inside[a:z] = True
    assert (out[0].cpu()[~inside] == 0).all()
    # a document in a batch gives the bits that it gives alone (same tiles: it starts on a tile of its own in both)
    if offsets == (0, 300):
        assert torch.equal(out, ops.attention(q, k, v, window=window))


def test_attention_bad_documents_stay_inside():
    q, k, v = qkv(1, 200, 200, 2, 2, 64, F16, 55)
    for offsets in ((-50, 100, 400), (100, 50, 10), (200, 0), (2**31 - 1, -(2**31) + 1, 0, 70), (0, 2**31 - 1)):
        out = ops.attention(q, k, v, doc_offsets=i32(*offsets), prefix=torch.full((len(offsets) - 1,), 2**31 - 1, dtype=torch.int32, device="cuda"))
        assert out.isfinite().all()


@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("t,d,n", [(F16, 64, 90), (BF16, 128, 90), (BF16, 128, 2), (F16, 96, 1)])
def test_attention_hidden_values(what, t, d, n):
    m = 200
    q, k, v = qkv(2, n, m, 4, 2, d, t, 60)
    lens = i32(131, 77)
    clean, cl = ops.attention(q, k, v, causal=True, k_len=lens, return_lse=True)
    k2, v2 = k.clone(), v.clone()
    for x, e in enumerate((131, 77)):
        k2[x, e:], v2[x, e:] = what, what
    got, gl = ops.attention(q, k2, v2, causal=True, k_len=lens, return_lse=True)
    assert torch.equal(got, clean) and torch.equal(gl, cl)
    # keys and values that later queries see and earlier ones do not
    v2, k2 = v.clone(), k.clone()
    v2[0, 100, 0, 3] = what
    v2[1, 60, 1, 7] = what
    k2[1, 70, 0, 0] = math.nan
    check(q, k2, v2, causal=True, k_len=lens)
    # all three in one tile
    v2[0, 97, 0, 3], v2[0, 98, 0, 5], v2[0, 99, 0, 5] = math.nan, math.inf, -math.inf
    check(q, k2, v2, causal=True, k_len=lens)


@pytest.mark.parametrize("d", [32, 128])
@pytest.mark.parametrize("n,m", [(1, 130), (1, 1200), (5, 300), (5, 1200), (40, 300), (40, 1200), (200, 1200)])
def test_attention_seen_values_of_no_weight(n, m, d):
    # a slope of 0.5 takes keys that are 210 away to weights below the smallest f32: their NaN and infinities arrive all the same,
    # in a pass over one part, in the join of waves and in that of parts
    q, k, v = qkv(2, n, m, 2, 1, d, BF16, 61)
    v[0, 0, 0, 1], v[0, 2, 0, 2], v[0, 3, 0, 3], v[1, m // 2, 0, 5], v[1, m // 3, 0, 5] = math.nan, math.inf, -math.inf, math.inf, -math.inf
    check(q, k, v, slopes=torch.tensor([0.5, 0.01]).cuda())


def test_attention_extreme_scores():
    q, k, v = qkv(1, 70, 140, 2, 1, 64, F16, 70)
    check(q * 20, k * 20, v)                                   # one key takes all
    rising = k * 0 + torch.arange(140, device="cuda", dtype=F16)[None, :, None, None] / 16
    check(q * 0 + 1, rising, v)                                # the maximum moves with every tile
    check(q * 0 + 1, rising.flip(1).contiguous(), v)
    z = ops.attention(q, torch.full_like(k, -math.inf), v, scale=1.0, return_lse=True)
    assert z[0].isnan().any() or (z[0] == 0).all()
    low = torch.full_like(k, -65504.0)                         # the type's lowest value as a key: finite scores of about -4e6
    check(q.abs(), low, v)
    check(q, k, v, scale=1e-6)
    check(q, k, v * 60000)


def test_attention_layouts():
    b, n, h, kh, d = 2, 200, 6, 2, 64
    buf = rnd((b, n, h + 2 * kh, d), F16, 80)
    q, k, v = buf[:, :, :h], buf[:, :, h:h + kh], buf[:, :, h + kh:]
    want = ops.attention(q.contiguous(), k.contiguous(), v.contiguous(), causal=True)
    assert torch.equal(ops.attention(q, k, v, causal=True), want)
    heads_first = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]     # [b, heads, tokens, d] in memory
    assert torch.equal(ops.attention(*heads_first, causal=True), want)
    out = torch.full((b, h, n + 3, d), 9.0, dtype=F16, device="cuda")
    ops.attention(q, k, v, causal=True, out=out.transpose(1, 2)[:, :n])
    assert torch.equal(out.transpose(1, 2)[:, :n], want) and (out[:, :, n:] == 9).all()
    one = k[:1].expand(b, n, kh, d)                                                      # one row's keys for the whole batch
    assert torch.equal(ops.attention(q, one, one), ops.attention(q, one.contiguous(), one.contiguous()))
    assert torch.equal(ops.attention(q, k, v, out=q.contiguous()), ops.attention(q, k, v))
    assert (ops.attention(q, k[:, :0], v[:, :0]) == 0).all()
    assert ops.attention(q[:, :0], k, v).shape == (b, 0, h, d) and ops.attention(q[:0], k[:0], v[:0]).shape == (0, n, h, d)


@pytest.mark.parametrize("d", [32, 64, 96])
@pytest.mark.parametrize("b,kh", [(2, 8), (8, 4), (16, 1), (3, 8), (4, 12)])
@pytest.mark.parametrize("n,m,kw", [(1, 200, {}), (1, 2100, {}), (12, 700, dict(causal=True)), (150, 150, {}), (150, 150, dict(causal=True)), (70, 1100, dict(window=(30, 5)))])
def test_attention_neighbouring_heads(b, kh, n, m, kw, d):
    # pairs of heads whose keys share cache lines are dealt to the same part of the chip; every pair is worked on once
    check(*qkv(b, n, m, kh, kh, d, F16, 75), **kw)


@pytest.mark.parametrize("n,m", [(1, 1200), (3, 40), (40, 1200), (300, 300)])
def test_attention_in_place(n, m):
    # the queries' columns of a packed q | k | v buffer receive the result; the others stay
    x = rnd((2, max(n, m), 8, 64), F16, 71)
    q, k, v = x[:, :n, :4], x[:, :m, 4:6], x[:, :m, 6:]
    before, want = x.clone(), ops.attention(q, k, v)
    assert ops.attention(q, k, v, out=q) is q and torch.equal(q, want)
    assert torch.equal(x[:, :, 4:], before[:, :, 4:]) and torch.equal(x[:, n:, :4], before[:, n:, :4])
    with pytest.raises(capi.MibcError, match="not k or v"):
        ops.attention(k, k, v, out=v)
    with pytest.raises((capi.MibcError, capi.MibcNotSupported)):
        ops.attention(q[..., :0], k[..., :0], v[..., :0])


def test_attention_long_axis_is_split_and_joined():
    q, k, v = qkv(1, 1, 20011, 4, 1, 128, BF16, 90)
    a = struct_args(q, k, v)
    assert ops._entry()[3](a) > 0
    check(q, k, v, causal=True)
    q, k, v = qkv(1, 40, 9001, 2, 2, 64, F16, 91)
    check(q, k, v, causal=True, k_len=i32(8003))
    check(q, k, v, window=(100, 0), prefix=i32(5))


def struct_args(q, k, v):
    return ops._ATTN_ARGS.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), q.data_ptr(), 0, 0, 0, 0, 0, 0, 0, *q.stride()[:3], *k.stride()[:3],
                               *v.stride()[:3], *q.stride()[:3], q.shape[0], q.shape[2], k.shape[2], q.shape[1], k.shape[1], q.shape[3], 0,
                               ops._TYPE[q.dtype], -1, -1, ops.ATTN_END, 0.1, 0.0, 0)


def test_numbers_outside_their_fields():
    x, f = rnd((1, 2, 2, 64), F16, 72), torch.ones(32, dtype=torch.float64).cuda()
    for bad in (1e39, None):        # infinite in f32, no number
        for call in (lambda: ops.rope(x, freqs=f, amplitude=bad), lambda: ops.attention(x, x, x, softcap=bad)):
            with pytest.raises(capi.MibcError):
                call()
    with pytest.raises(capi.MibcError, match="rms_norm: "):
        ops.rms_norm(x, eps=None)
    with pytest.raises(capi.MibcError, match="rms_norm: "):
        ops.rms_norm(x, quant="int8", group=1 << 40)
    with pytest.raises(capi.MibcError, match="rope: "):
        ops.rope(x, freqs=f, start=1 << 64)
    with pytest.raises(capi.MibcError, match="attention: "):
        ops.attention(x, x, x, scale=-1e39)


@pytest.mark.parametrize("n", [1, 17])
def test_attention_many_pairs(n):
    # more than 2^20 workgroups; any slice of the batch gives the same bits by itself
    b = (1 << 17) + 3
    q, k, v = qkv(1, n, 3, 8, 8, 32, F16, 76)
    scale = (torch.arange(b, device="cuda") % 61 + 1).to(F16)[:, None, None, None] / 32
    q = q * scale
    k, v = (x.expand(b, -1, -1, -1) for x in (k, v))
    out = ops.attention(q, k, v)
    for x in (0, 70000, b - 40):
        assert torch.equal(out[x:x + 37], ops.attention(q[x:x + 37], k[:37], v[:37]))
    assert torch.equal(out[-1], out[(b - 1) % 61])


def test_rms_norm_many_rows():
    rows = (1 << 22) + 5        # four to a workgroup: more than 2^20 of them
    x = rnd((61, 136), F16, 77)[torch.arange(rows, device="cuda") % 61]
    y = ops.rms_norm(x)
    assert torch.equal(y, ops.rms_norm(x[:61])[torch.arange(rows, device="cuda") % 61])


@pytest.mark.parametrize("cols", [8, 24, 32, 33, 64, 65])
@pytest.mark.parametrize("quant", ["int8", "e4m3"])
def test_rms_norm_narrow_8bit(cols, quant):
    # 4, 8 and 16 lanes to a row: scales and codes of a row are those of the row alone
    x, w = rnd((1001, cols), BF16, 78), rnd((cols,), BF16, 79)
    y = R.rms_norm(x, w)[0]
    q, s = ops.rms_norm(x, w, quant=quant)
    most = 127.0 if quant == "int8" else 448.0
    want = y.abs().amax(1, keepdim=True) / most
    assert ((s.cpu().to(R.F64) - want).abs() <= 2.0 ** -18 * want).all()
    # int8: half a code.  e4m3: half a step, 2^-4 of the value (2^-10 of the scale below its normal range), plus the norm's own 2^-18
    near = 0.5 * want if quant == "int8" else torch.maximum(y.abs() * 2.0 ** -4, want * 2.0 ** -10)
    off = (q.cpu().to(R.F64) * s.cpu().to(R.F64) - y).abs()
    assert (off <= near * (1 + 2.0 ** -16) + 2.0 ** -16 * most * want).all()
    one = [ops.rms_norm(x[r:r + 1], w, quant=quant) for r in (0, 7, 500, 1000)]
    for r, (q1, s1) in zip((0, 7, 500, 1000), one):
        assert torch.equal(q[r].view(torch.uint8), q1[0].view(torch.uint8)) and torch.equal(s[r], s1[0])


def test_attention_offsets_beyond_32_bits():
    """A cache of more than 2^31 elements: the last batch row and the last tokens lie behind it."""
    m, kh, d = 70000, 8, 128
    cache = torch.empty((2, 17, m, kh, d), dtype=F16, device="cuda")
    assert cache[0].numel() > 1 << 30 and cache.numel() * 2 > 1 << 32
    cache[:, 16] = rnd((2, 1, kh, d), F16, 95).expand(2, m, kh, d)
    cache[:, 16, -300:] = rnd((2, 300, kh, d), F16, 96)
    k, v = cache[0, 15:17], cache[1, 15:17]
    k[0], v[0] = 0, 0
    q = rnd((2, 2, 8, d), F16, 97)
    got = ops.attention(q, k, v, window=(250, 0))
    want = ops.attention(q[1:].contiguous(), k[1:, -300:].contiguous(), v[1:, -300:].contiguous(), window=(250, 0))
    tol = R.attention(q[1:], k[1:, -300:], v[1:, -300:], window=(250, 0))[2]
    R.close(got[1:], want.cpu().double(), 2 * tol, "far rows")


def test_results_repeat():
    """The same bits every time: nothing depends on the order in which workgroups finish."""
    q, k, v = qkv(3, 5, 9000, 8, 2, 128, BF16, 100)
    a = [ops.attention(q, k, v, causal=True, return_lse=True) for _ in range(4)]
    assert all(torch.equal(x[0], a[0][0]) and torch.equal(x[1], a[0][1]) for x in a)


# -------------------------------------------------------------------------------------------------- together, as they are used
def layer(x, res, w, wqkv, f, heads, kv, d, lens=None):
    b, n, c = x.shape
    y, s = ops.rms_norm(x, w, residual=res, alpha=2.0, return_sum=True)
    z = (y @ wqkv.T).view(b, n, heads + 2 * kv, d)
    qk = z[:, :, :heads + kv]
    ops.rope(qk, freqs=f, out=qk)
    return ops.attention(z[:, :, :heads], z[:, :, heads:heads + kv], z[:, :, heads + kv:], window=(31, 32), k_len=lens), s


def test_layer_of_the_three():
    """norm -> projection -> rotary positions in place -> window attention, as a transformer layer runs them, against f64 with the
    same roundings between the operators; then captured into a graph, replayed with other inputs between eager calls."""
    b, n, heads, kv, d = 2, 190, 4, 2, 64
    c = heads * d
    x, res, w = rnd((b, n, c), F16, 110), rnd((b, n, c), F16, 111), rnd((c,), F32, 112) * 0.1 + 1
    wqkv = rnd(((heads + 2 * kv) * d, c), F16, 113, c ** -0.5)
    f = ops.rope_frequencies(d)
    got, s = layer(x, res, w, wqkv, f, heads, kv, d)
    y, h = R.rms_norm(x, w, res, 2.0)
    z = (y.to(F16).double() @ wqkv.cpu().double().T).view(b, n, heads + 2 * kv, d).to(F16)
    qk = R.rope(z[:, :, :heads + kv], f, torch.arange(n)).to(F16)
    want, _, tol, _ = R.attention(qk[:, :, :heads], qk[:, :, heads:], z[:, :, heads + kv:], window=(31, 32))
    # a rounding of y, q, k or v to f16 may fall the other way: one step of each, through scores of spread below 4 and sums of c terms
    R.close(got, want, tol + 2.0 ** -10 * 8, "layer")
    R.close(s, h, R.u(F16) * h.abs() + 2.0 ** -20, "sum")

    graph = torch.cuda.CUDAGraph()
    xs = x.clone()
    with torch.no_grad():
        layer(xs, res, w, wqkv, f, heads, kv, d)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            out, total = layer(xs, res, w, wqkv, f, heads, kv, d)
        for seed in (120, 121, 122, 123):
            new = rnd((b, n, c), F16, seed)
            xs.copy_(new)
            graph.replay()
            eager, esum = layer(new, res, w, wqkv, f, heads, kv, d)
            torch.cuda.synchronize()
            assert torch.equal(out, eager) and torch.equal(total, esum)


def test_split_attention_in_two_graphs():
    """Two captured graphs of a split attention, replayed in turn and on two streams at once, each with its own workspace."""
    q, k, v = qkv(2, 1, 6000, 8, 2, 128, F16, 130)
    graphs, outs, qs = [], [], [q.clone(), (q * 0.5).contiguous()]
    for x in qs:
        ops.attention(x, k, v)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.attention(x, k, v))
        graphs.append(g)
    want = [ops.attention(x, k, v) for x in qs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


def test_other_stream_and_threads():
    import threading
    q, k, v = qkv(2, 3, 4000, 8, 2, 128, BF16, 140)
    x = rnd((300, 512), F16, 141)
    want, wn = ops.attention(q, k, v, causal=True), ops.rms_norm(x)
    torch.cuda.synchronize()
    res, errors = {}, []

    def work(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(10):
                    a, y = ops.attention(q, k, v, causal=True), ops.rms_norm(x)
            s.synchronize()
            res[i] = torch.equal(a, want) and torch.equal(y, wn)
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    ts = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert not errors and all(res[i] for i in range(4))


def test_work_follows_the_current_stream():
    s = torch.cuda.Stream()
    x = torch.zeros((4096, 4096), dtype=F16, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        for _ in range(20):
            x.add_(1)
        y = ops.rms_norm(x, eps=0.0)
    s.synchronize()
    assert (y == 1).all()


def test_gradients_are_refused():
    x = torch.zeros((2, 64), device="cuda", requires_grad=True)
    with pytest.raises(capi.MibcNotSupported):
        ops.rms_norm(x)
    with torch.no_grad():
        ops.rms_norm(x)
