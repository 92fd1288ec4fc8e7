"""Transformer-layer operators (dorado_amd.ops) at the ends of their ranges, against 64-bit implementations: large caps, weights far below
the largest, values near the type's end, 8-bit codes that have to be the rounded quotients themselves, pytest -m gpu.  The bounds are
narrower than those of tests/ops_reference.py: none grows with the cap or with the number of keys."""
import ctypes
import math

import pytest
import torch

from dorado_amd import capi, ops
from tests import ops_reference as R

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
F64 = torch.float64


def rnd(shape, t, seed, mul=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * mul).to(t).cuda()


def reference(q, k, v, softcap=0.0, slopes=None, causal=False):
    """(out, lse, bound of out, bound of lse) in f64.

    A score is off by (d + 8) 2^-24 of its products' magnitudes (an f32 sum of d of them and the scale), by 2^-20 of itself (the exponent's
    own roundings and, where it is capped, those of tanh: at most eight of 2^-23) and, caps up to 64, by cap 2^-21 (the cap's form there
    adds numbers of the cap's size: a reciprocal of 1 ulp near 1/2, twice the cap times; two f32 roundings of the cap).  Probabilities are
    rounded to the type t before the product with v, by at most u(t) of themselves (f16: by at most 2^-36 of the largest: half a step of
    2^-24, with 2^11 in front); up to 16 rows
    per key head by two parts, so u(t)^2.  2^-19: sums of keys in f32, joins.  Then one rounding of the output."""
    t, (b, n, h, d) = q.dtype, q.shape
    m, kh = k.shape[1], k.shape[2]
    q, k, v = (x.cpu().to(F64) for x in (q, k, v))
    i, j = torch.arange(m - n, m)[:, None], torch.arange(m)[None]
    hidden = (j > i) if causal else torch.zeros(n, m, dtype=torch.bool)
    out, tol = torch.zeros(b, n, h, d, dtype=F64), torch.zeros(b, n, h, d, dtype=F64)
    lse, ltol = torch.zeros(b, h, n, dtype=F64), torch.zeros(b, h, n, dtype=F64)
    pu = R.u(t) ** 2 if n * (h // kh) <= 16 else R.u(t)
    for x in range(b):
        for y in range(h):
            kk, vv, qq = k[x, :, y * kh // h], v[x, :, y * kh // h], q[x, :, y]
            s = (qq @ kk.T) * d ** -0.5
            es = (d + 8) * 2.0 ** -24 * (qq.abs() @ kk.abs().T) * d ** -0.5
            if softcap > 0:
                s = softcap * torch.tanh(s / softcap)
                es = es + (softcap * 2.0 ** -21 if softcap <= 64 else 0.0)
            if slopes is not None:
                s = s - float(slopes[y]) * (i - j).abs()
                es = es + abs(float(slopes[y])) * (i - j).abs() * 2.0 ** -20
            es = (es + 2.0 ** -20 * s.abs()).nan_to_num(0.0, 0.0, 0.0).masked_fill(hidden, 0.0).amax(1, keepdim=True)
            s = s.masked_fill(hidden, -math.inf)
            top = s.amax(1, keepdim=True)
            p = torch.exp(s - top)
            total = p.sum(1, keepdim=True)
            out[x, :, y] = (p @ vv) / total
            floor = ((~hidden).to(F64) @ vv.abs()) * (2.0 ** -36 if t is F16 else 0.0)
            tol[x, :, y] = ((p @ vv.abs()) * (pu + 2 * es + 2.0 ** -19) + floor) / total + R.u(t) * out[x, :, y].abs() + R.least(t)
            lse[x, y] = (top + torch.log(total))[:, 0]
            ltol[x, y] = es[:, 0] + 2.0 ** -19 + 2.0 ** -21 * lse[x, y].abs()
    return out, lse, tol, ltol


def check(q, k, v, **kw):
    out, lse = ops.attention(q, k, v, return_lse=True, **{x: (y.cuda() if isinstance(y, torch.Tensor) else y) for x, y in kw.items()})
    want, wlse, tol, ltol = reference(q, k, v, **kw)
    R.close(out, want, tol, "out")
    R.close(lse, wlse, ltol, "lse")
    return out, lse


# rows per key head and keys: single tokens, a few, one tile, several tiles, each whole and in parts
PATHS = [(1, 300), (3, 2100), (40, 300), (40, 2100), (200, 260)]


# ------------------------------------------------------------------------------------------------------------------- caps
@pytest.mark.parametrize("n,m", PATHS)
@pytest.mark.parametrize("t,d", [(F16, 64), (BF16, 128)])
@pytest.mark.parametrize("cap,mul", [(5.0, 1.5), (64.0, 1.5), (65.0, 1.5), (65.0, 60.0), (300.0, 1.5), (300.0, 150.0), (1e4, 1.5), (1e4, 3000.0),
                                     (1e6, 1.5), (1e8, 30.0), (1e30, 1.5)])
def test_caps(cap, mul, t, d, n, m):
    q, k, v = rnd((2, n, 2, d), t, 1, mul), rnd((2, m, 1, d), t, 2), rnd((2, m, 1, d), t, 3)
    check(q, k, v, softcap=cap, causal=True)


@pytest.mark.parametrize("n,m", PATHS)
def test_caps_with_slopes(n, m):
    q, k, v = rnd((1, n, 2, 96), BF16, 4, 2.0), rnd((1, m, 1, 96), BF16, 5), rnd((1, m, 1, 96), BF16, 6)
    for cap in (20.0, 1e3, 1e7):
        check(q, k, v, softcap=cap, slopes=torch.tensor([0.25, -0.001]))


@pytest.mark.parametrize("n,m", PATHS)
@pytest.mark.parametrize("t,d", [(F16, 32), (BF16, 128)])
def test_a_cap_far_above_the_scores_changes_nothing(t, d, n, m):
    q, k, v = rnd((2, n, 2, d), t, 7, 2.0), rnd((2, m, 2, d), t, 8), rnd((2, m, 2, d), t, 9)
    plain, capped = (ops.attention(q, k, v, softcap=c, return_lse=True) for c in (0.0, 1e30))
    assert torch.equal(plain[0], capped[0]) and torch.equal(plain[1], capped[1])


@pytest.mark.parametrize("n,m", PATHS)
@pytest.mark.parametrize("cap", [30.0, 1e3])
def test_infinite_scores_are_capped(cap, n, m):
    q, k, v = rnd((1, n, 2, 64), BF16, 10).abs() + 0.1, rnd((1, m, 1, 64), BF16, 11), rnd((1, m, 1, 64), BF16, 12)
    k[0, 5], k[0, 6] = math.inf, -math.inf
    check(q, k, v, softcap=cap)


# ------------------------------------------------------------------------------------------- weights far below the largest
@pytest.mark.parametrize("away", [12.0, 17.0, 18.0, 21.0])
@pytest.mark.parametrize("t,d", [(F16, 64), (F16, 128), (BF16, 64)])
@pytest.mark.parametrize("n,m", [(1, 131072), (4, 20000), (40, 20000), (130, 3000)])
def test_many_keys_far_below_a_sink(n, m, t, d, away):
    # one key without a value of its own stands `away` above all others, whose weights then make up the whole result
    q, k, v = torch.zeros((1, n, 1, d), dtype=t), torch.zeros((1, m, 1, d), dtype=t), rnd((1, m, 1, d), t, 13).abs().cpu() + 0.5
    q[..., 0], k[0, m // 3, 0, 0], v[0, m // 3] = 1.0, away * d ** 0.5, 0.0
    check(q.cuda(), k.cuda(), v.cuda())


@pytest.mark.parametrize("n,m", PATHS)
@pytest.mark.parametrize("away", [8.0, 16.0])
def test_weights_far_below_a_sink_of_all_sizes(away, n, m):
    q, k, v = rnd((2, n, 2, 64), F16, 14), rnd((2, m, 1, 64), F16, 15), rnd((2, m, 1, 64), F16, 16).abs()
    q[..., 0], k[..., 0] = 1.0, 0.0
    k[:, 1, :, 0], v[:, 1] = away * 8, 0.0
    check(q, k, v, causal=n > 1 and m > n)


# ------------------------------------------------------------------------------------------------------------ 8-bit codes
def codes_of(y, s, quant):
    """round(y / s) in f32 as a whole number or e4m3 (nearest, ties to even), where s is a rounded quotient of the group's largest |y|."""
    v = (y.view(*s.shape, -1) / s[..., None]).view(y.shape)
    most = 127.0 if quant == "int8" else 448.0
    v = v.clamp(-most, most)
    return v.round().to(torch.int8) if quant == "int8" else v.to(torch.float8_e4m3fn)


@pytest.mark.parametrize("quant", ["int8", "e4m3"])
@pytest.mark.parametrize("cols,group,rows", [(4096, 0, 4096), (4096, 128, 4096), (1000, 0, 8000), (64, 32, 60000), (11320, 0, 999), (20000, 0, 300)])
def test_codes_are_rounded_quotients(cols, group, rows, quant):
    x, w = rnd((rows, cols), F32, 17), rnd((cols,), F32, 18) + 1
    y = ops.rms_norm(x, w).cpu()
    q, s = ops.rms_norm(x, w, quant=quant, group=group)
    q, s = q.cpu(), s.cpu()
    most = 127.0 if quant == "int8" else 448.0
    largest = y.view(rows, -1, group or cols).abs().amax(-1)
    assert torch.equal(s, largest / torch.tensor(most))
    want = codes_of(y, s, quant)
    assert torch.equal(q.view(torch.uint8), want.view(torch.uint8)), int((q.view(torch.uint8) != want.view(torch.uint8)).sum())
    assert (q.float().view(rows, -1, group or cols).abs().amax(-1) == most).all()      # the group's largest value gets the largest code


@pytest.mark.parametrize("quant,most", [("int8", 127), ("e4m3", 448)])
def test_scales_of_few_bits(quant, most):
    # values of some hundred of f32's smallest steps: the scale is a step or two, off by up to a third, and codes end at the largest one
    step = 2.0 ** -149
    for top in (0.4, 0.6, 1.0, 1.4, 1.49, 2.4, 3.5, 100.0, 1e4):
        w = (torch.linspace(-1.0, 1.0, 64, dtype=F64) * (top * most)).round() * step
        x = torch.ones((3, 64), device="cuda")
        y = ops.rms_norm(x, w.float().cuda(), eps=0.0).cpu()
        assert torch.equal(y[0], w.float())                 # 1 / sqrt(1) and the product are exact
        q, s = ops.rms_norm(x, w.float().cuda(), eps=0.0, quant=quant)
        want = (y.abs().amax(1, keepdim=True).double() / step / most).round() * step
        want = torch.where(want == 0, torch.ones_like(want), want)
        assert torch.equal(s.cpu().double(), want), (float(s[0]), float(want[0]))
        ratio = (y.double() / want).float().clamp(-most, most)      # exact: both are whole numbers of steps below 2^24
        code = ratio.round().to(torch.int8) if quant == "int8" else ratio.to(torch.float8_e4m3fn)
        assert torch.equal(q.cpu().view(torch.uint8), code.view(torch.uint8)), top


# ------------------------------------------------------------------------------------------------ values near the type's end
@pytest.mark.parametrize("n,m", PATHS + [(1, 9000), (16, 20), (40, 9000)])
@pytest.mark.parametrize("d", [32, 128])
@pytest.mark.parametrize("size", [1e31, 1e36, 3.3e38])
def test_sums_of_values_near_the_end_of_bf16(size, d, n, m):
    # a mean of finite values is finite, however many of them there are
    q, k = rnd((2, n, 2, d), BF16, 19), rnd((2, m, 1, d), BF16, 20)
    v = (torch.rand((2, m, 1, d), generator=torch.Generator().manual_seed(21)) * 0.5 + 0.5) * size
    v[1, :, :, ::2] *= -1
    v[0, :, :, 1] = 1.0                            # an ordinary column beside them
    out, _ = check(q, k, v.to(BF16).cuda(), causal=n > 1)
    assert out.isfinite().all()


@pytest.mark.parametrize("n,m", PATHS)
def test_infinities_beside_values_near_the_end(n, m):
    q, k = rnd((1, n, 1, 64), BF16, 22), rnd((1, m, 1, 64), BF16, 23)
    v = torch.full((1, m, 1, 64), 3.3e38, dtype=BF16)
    v[0, 3, 0, 5], v[0, 4, 0, 6], v[0, 5, 0, 7] = math.inf, -math.inf, math.nan
    out = ops.attention(q, k, v.cuda())
    assert (out[..., 5] == math.inf).all() and (out[..., 6] == -math.inf).all() and out[..., 7].isnan().all()
    want = reference(q, k, torch.full_like(v, 3.3e38))
    rest = [c for c in range(64) if c not in (5, 6, 7)]
    R.close(out[..., rest], want[0][..., rest], want[2][..., rest], "other columns")


# ------------------------------------------------------------------------------------------------------- scores of -infinity
@pytest.mark.parametrize("n,m", PATHS + [(1, 9000), (40, 9000)])
@pytest.mark.parametrize("slopes", [False, True])
@pytest.mark.parametrize("t,d", [(F16, 64), (BF16, 128)])
def test_only_scores_of_minus_infinity(t, d, slopes, n, m):
    q, k, v = rnd((1, n, 2, d), t, 24).abs() + 0.1, rnd((1, m, 1, d), t, 25), rnd((1, m, 1, d), t, 26)
    low = torch.full_like(k, -math.inf)
    kw = dict(slopes=torch.tensor([0.5, 0.01], device="cuda")) if slopes else {}
    out, lse = ops.attention(q, low, v, return_lse=True, **kw)
    assert (out == 0).all() and (lse == -math.inf).all()
    # the first keys only: rows that see no other give zeros, the others what they would without those keys
    first = m - n // 2 - 1
    low[:, first:] = k[:, first:]
    out, lse = ops.attention(q, low, v, causal=True, return_lse=True, **kw)
    blind = first - (m - n)          # rows 0 .. blind - 1 stand before key `first`
    assert blind >= 0 and (out[:, :blind] == 0).all() and (lse[:, :, :blind] == -math.inf).all()
    want, wlse = ops.attention(q[:, blind:], k[:, first:], v[:, first:], causal=True, return_lse=True, **kw)
    bound = reference(q[:, blind:], k[:, first:], v[:, first:], causal=True, slopes=kw["slopes"].cpu() if slopes else None)
    R.close(out[:, blind:], bound[0], bound[2], "out")
    R.close(lse[:, :, blind:], bound[1], bound[3], "lse")
    R.close(want, bound[0], bound[2], "alone")
    R.close(wlse, bound[1], bound[3], "lse alone")


# ----------------------------------------------------------------------------------------------------- errors of other calls
def hip_runtime():
    path = next(line.split()[-1] for line in open("/proc/self/maps") if "libamdhip64" in line)
    return ctypes.CDLL(path)


@pytest.mark.parametrize("which", ["norm", "rope", "attention", "parts"])
def test_an_older_error_is_not_taken_for_the_calls_own(which):
    # a call of the program's own that failed (here: a device that does not exist) leaves its error behind for who asks next
    x, f, long = rnd((1, 4, 2, 64), F16, 27), ops.rope_frequencies(64), rnd((1, 6000, 2, 64), F16, 28)
    call = {"norm": lambda: ops.rms_norm(x), "rope": lambda: ops.rope(x, freqs=f), "attention": lambda: ops.attention(x, x, x),
            "parts": lambda: ops.attention(x, long, long)}[which]
    want, hip = call(), hip_runtime()
    torch.cuda.synchronize()
    assert hip.hipSetDevice(99) != 0
    try:
        got = call()
    finally:
        left = hip.hipGetLastError()
    assert left != 0 and torch.equal(got, want)      # nor is it taken away from the program


def test_a_failed_call_leaves_no_error_behind():
    x, hip = rnd((4, 64), F16, 29), hip_runtime()
    args = ops._NORM_ARGS.pack(x.data_ptr(), 0, 0, 0, x.data_ptr(), 0, 4, 64, 64, 64, 64, 0, 64, 0, 0, 0, 0, 1.0, 1e-5, 0)
    hip.hipGetLastError()
    assert ops._entry()[0](99, 0, args) == -2 and capi.lib().mibc_last_error(None).decode().startswith("rms_norm: device: ")
    assert hip.hipGetLastError() == 0


@pytest.mark.parametrize("n,m", PATHS + [(1, 9000), (40, 9000)])
def test_values_beside_scores_of_minus_infinity(n, m):
    # no key has a weight: zeros, and NaN in the columns where a seen value is not finite
    q, k, v = rnd((1, n, 1, 64), BF16, 30).abs() + 0.1, torch.full((1, m, 1, 64), -math.inf, dtype=BF16, device="cuda"), rnd((1, m, 1, 64), BF16, 31)
    v[0, m // 2, 0, 3], v[0, m // 3, 0, 4], v[0, 0, 0, 5] = math.nan, math.inf, -math.inf
    out, lse = ops.attention(q, k, v, return_lse=True)
    assert out[..., 3:6].isnan().all() and (out[..., :3] == 0).all() and (out[..., 6:] == 0).all() and (lse == -math.inf).all()


# ----------------------------------------------------------------------------------------------------------- scores of any size
@pytest.mark.parametrize("n,m", PATHS + [(1, 9000), (40, 9000)])
@pytest.mark.parametrize("t,size", [(F16, 3.0), (F16, 1000.0), (F16, 8000.0), (F16, 60000.0), (BF16, 1e4), (BF16, 1e8), (BF16, 1e13), (BF16, 1e17)])
@pytest.mark.parametrize("cap", [0.0, 1e25])
def test_one_key_takes_all(cap, t, size, n, m):
    # one key along the queries, the others against them: its value and nothing else, at scores from 1e2 to 1e36
    q, v = torch.full((2, n, 2, 64), size, dtype=t), rnd((2, m, 1, 64), t, 32)
    q[1] *= 0.7
    k = torch.full((2, m, 1, 64), -size, dtype=t)
    at = (m - n) // 2                                  # seen by every row
    k[:, at] *= -0.9
    out, lse = ops.attention(q.cuda(), k.cuda(), v, causal=True, return_lse=True, softcap=cap)
    assert torch.equal(out, v[:, at:at + 1].expand(2, n, 2, 64))
    s = (q.double() * k[:, at:at + 1].double()).sum(-1).transpose(1, 2) * 64 ** -0.5
    if cap:
        s = cap * torch.tanh(s / cap)
    assert ((lse.cpu().double() - s).abs() <= 2.0 ** -18 * s).all()


@pytest.mark.parametrize("n,m", PATHS)
@pytest.mark.parametrize("t,low,size", [(F16, -65504.0, 1.0), (F16, -65504.0, 300.0), (BF16, torch.finfo(BF16).min, 1e-3), (BF16, -1e30, 1e-3), (BF16, 1e20, 1e10)])
def test_equal_scores_of_any_size_give_the_mean(t, low, size, n, m):
    # every key at the type's lowest value (or far up): finite scores, all the same
    q, k, v = torch.full((1, n, 1, 128), size, dtype=t, device="cuda"), torch.full((1, m, 1, 128), low, dtype=t, device="cuda"), rnd((1, m, 1, 128), t, 33)
    out, lse = ops.attention(q, k, v, return_lse=True)
    want = v.double().mean(1, keepdim=True).expand(1, n, 1, 128).cpu()
    # in parts, weights of parts whose lengths differ by a tile of at most 64 keys in at least 256 are equal to within the score's rounding
    parts = v.double().abs().mean().cpu() * 0.5 if m >= 512 else 0.0
    R.close(out, want, R.u(t) * want.abs() + v.double().abs().mean(1, keepdim=True).cpu() * (R.u(t) + 2.0 ** -19) + parts, "mean")
    s = float(q[0, 0, 0, 0]) * float(k[0, 0, 0, 0]) * 128 ** 0.5 + math.log(m)
    assert ((lse.cpu().double() - s).abs() <= 2.0 ** -18 * abs(s)).all()


@pytest.mark.parametrize("n,m", PATHS)
def test_large_scores_behind_ordinary_ones(n, m):
    # keys at the lowest value first, ordinary ones behind them: as if the first were not there
    q, k, v = rnd((1, n, 2, 64), BF16, 34).abs() + 0.1, rnd((1, m, 1, 64), BF16, 35), rnd((1, m, 1, 64), BF16, 36)
    low = k.clone()
    low[:, :m - n - 20] = -1e37
    want = reference(q, k[:, m - n - 20:], v[:, m - n - 20:], causal=True)
    out, lse = ops.attention(q, low, v, causal=True, return_lse=True)
    R.close(out, want[0], want[2], "out")
    R.close(lse, want[1], want[3], "lse")
