"""Plain 64-bit implementations of the transformer-layer operators (dorado_amd.ops), on the CPU, and how far a kernel that keeps
sums, statistics and products in f32 may be from them.  u(t) = half a step of t relative to the value."""
import math

import torch

F64 = torch.float64


def u(t):
    return torch.finfo(t).eps / 2


def least(t):
    """Half the distance of t's subnormal values: what a rounding below its normal range is off by (f16: steps of 2^-24)."""
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def rms_norm(x, weight=None, residual=None, alpha=1.0, eps=1e-5):
    """(y, h) in f64."""
    h = x.cpu().to(F64)
    if residual is not None:
        h = h + alpha * residual.cpu().to(F64)
    y = h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps)
    return (y if weight is None else y * weight.cpu().to(F64)), h


def rms_norm_tolerance(y, x, weight, residual, alpha, t):
    """Rounding of the output, and f32 arithmetic on the way: the sum x + alpha r is off by 2^-24 of its terms (which may cancel),
    the sum of squares of C <= 32768 values in chains of at most 32 + 10 additions by 2^-18.6, the root and the products by a few
    2^-24: 2^-18 of the terms in all."""
    terms = x.cpu().to(F64).abs()
    if residual is not None:
        terms = terms + abs(alpha) * residual.cpu().to(F64).abs()
    h = x.cpu().to(F64) + (0 if residual is None else alpha * residual.cpu().to(F64))
    grow = terms / torch.sqrt(h.square().mean(-1, keepdim=True) + 1e-5)
    if weight is not None:
        grow = grow * weight.cpu().to(F64).abs()
    return u(t) * y.abs() + 2.0 ** -18 * (grow + y.abs()) + least(t)


def rope(x, freqs, positions, interleaved=False, amplitude=1.0):
    """x [batch, tokens, heads, d]; positions [batch, tokens] or [tokens]."""
    x = x.cpu().to(F64)
    f = freqs.cpu().to(F64)
    half, r = f.shape[0], 2 * f.shape[0]
    p = positions.cpu().to(F64)
    angle = (p[..., None] * f)[..., None, :]
    if angle.dim() == 3:
        angle = angle[None]
    c, s = angle.cos() * amplitude, angle.sin() * amplitude
    y = x.clone()
    ia, ib = (torch.arange(0, r, 2), torch.arange(1, r, 2)) if interleaved else (torch.arange(half), torch.arange(half, r))
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, a * s + b * c
    return y


def rope_tolerance(y, x, freqs, positions, amplitude, t, interleaved=False):
    """Output rounding; sine and cosine off by 2^-22 (f32 turns and polynomial), four f32 roundings; angles from a product in
    f64 on both sides, off by 2^-52 of the angle each."""
    x = x.cpu().to(F64).abs()
    r = 2 * freqs.shape[0]
    pair = torch.zeros_like(x)
    if interleaved:
        s = x[..., 0:r:2] + x[..., 1:r:2]
        pair[..., 0:r:2], pair[..., 1:r:2] = s, s
    else:
        s = x[..., :r // 2] + x[..., r // 2:r]
        pair[..., :r // 2], pair[..., r // 2:r] = s, s
    angle = float(positions.abs().max()) * float(freqs.max()) if positions.numel() else 0.0
    return u(t) * y.abs() + abs(amplitude) * pair * (2.0 ** -21 + angle * 2.0 ** -51) + least(t)


def visible(b, n, m, window=(-1, -1), k_len=None, prefix=None, doc_offsets=None, q_start=None):
    """bool [b, n, m] and the positions [b, n] of the queries."""
    see = torch.zeros(b, n, m, dtype=torch.bool)
    pos = torch.zeros(b, n, dtype=torch.int64)
    j = torch.arange(m)
    for x in range(b):
        for t in range(n):
            first, last, pre = 0, m, 0
            if doc_offsets is not None:
                o = doc_offsets.tolist()
                d = [e for e in range(len(o) - 1) if o[e] <= t < o[e + 1]]
                pos[x, t] = t
                if not d:
                    continue
                first, last = o[d[0]], o[d[0] + 1]
                pre = 0 if prefix is None else int(prefix[d[0]])
                i = t
            else:
                last = m if k_len is None else max(0, min(m, int(k_len[x])))
                pre = 0 if prefix is None else int(prefix[x])
                i = (last - n if q_start is None else q_start) + t
                pos[x, t] = i
            ok = torch.ones(m, dtype=torch.bool)
            if window[0] >= 0:
                ok &= j >= i - window[0]
            if window[1] >= 0:
                ok &= j <= i + window[1]
            ok |= j < first + pre
            see[x, t] = ok & (j >= first) & (j < last)
    return see, pos


def attention(q, k, v, scale=None, window=(-1, -1), softcap=0.0, slopes=None, k_len=None, prefix=None, doc_offsets=None,
              q_start=None):
    """(out, lse, tolerance of out, tolerance of lse); what a query does not see is left out of its sums altogether."""
    t = q.dtype
    b, n, h, d = q.shape
    m, kh = k.shape[1], k.shape[2]
    scale = d ** -0.5 if scale is None else scale
    q, k, v = (x.cpu().to(F64) for x in (q, k, v))
    see, pos = visible(b, n, m, window, k_len, prefix, doc_offsets, q_start)
    out, tol = torch.zeros(b, n, h, d, dtype=F64), torch.zeros(b, n, h, d, dtype=F64)
    lse, ltol = torch.full((b, h, n), -math.inf, dtype=F64), torch.zeros(b, h, n, dtype=F64)
    for x in range(b):
        hidden = ~see[x]
        far = (pos[x][:, None] - torch.arange(m)).abs().to(F64)
        for y in range(h):
            kk, vv = k[x, :, y * kh // h], v[x, :, y * kh // h]
            s = (q[x, :, y] @ kk.T) * scale
            size = (q[x, :, y].abs() @ kk.abs().T) * scale
            # f32 sums of d products, the scale, the exponent's own rounding
            es = (d + 8) * 2.0 ** -24 * size + 2.0 ** -22 * s.abs()
            if softcap > 0:
                s = softcap * torch.tanh(s / softcap)
                es = es + softcap * 2.0 ** -20        # exp2, reciprocal and two f32 roundings of cap-sized numbers
            if slopes is not None:
                s = s - float(slopes[y]) * far
                es = es + abs(float(slopes[y])) * far * 2.0 ** -22
            s = s.masked_fill(hidden, -math.inf)
            top = s.max(1, keepdim=True).values if m else torch.full((n, 1), -math.inf, dtype=F64)
            base = torch.where(top.isinf() & (top < 0), torch.zeros_like(top), top)
            p = torch.exp(s - base).masked_fill(hidden, 0.0)
            total = p.sum(1, keepdim=True)
            empty = total[:, 0] == 0
            zero = torch.zeros((), dtype=F64)
            # rows apart: 0 * NaN of what a row does not see must stay out
            strange = ~vv.isfinite().all(1) if m else torch.zeros(0, dtype=torch.bool)
            o = p[:, ~strange] @ vv[~strange]
            for j in strange.nonzero()[:, 0].tolist():
                o = o + torch.where(hidden[:, j, None], zero, p[:, j, None] * vv[j])
            # a column's bound sums over all its finite values, those of keys with a NaN or infinity in another column too: their
            # rounded probabilities enter this column like any other key's
            size_v = vv.abs().masked_fill(~vv.isfinite(), 0.0)
            av = p @ size_v
            e = es.masked_fill(hidden, 0.0).nan_to_num(0.0, 0.0, 0.0).amax(1, keepdim=True) if m else torch.zeros(n, 1, dtype=F64)
            div = torch.where(total == 0, torch.ones_like(total), total)
            out[x, :, y] = torch.where(empty[:, None], zero, o / div)
            # probabilities rounded to t (f16: to 2^-25 below 2^-14), sums of m terms in f32, joins of parts
            sub = (~hidden).to(F64) @ size_v * (2.0 ** -25 if t is torch.float16 else 0.0)
            tol[x, :, y] = (av * (u(t) + 2 * e + 2.0 ** -19) + sub) / div + u(t) * out[x, :, y].abs() + 2.0 ** -25
            lse[x, y] = torch.where(empty, torch.full_like(base[:, 0], -math.inf), base[:, 0] + torch.log(total[:, 0]))
            ltol[x, y] = e[:, 0] + 2.0 ** -19 + 2.0 ** -21 * lse[x, y].abs().nan_to_num(0.0, 0.0, 0.0)
    return out, lse, tol, ltol


def close(got, want, tol, what=""):
    """got within tol of want; infinities and NaN in the same places."""
    got = got.cpu().to(F64)
    fine = want.isfinite()
    assert torch.equal(got.isnan(), want.isnan()), f"{what}: NaN in other places ({int(got.isnan().sum())} / {int(want.isnan().sum())})"
    odd = ~fine & ~want.isnan()
    assert torch.equal(got[odd], want[odd]), f"{what}: infinities differ"
    off = (got - want).abs()[fine]
    over = off > tol.expand_as(want)[fine]
    worst = float((off / tol.expand_as(want)[fine].clamp(min=1e-300)).max()) if off.numel() else 0.0
    print(f"{what}: worst {worst:.3f} of the tolerance")
    assert not over.any(), f"{what}: {int(over.sum())} of {off.numel()} values off, worst {worst:.2f} x tolerance, by {float(off.max()):.3e}"
